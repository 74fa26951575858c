"""Paths of the verifier's step on the 8-bit cache that need a model or a batch of a certain size."""
import numpy as np
import pytest
import torch

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from pilm_b200.engine import MTPVerifyEngine
from pilm_b200.qwen3 import PagedKVCacheKV8, Qwen3Shape, Qwen3Verifier, Qwen3Weights
from tests import _kv8 as ref
from tests._gpu import dev
from tests.test_gpu_kv8 import i32, make_desc, table_of

pytestmark = pytest.mark.gpu
HD = 128


@pytest.fixture(scope="module", autouse=True)
def _init():
    abi.init()
    yield


@pytest.mark.parametrize("gated,window,sinks", [(False, 0, 0), (True, 30, 2)])
def test_the_projections_partial_sums_give_the_same_step(monkeypatch, gated, window, sinks):
    """A hidden size whose q/k/v projection runs split over K: the append takes its partial sums, in
    prompt chunks and in verify passes, and the step's results, cache and queries are those of the
    summed projection."""
    shape = Qwen3Shape(hidden=2048, layers=2, n_heads=8, n_kv_heads=2, head_dim=HD, intermediate=512, vocab=1024, gated=gated)
    w = Qwen3Weights.synthetic(shape, 5, dev())
    calls = {"splits": [], "whole": 0}
    real, real_whole = ck.qk_norm_rope_kv_append_kv8_splitk, ck.qk_norm_rope_kv_append_kv8

    def splitk(desc, part, splits, *rest):
        calls["splits"].append((int(desc.total_q), splits))
        real(desc, part, splits, *rest)

    def whole(*a):
        calls["whole"] += 1
        real_whole(*a)
    monkeypatch.setattr(ck, "qk_norm_rope_kv_append_kv8_splitk", splitk)
    monkeypatch.setattr(ck, "qk_norm_rope_kv_append_kv8", whole)
    runs = []
    for defer in (True, False):
        calls.update(splits=[], whole=0)
        kv = PagedKVCacheKV8(shape, 64, dev())
        ver = Qwen3Verifier(w, kv, max_rows=256, max_pos=512, device=dev(), window=window, sinks=sinks)
        ver.defer_splitk = defer
        eng = MTPVerifyEngine(ver, num_blocks=64, max_model_len=512, use_graphs=False, page_aligned_chunks=False,
                              max_num_batched_tokens=100)
        rng = np.random.default_rng(4)
        sids = [eng.add_request([int(t) for t in rng.integers(0, 1024, 20 + 3 * i)], 24) for i in range(8)]
        first = eng.prefill()
        prompt_calls = len(calls["splits"])
        res = eng.verify_step({s: [11, 12] for s in sids})
        if defer:
            assert prompt_calls and len(calls["splits"]) > prompt_calls, "no projection was left as partial sums"
            assert all(n > 1 for _, n in calls["splits"]) and {t for t, _ in calls["splits"]} >= {24}
        else:
            assert not calls["splits"] and calls["whole"]
        runs.append((first, [(r.accepted, r.next_token) for r in res], ver.q[:24].clone(),
                     [t.clone() for t in kv.k + kv.v + kv.k_scale + kv.v_scale]))
    assert runs[0][:2] == runs[1][:2] and torch.equal(runs[0][2], runs[1][2])
    assert all(torch.equal(x, y) for x, y in zip(runs[0][3], runs[1][3]))


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv,window", [
    ([1], [301], 16, 8, 0), ([3] * 40, [900] * 40, 32, 8, 0), ([1], [20000], 16, 2, 0), ([12], [9000], 32, 8, 0),
    ([300, 200], [300, 900], 8, 2, 50)])
def test_calls_allocate_nothing_in_the_library(q_lens, ctxs, nh, nkv, window):
    """Append and attention of a new shape, called and captured: the library's own allocations stay what
    they were (both calls run its host code, unlike a replay)."""
    d = dev()
    b = ref.batch(q_lens, ctxs, 1)
    desc = make_desc(b, nh, nkv, rope_rows=max(ctxs))
    g = torch.Generator(device=d).manual_seed(0)
    qkv = torch.randn((b.total, (nh + 2 * nkv) * HD), generator=g, device=d).to(torch.bfloat16)
    one = torch.ones(HD, dtype=torch.bfloat16, device=d)
    cos, sin = torch.ones((max(ctxs), 64), device=d), torch.zeros((max(ctxs), 64), device=d)
    cache = ref.random_cache(b.blocks, nkv, 1, d)
    q, out = torch.empty((b.total, nh * HD), dtype=torch.bfloat16, device=d), torch.empty((b.total, nh * HD), dtype=torch.bfloat16, device=d)
    meta = i32(b.positions), i32(b.slots), table_of(b), i32(b.cu), i32(b.ctxs)
    ws = torch.empty(ck.paged_attention_kv8_workspace_bytes(desc, window, 0), dtype=torch.uint8, device=d)

    def step():
        ck.qk_norm_rope_kv_append_kv8(desc, qkv, one, one, cos, sin, meta[0], meta[1], *cache, q)
        ck.paged_attention_verify_kv8(desc, q, *cache, *meta[2:], None, out, window=window, workspace=ws)
    before, launches = abi.alloc_count(), abi.launch_count()
    step()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert abi.launch_count() - launches >= 6 and abi.alloc_count() == before
    assert torch.equal(out, want)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv,window", [
    ([1], [301], 16, 8, 0), ([3] * 40, [900] * 40, 32, 8, 0), ([1], [20000], 16, 2, 0), ([12], [9000], 32, 8, 0),
    ([300, 200], [300, 900], 8, 2, 50), ([8, 5], [700, 650], 8, 2, 0)])
def test_the_same_call_gives_the_same_bits(q_lens, ctxs, nh, nkv, window):
    """Whatever the workspace held before: nothing is added in an order that varies."""
    d = dev()
    b = ref.batch(q_lens, ctxs, 2)
    desc = make_desc(b, nh, nkv)
    q = torch.randn((b.total, nh * HD), generator=torch.Generator(device=d).manual_seed(1), device=d).to(torch.bfloat16)
    cache = ref.random_cache(b.blocks, nkv, 3, d)
    ws = torch.empty(ck.paged_attention_kv8_workspace_bytes(desc, window, 0), dtype=torch.uint8, device=d)
    want = None
    for fill in (0, 0xFF, 0x7F, None, None):
        ws.fill_(fill) if fill is not None else ws.random_(0, 256)
        out = torch.empty_like(q)
        ck.paged_attention_verify_kv8(desc, q, *cache, table_of(b), i32(b.cu), i32(b.ctxs), None, out, window=window, workspace=ws)
        want = out if want is None else want
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("seqs,rows", [(0, 0), (2, 0), (0, 3)])
@pytest.mark.parametrize("max_q", [1, 64])
def test_empty_batches_through_the_wrappers(seqs, rows, max_q):
    """No rows, no sequences or neither, with the workspace allocated by the call: nothing is written."""
    d, nh, nkv = dev(), 8, 2
    cache = ref.random_cache(4, nkv, 1, d)
    before = [t.clone() for t in cache]
    desc = ck.attn_desc(num_seqs=seqs, total_q=rows, max_q_len=max_q, n_heads=nh, n_kv_heads=nkv, head_dim=HD, block_size=16,
                        num_blocks=4, max_blocks_per_seq=4, max_context=64, qkv_stride=(nh + 2 * nkv) * HD, rope_rows=64,
                        rot_dim=HD, eps=1e-6, add_one=0, output_gate=0)
    q = torch.zeros((rows, nh * HD), dtype=torch.bfloat16, device=d)
    out = torch.full_like(q, 7.25)
    table = torch.zeros((seqs, 4), dtype=torch.int32, device=d)
    ck.paged_attention_verify_kv8(desc, q, *cache, table, i32([0] * (seqs + 1)), i32([0] * seqs), None, out)
    if rows == 0:
        one, angle = torch.ones(HD, dtype=torch.bfloat16, device=d), torch.ones((64, 64), device=d)
        none = i32([])
        ck.qk_norm_rope_kv_append_kv8(desc, torch.empty((0, (nh + 2 * nkv) * HD), dtype=torch.bfloat16, device=d), one, one, angle,
                                      angle, none, none, *cache, q)
    torch.cuda.synchronize()
    assert (out == 7.25).all() and all(torch.equal(x, y) for x, y in zip(before, cache))
