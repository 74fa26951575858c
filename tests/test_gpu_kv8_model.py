"""The Qwen3 verifier and the verify engine on the 8-bit KV cache."""
import numpy as np
import pytest
import torch

from oracle import model as om
from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from pilm_b200 import qwen3
from pilm_b200.engine import MTPVerifyEngine
from pilm_b200.qwen3 import PagedKVCache, PagedKVCacheKV8, Qwen3Shape, Qwen3Verifier, Qwen3VerifierF32, Qwen3Weights
from tests import _kv8 as ref
from tests._gpu import dev
from tests.test_gpu_kv8 import check_store

pytestmark = pytest.mark.gpu
HD = 128


@pytest.fixture(scope="module", autouse=True)
def _init():
    abi.init()
    yield


def weights(gated=False, gemma=False, partial=1.0, layers=2, seed=7):
    shape = Qwen3Shape(hidden=256, layers=layers, n_heads=8, n_kv_heads=2, head_dim=HD, intermediate=512, vocab=1024,
                       gated=gated, gemma_norm=gemma, partial_rotary=partial)
    return Qwen3Weights.synthetic(shape, seed, dev())


def verifier(w, window=0, sinks=0, kv8=True, blocks=64):
    kv = (PagedKVCacheKV8 if kv8 else PagedKVCache)(w.shape, blocks, dev())
    return Qwen3Verifier(w, kv, max_rows=256, max_pos=512, device=dev(), **(dict(window=window, sinks=sinks) if kv8 else {}))


def engine(w, prompts, new=24, **kw):
    eng_kw = {k: kw.pop(k) for k in list(kw) if k in ("use_graphs", "page_aligned_chunks", "max_num_batched_tokens",
                                                      "temperature", "sample_seed")}
    ver = verifier(w, **kw)
    eng = MTPVerifyEngine(ver, num_blocks=64, max_model_len=512, **eng_kw)
    sids = [eng.add_request(list(p), new) for p in prompts]
    return eng, sids


def prompts(n=3, seed=0, lens=(70, 19, 133)):
    rng = np.random.default_rng(seed)
    return [[int(t) for t in rng.integers(0, 1024, lens[i])] for i in range(n)]


@pytest.mark.parametrize("gated,gemma,partial", [(False, False, 1.0), (True, True, 0.25)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_every_layer_of_a_forward_matches_the_operators_restated(monkeypatch, gated, gemma, partial, window, sinks):
    """Prompt chunks and a verify pass: each append and attention that the forward calls is
    checked against its float64 restatement on that call's own inputs.  (Two whole runs are not
    compared: a bf16 unit of difference in a layer's input moves one e4m3 code in 2^5 by a step,
    2^-3 of its value, so their hidden states differ by more than the model tolerance.)"""
    w = weights(gated, gemma, partial)
    eng, sids = engine(w, prompts(), window=window, sinks=sinks, use_graphs=False, page_aligned_chunks=False,
                       max_num_batched_tokens=100)
    calls = {"append": 0, "attend": 0}
    real_append, real_attend = ck.qk_norm_rope_kv_append_kv8, ck.paged_attention_verify_kv8

    def append(desc, qkv, qn, kn, cos, sin, pos, slots, kc, vc, ks, vs, q_out, gate=None):
        calls["append"] += 1
        before = [t.clone() for t in (kc, vc, ks, vs)]
        real_append(desc, qkv, qn, kn, cos, sin, pos, slots, kc, vc, ks, vs, q_out, gate)
        nh, nkv, T, rot = desc.n_heads, desc.n_kv_heads, desc.total_q, desc.rot_dim
        x = qkv.double()
        qw = nh * HD * (2 if desc.output_gate else 1)
        c, s = cos.double()[pos.long()], sin.double()[pos.long()]
        heads = x[:, :qw].reshape(T, nh, -1)
        q = ref.rms_rope(heads[..., :HD], qn, c, s, rot, desc.eps, desc.add_one)
        assert ((q_out.double().view(T, nh, HD) - q).abs() <=
                2.0 ** -8 * q.abs() + 2.0 ** -20 * q.abs().amax(-1, keepdim=True)).all()
        if desc.output_gate:
            assert torch.equal(gate.view(T, nh, HD), qkv[:, :qw].reshape(T, nh, -1)[..., HD:])
        k = ref.rms_rope(x[:, qw:qw + nkv * HD].reshape(T, nkv, HD), kn, c, s, rot, desc.eps, desc.add_one)
        v = x[:, qw + nkv * HD:qw + 2 * nkv * HD].reshape(T, nkv, HD)
        check_store(k, slots.tolist(), before[0], before[2], kc, ks)
        check_store(v, slots.tolist(), before[1], before[3], vc, vs)

    def attend(desc, q, kc, vc, ks, vs, table, cu, ctx, gate, out, window=0, sinks=0, workspace=None):
        calls["attend"] += 1
        real_attend(desc, q, kc, vc, ks, vs, table, cu, ctx, gate, out, window=window, sinks=sinks, workspace=workspace)
        c = cu.tolist()
        want, pv, sb = ref.attention(q, kc, vc, ks, vs, table.tolist(), [y - x for x, y in zip(c, c[1:])], ctx.tolist(),
                                     desc.n_kv_heads, gate, window, sinks)
        ref.assert_attention(out, want, pv, sb, 512)

    monkeypatch.setattr(ck, "qk_norm_rope_kv_append_kv8", append)
    monkeypatch.setattr(ck, "paged_attention_verify_kv8", attend)
    eng.v.defer_splitk = False
    eng.prefill()
    eng.verify_step({s: [11, 12] for s in sids})
    assert calls["append"] == calls["attend"] >= 6


def test_deferred_partials_give_the_same_cache_and_queries():
    """The forward with the projections' split-K partials summed by the append, and without."""
    w = weights()
    runs = []
    for defer in (True, False):
        eng, sids = engine(w, prompts(), use_graphs=False, page_aligned_chunks=False)
        eng.v.defer_splitk = defer
        first = eng.prefill()
        res = eng.verify_step({s: [11, 12] for s in sids})
        runs.append((first, [(r.accepted, r.next_token) for r in res],
                     [t.clone() for t in eng.v.kv.k + eng.v.kv.v + eng.v.kv.k_scale + eng.v.kv.v_scale]))
    assert runs[0][:2] == runs[1][:2]
    for x, y in zip(runs[0][2], runs[1][2]):
        assert torch.equal(x, y)


def test_close_to_the_bf16_cache():
    """The same prompts through both caches: hidden states within the e4m3 rounding of K and V (2^-4
    of each element at most, 2^-4 / sqrt(3) rms, averaged over a row's keys and dims)."""
    w = weights()
    outs = []
    for kv8 in (True, False):
        eng, _ = engine(w, prompts(), kv8=kv8, use_graphs=False, page_aligned_chunks=False)
        h = []
        fwd = eng.v.forward
        eng.v.forward = lambda b, fwd=fwd, h=h: h.append(fwd(b).float().clone()) or h[-1].to(torch.bfloat16)
        eng.prefill()
        outs.append(h[0])
    a, b = outs
    assert float((a - b).norm() / b.norm()) <= 2 * 2.0 ** -4 / 3 ** 0.5


@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 2)])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_engine_graphs_match_eager_steps(window, sinks, temperature):
    """Whole verify steps from captured graphs and launched eagerly give the same tokens, with
    drafts accepted, rejected and rolled back; no library allocation happens in a replay."""
    w = weights(seed=9)
    runs = []
    for graphs in (True, False):
        eng, sids = engine(w, prompts(), window=window, sinks=sinks, use_graphs=graphs, temperature=temperature,
                           sample_seed=5)
        first = eng.prefill()
        toks = []
        rng = np.random.default_rng(3)
        for step in range(10):
            drafts = {s: [int(t) for t in rng.integers(0, 1024, 2)] for s in sids}
            for r in eng.verify_step(drafts):
                toks.append((r.seq_id, r.accepted, r.next_token))
        runs.append((first, toks))
        if graphs:
            before = abi.alloc_count()
            for g in eng.graphs.values():
                g.replay()
            torch.cuda.synchronize()
            assert abi.alloc_count() == before
    assert runs[0] == runs[1]


def test_accepted_drafts_are_the_models_own_continuation():
    """Feeding the engine its own greedy continuation as drafts accepts them all, over the cache as
    the steps leave it.  A decode without drafts and a verify with them see the same cache values
    only up to page scales (rows of one pass share their page's), so the drafts come from a run of
    the same shape."""
    w = weights(seed=11)
    eng, sids = engine(w, prompts(), new=40)
    eng.prefill()
    accepted = tried = 0
    for step in range(6):
        state = {s: (list(eng.sched.seqs[s].tokens), list(eng.sched.seqs[s].outputs), eng.sched.seqs[s].num_computed)
                 for s in sids}
        drafts = {s: [] for s in sids}
        for k in range(2):  # the tokens that verifying one more position gives
            for r in eng.verify_step({s: drafts[s] + [0] for s in sids}):
                if len(r.drafts) > len(drafts[r.seq_id]):
                    n = len(drafts[r.seq_id])
                    drafts[r.seq_id] = (drafts[r.seq_id] + [r.next_token]) if r.accepted == n else drafts[r.seq_id]
            for s in sids:
                seq = eng.sched.seqs[s]
                seq.tokens[:], seq.outputs[:], seq.num_computed = list(state[s][0]), list(state[s][1]), state[s][2]
        for r in eng.verify_step(drafts):
            tried += len(r.drafts)
            accepted += r.accepted
    assert tried >= 12 and accepted >= 0.9 * tried


def test_cache_and_verifier_refusals():
    w = weights()
    with pytest.raises(ValueError, match="window"):
        Qwen3Verifier(w, PagedKVCache(w.shape, 4, dev()), max_rows=16, max_pos=64, device=dev(), window=8)
    with pytest.raises(ValueError, match="negative"):
        Qwen3Verifier(w, PagedKVCacheKV8(w.shape, 4, dev()), max_rows=16, max_pos=64, device=dev(), window=-8)
    with pytest.raises(ValueError, match="fp32"):
        Qwen3VerifierF32(w, PagedKVCacheKV8(w.shape, 4, dev()), max_rows=16, max_pos=64, device=dev())
    bad = Qwen3Shape(hidden=256, layers=1, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=512, vocab=64)
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCacheKV8(bad, 4, dev())


def test_random_fill_is_what_the_append_would_store():
    shape = Qwen3Shape(hidden=256, layers=1, n_heads=8, n_kv_heads=2, head_dim=HD, intermediate=512, vocab=1024)
    kv, bf = PagedKVCacheKV8(shape, 9, dev(), "random", 3), PagedKVCache(shape, 9, dev(), "random", 3)
    for codes, scale, x in ((kv.k[0], kv.k_scale[0], bf.k[0]), (kv.v[0], kv.v_scale[0], bf.v[0])):
        val, sc = ref.store(x.double().view(-1, 2, HD), list(range(9 * 16)), torch.zeros_like(codes),
                            torch.ones_like(scale))
        assert torch.equal(sc, scale.double()) and torch.equal(val, ref.values(codes))
    assert kv.bytes_per_token == 2 * 2 * HD + 1
    assert qwen3.attention_bytes(shape, [33], [1], 1) == 33 * 512 + 3 * 16 + 8 * HD * 4 + 512
