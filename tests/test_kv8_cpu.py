"""The 8-bit KV cache calls refuse what they do not take before touching a GPU, and their
float64 restatement agrees with hand-worked values."""
import math

import pytest
import torch

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests import _kv8 as ref

ADDR = 4096  # a stand-in for a device pointer: refused calls never read it


def desc(**over):
    a = dict(num_seqs=1, total_q=1, max_q_len=1, n_heads=4, n_kv_heads=2, head_dim=128, block_size=16, num_blocks=4,
             max_blocks_per_seq=4, max_context=16, qkv_stride=1024, rope_rows=16, rot_dim=128, eps=1e-6, add_one=0,
             output_gate=0)
    a.update(over)
    return ck.attn_desc(**a)


def append(d, **over):
    names = ["qkv", "qn", "kn", "cos", "sin", "pos", "slots", "kc", "vc", "ks", "vs", "q_out", "gate"]
    a = {n: ADDR for n in names}
    a.update(over)
    return abi.lib().ekernel_qk_norm_rope_kv_append_kv8(d, *[a[n] for n in names])


def attend(d, window=0, sinks=0, ws=ADDR, ws_bytes=1 << 40, **over):
    names = ["q", "kc", "vc", "ks", "vs", "table", "cu", "ctx", "gate"]
    a = {n: ADDR for n in names}
    a.update(over)
    out = a.pop("out", ADDR)
    return abi.lib().ekernel_paged_attention_verify_kv8(d, *[a[n] for n in names], window, sinks, ws, ws_bytes, out)


BAD_DESC = [(dict(head_dim=64), -5), (dict(block_size=32), -5), (dict(n_kv_heads=0), -1), (dict(n_heads=0), -1),
            (dict(n_heads=5), -1), (dict(num_blocks=0), -1), (dict(num_blocks=1 << 27), -1),
            (dict(num_seqs=1 << 16), -1), (dict(total_q=1 << 23), -1), (dict(n_heads=2048), -1)]


@pytest.mark.parametrize("over,rc", BAD_DESC + [(dict(rot_dim=3), -1), (dict(rot_dim=130), -1),
                                                (dict(qkv_stride=1023), -1)])
def test_append_refuses_descriptors(over, rc):
    assert append(desc(**over)) == rc and abi.last_error()


@pytest.mark.parametrize("over,rc", BAD_DESC)
def test_attention_refuses_descriptors(over, rc):
    assert attend(desc(**over)) == rc and abi.last_error()


@pytest.mark.parametrize("name", ["qkv", "qn", "kn", "cos", "sin", "pos", "slots", "kc", "vc", "ks", "vs", "q_out"])
def test_append_refuses_null(name):
    assert append(desc(), **{name: None}) == -1 and "null" in abi.last_error()


def test_append_refuses_misaligned_caches_and_a_missing_gate():
    assert append(desc(), kc=ADDR + 8) == -1 and "16-byte" in abi.last_error()
    assert append(desc(), vc=ADDR + 1) == -1 and "16-byte" in abi.last_error()
    assert append(desc(output_gate=1, qkv_stride=1536), gate=None) == -1 and "gate" in abi.last_error()
    f = abi.lib().ekernel_qk_norm_rope_kv_append_kv8_splitk
    assert f(desc(), ADDR, 0, *[ADDR] * 12) == -1 and "splits" in abi.last_error()
    assert f(desc(), None, 1, *[ADDR] * 12) == -1 and "null" in abi.last_error()


@pytest.mark.parametrize("name", ["q", "kc", "vc", "ks", "vs", "table", "cu", "ctx", "out"])
def test_attention_refuses_null(name):
    assert attend(desc(), **{name: None}) == -1 and "null" in abi.last_error()


def test_attention_refuses_bad_workspaces_and_alignment():
    d = desc(num_seqs=8, total_q=8, max_context=8192, max_blocks_per_seq=512)
    need = ck.paged_attention_kv8_workspace_bytes(d)
    assert need > 0
    for kw in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=ADDR + 8)):
        assert attend(d, **kw) == -1 and "workspace" in abi.last_error(), kw
    for n in ("kc", "vc", "q", "out"):
        assert attend(d, **{n: ADDR + 8}) == -1 and "16-byte" in abi.last_error()
    assert attend(desc(output_gate=1), gate=None) == -1 and "gate" in abi.last_error()


def test_empty_calls_do_nothing():
    assert append(desc(total_q=0), qkv=None) == 0
    assert attend(desc(total_q=0), q=None) == 0
    assert attend(desc(num_seqs=0), q=None) == 0


def test_workspace_bytes_of_a_refused_descriptor_is_zero():
    assert ck.paged_attention_kv8_workspace_bytes(desc(head_dim=64)) == 0
    with pytest.raises(ValueError):
        ck.paged_attention_kv8_workspace_bytes(desc(), window=-1)
    with pytest.raises(ValueError):
        ck.paged_attention_kv8_workspace_bytes(desc(), sinks=-1)


def test_wrappers_refuse_cpu_tensors():
    t = torch.zeros(4 * 16 * 2 * 128, dtype=torch.uint8)
    s = torch.zeros(8)
    with pytest.raises(ValueError, match="CUDA"):
        ck.paged_attention_verify_kv8(desc(), t, t, t, s, s, t, t, t, None, t)
    with pytest.raises(ValueError):
        ck.qk_norm_rope_kv_append_kv8(desc(), t, t, t, s, s, t, t, t, t, s, s, t)


def test_argument_module_refuses_what_is_no_call():
    m, t = abi.args(), torch.zeros(1)
    with pytest.raises(TypeError):
        m.append(0, desc())
    with pytest.raises(TypeError):
        m.attention(*range(14))
    with pytest.raises(ValueError, match="PagedAttnDesc"):
        m.append(0, b"short", t, 0, *[t] * 12)
    with pytest.raises(TypeError):
        m.append(0, object(), t, 0, *[t] * 12)
    with pytest.raises(ValueError, match="qkv must be a tensor"):
        m.append(0, desc(), 5, 0, *[t] * 12)
    with pytest.raises(ValueError, match="qkv must be a contiguous"):
        m.append(0, desc(), t, 0, *[t] * 12)
    with pytest.raises(ValueError, match="negative"):
        m.attention(0, desc(), *[t] * 10, -1, 0, t)
    with pytest.raises(ValueError, match="CUDA"):  # a tensor without storage
        m.append(0, desc(), torch.zeros(1024, dtype=torch.bfloat16, device="meta"), 0, *[t] * 12)
    with pytest.raises(ValueError):
        m.bind(1, 2, 0)


# ---- the restatement -------------------------------------------------------------------------

def test_restated_scales_and_steps():
    a = torch.tensor([0.0, 448.0, 449.0, 448 * 2.0 ** -20, 1.0, 1e-30], dtype=torch.float64)
    e = ref.scale_exponent(a)
    assert e[:4].tolist() == [0, 0, 1, -20]
    assert (a[1:] <= torch.ldexp(torch.full((5,), 448.0, dtype=torch.float64), e[1:])).all()
    assert (a[1:] > torch.ldexp(torch.full((5,), 448.0, dtype=torch.float64), e[1:] - 1)).all()
    assert ref.e4m3_step(torch.tensor([1.0, 1.9, 448.0, 2.0 ** -9, 0.0])).tolist() == [2 ** -3, 2 ** -3, 32, 2 ** -9,
                                                                                      2 ** -9]


def test_restated_store_rounds_like_torch_and_keeps_earlier_tokens():
    g = torch.Generator().manual_seed(0)
    codes = (torch.randn((3, 16, 2, 128), generator=g) * 80).to(ref.F8).view(torch.uint8)
    scale = torch.full((3, 2), 2.0 ** -6)
    x = torch.randn((4, 2, 128), generator=g, dtype=torch.float64)
    x[0] *= 100
    val, sc = ref.store(x, [16 + 3, 16 + 4, -1, 40], codes, scale)
    assert torch.equal(val[0], ref.values(codes)[0])
    for h in range(2):
        e = math.log2(sc[1, h])
        assert e == int(e) and x[0, h].abs().max() <= 448 * sc[1, h]
        assert torch.equal(val[1, 3, h], (x[0, h] / sc[1, h]).float().to(ref.F8).double())
        kept = ref.values(codes)[1, :3, h] * 2.0 ** -6
        assert torch.equal(val[1, :3, h], (kept / sc[1, h]).float().to(ref.F8).double())
    assert torch.equal(val[2, 8], (x[3] / sc[2][:, None]).float().to(ref.F8).double())


def test_restated_attention_of_one_visible_key():
    codes = torch.zeros((2, 16, 1, 128), dtype=torch.uint8)
    v = codes.clone()
    v[1] = torch.full((16, 1, 128), 2.0).to(ref.F8).view(torch.uint8)
    v[1, 3] = torch.full((1, 128), 3.0).to(ref.F8).view(torch.uint8)
    s = torch.full((2, 1), 0.5)
    q = torch.ones((1, 128), dtype=torch.bfloat16)
    out, _, _ = ref.attention(q, codes, v, s, s, [[1]], [1], [4], 1, window=1)
    assert (out == 1.5).all()
    out, _, _ = ref.attention(q, codes, v, s, s, [[1]], [1], [4], 1)
    assert torch.allclose(out, torch.full_like(out, (3 * 1.0 + 1.5) / 4))
    out, _, _ = ref.attention(q, codes, v, s, s, [[7]], [1], [4], 1)  # an invalid block reads as zeros
    assert (out == 0).all()
