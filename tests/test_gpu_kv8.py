"""The 8-bit KV cache operators on the GPU against their float64 restatement (tests/_kv8.py)."""
import math

import pytest
import torch

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests import _kv8 as ref
from tests._gpu import dev
from tests._kv8 import HD, PAGE

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    abi.init()
    yield


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=dev())


def make_desc(b, nh, nkv, gated=False, rot=HD, rope_rows=1, stride=None, add_one=False, max_q=None, max_ctx=None):
    width = (nh * (2 if gated else 1) + 2 * nkv) * HD
    return ck.attn_desc(num_seqs=len(b.q_lens), total_q=b.total, max_q_len=max_q or max([1] + b.q_lens), n_heads=nh,
                        n_kv_heads=nkv, head_dim=HD, block_size=PAGE, num_blocks=b.blocks,
                        max_blocks_per_seq=b.max_pages, max_context=max_ctx or max(1, max(b.ctxs)),
                        qkv_stride=stride or width, rope_rows=rope_rows, rot_dim=rot, eps=1e-6, add_one=add_one,
                        output_gate=gated)


def table_of(b, width=None):
    return i32([t + [0] * ((width or b.max_pages) - len(t)) for t in b.tables])


# ---- append ----------------------------------------------------------------------------------

def check_store(x, slots, before, scale_before, after, scale_after):
    """The cache after a call against exact rows x [T, kv, 128]: a new code is the nearest to its
    exact value, scales and kept codes are exact, everything else is unchanged.
    Nearest up to the fp32 error of that value: the norm's roundings (the sum of squares nine
    deep, halved by the root; the reciprocal root, 2 units; three products) are 10 * 2^-24 of each
    value; a rotation adds two products (one more rounding each) and rounds: 12 * 2^-24 *
    (|a| + |b|), and |a| + |b| <= 2 sqrt(2) times the head's largest rotated value (a rotation
    keeps a pair's norm), so 34 * 2^-24 < 2^-18 of that largest value."""
    val, sc = ref.store(x, slots, before, scale_before)
    assert torch.equal(scale_after.double().nan_to_num(-1), sc.nan_to_num(-1))
    blocks, _, nkv, _ = before.shape
    new = torch.zeros((blocks, PAGE), dtype=torch.bool, device=before.device)
    exact = torch.zeros(before.shape, dtype=torch.float64, device=before.device)
    for r, s in enumerate(slots):
        if 0 <= s < blocks * PAGE:
            new[s // PAGE, s % PAGE] = True
            exact[s // PAGE, s % PAGE] = torch.nan_to_num(x[r], nan=0.0, posinf=1e300, neginf=-1e300)
    got = ref.values(after)
    same = torch.equal(torch.where(new[:, :, None, None], torch.zeros_like(got), got).nan_to_num(-1000),
                       torch.where(new[:, :, None, None], torch.zeros_like(val), val).nan_to_num(-1000))
    assert same, "kept or untouched codes changed"
    y = (exact / sc[:, None, :, None]).clamp(-448, 448)
    err = (got - y).abs()
    tol = ref.e4m3_step(y) * 0.5 + y.abs().amax(-1, keepdim=True) * 2.0 ** -18
    bad = new[:, :, None, None] & ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], y[bad][:4])


def append_case(q_lens, ctxs, nh, nkv, gated=False, rot=HD, add_one=False, seed=0, splits=0, pad=0, misalign=False,
                edit=None, rope_rows=None, max_q=None):
    d = dev()
    b = ref.batch(q_lens, ctxs, seed)
    g = torch.Generator(device=d).manual_seed(seed)
    width = (nh * (2 if gated else 1) + 2 * nkv) * HD
    stride, T = width + pad, b.total
    qkv = (torch.randn((T, stride), generator=g, device=d) * 1.5).to(torch.bfloat16)
    slots = b.slots
    if edit:
        slots = edit(slots, qkv, b)
    qn = (torch.randn(HD, generator=g, device=d) * 0.2 + (0 if add_one else 1)).to(torch.bfloat16)
    kn = (torch.randn(HD, generator=g, device=d) * 0.2 + (0 if add_one else 1)).to(torch.bfloat16)
    rows = rope_rows or max(ctxs)
    freq = 1e6 ** (-torch.arange(rot // 2, dtype=torch.float64, device=d) / max(1, rot // 2))
    ang = torch.arange(rows, dtype=torch.float64, device=d)[:, None] * freq
    cos, sin = ang.cos().float(), ang.sin().float()
    kc, vc, ks, vs = ref.random_cache(b.blocks, nkv, seed + 1, d)
    ref.poison_unused(b, kc, vc, ks, vs)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    desc = make_desc(b, nh, nkv, gated, rot, rows, stride, add_one, max_q=max_q)
    if misalign:  # outputs and projection one element off the vector alignment
        hold = torch.empty(T * nh * HD + 1, dtype=torch.bfloat16, device=d)
        q_out = hold[1:]
        pq = torch.empty(T * stride + 1, dtype=torch.bfloat16, device=d)
        pq[1:] = qkv.flatten()
        src = pq[1:]
    else:
        q_out, src = torch.empty((T, nh * HD), dtype=torch.bfloat16, device=d), qkv
    gate = torch.empty((T, nh * HD), dtype=torch.bfloat16, device=d) if gated else None
    pos, sl = i32(b.positions), i32(slots)
    if splits:
        part = torch.randn((splits, T, stride), generator=g, device=d)
        part[0] = qkv.float() - part[1:].sum(0)
        acc = part[0].clone()  # the kernel's sum, in its order, rounded to bf16
        for s in range(1, splits):
            acc += part[s]
        qkv = acc.to(torch.bfloat16)
        ck.qk_norm_rope_kv_append_kv8_splitk(desc, part, splits, qn, kn, cos, sin, pos, sl, kc, vc, ks, vs, q_out, gate)
    else:
        ck.qk_norm_rope_kv_append_kv8(desc, src, qn, kn, cos, sin, pos, sl, kc, vc, ks, vs, q_out, gate)
    torch.cuda.synchronize()
    x = qkv[:, :width].double()
    p = torch.tensor(b.positions, device=d)
    ok = (p >= 0) & (p < rows)
    at = torch.where(ok, p, 0)
    c = torch.where(ok[:, None], cos.double()[at], 1.0)
    s = torch.where(ok[:, None], sin.double()[at], 0.0)
    qw = nh * (2 if gated else 1) * HD
    heads = x[:, :qw].reshape(T, nh, -1)
    q = ref.rms_rope(heads[..., :HD], qn, c, s, rot, 1e-6, add_one)
    got = q_out.view(T, nh, HD).double()
    # one rounding to bf16; fp32 norm and rotation: a few 2^-24 of the pair's magnitude
    big = q.abs().amax(-1, keepdim=True)
    assert ((got - q).abs() <= 2.0 ** -8 * q.abs() + 2.0 ** -20 * big).all()
    if gated:
        assert torch.equal(gate.view(T, nh, HD), qkv[:, :qw].reshape(T, nh, -1)[..., HD:])
    k = ref.rms_rope(x[:, qw:qw + nkv * HD].reshape(T, nkv, HD), kn, c, s, rot, 1e-6, add_one)
    check_store(k, slots, before[0], before[2], kc, ks)
    check_store(x[:, qw + nkv * HD:].reshape(T, nkv, HD), slots, before[1], before[3], vc, vs)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", [
    ([1], [1], 16, 8),
    ([1], [301], 16, 8),
    ([3, 3, 1, 3], [40, 99, 16, 131], 8, 2),        # rows that end, start and cross pages
    ([5, 4, 3, 2, 1, 6], [21, 16, 33, 18, 17, 70], 16, 2),
    ([16, 17, 33, 1], [16, 17, 40, 5], 32, 8),      # whole pages, and runs over two and three
    ([100, 7], [100, 300], 6, 3),
    ([1733], [1733], 8, 8),
    ([2, 2], [9, 500], 11, 11),
    ([64] * 3, [64, 80, 1000], 40, 8),
])
def test_append(q_lens, ctxs, nh, nkv):
    append_case(q_lens, ctxs, nh, nkv, seed=len(q_lens) + nh)


@pytest.mark.parametrize("rot", [0, 2, 6, 32, 64, 96, 128])
@pytest.mark.parametrize("gated,add_one", [(False, False), (True, True)])
def test_append_rotary_gate_and_gemma(rot, gated, add_one):
    append_case([3, 20], [35, 51], 8, 2, gated, rot, add_one, seed=rot)


@pytest.mark.parametrize("splits", [1, 2, 5])
def test_append_splitk(splits):
    append_case([3, 1, 18], [33, 80, 18], 8, 2, gated=True, seed=splits, splits=splits)


def test_append_unaligned_buffers_and_padded_rows():
    append_case([3, 17], [35, 51], 4, 2, seed=3, misalign=True)
    append_case([3, 17], [35, 51], 4, 2, seed=4, pad=3)
    append_case([3, 17], [35, 51], 4, 2, seed=5, pad=8, splits=2)


def test_append_positions_past_the_rope_table_are_not_rotated():
    append_case([4, 2], [40, 7], 4, 2, seed=6, rope_rows=38)


@pytest.mark.parametrize("rows", [1, 16])
def test_append_rows_without_a_slot(rows):
    """-1 rows (and slots past the pool) anywhere: before, inside and after a page's run, and
    longer stretches of them than a warp looks at once."""
    def edit(slots, qkv, b):
        out = list(slots)
        for i in (0, 2, 3, len(out) - 1):
            out[i] = -1
        for i in range(40, 100):
            out[i] = -1 if i % 3 else b.blocks * PAGE + i
        return out
    append_case([20, 120, 5], [30, 125, 21], 4, 2, seed=7, edit=edit, max_q=rows if rows > 1 else None)


def test_append_a_repeated_slot_keeps_the_last_row():
    def edit(slots, qkv, b):
        return [slots[0]] * 3 + [slots[3]] + [slots[4]] * 40 + slots[44:]
    append_case([50], [70], 4, 2, seed=8, edit=edit)


def test_append_nan_and_infinities():
    def edit(slots, qkv, b):
        v = qkv[:, -2 * HD:]
        v[0, 3], v[1, 5], v[2, 130], v[3, 7] = math.nan, math.inf, -math.inf, 3e38
        qkv[4, -3 * HD] = math.nan   # one NaN makes a whole normalized key NaN: stored as zeros
        return slots
    d = dev()
    b = ref.batch([6], [22], 9)
    append = append_case  # q of row 4 is finite: only K and V hold the values above
    append([6], [22], 4, 2, seed=9, edit=edit)


def test_append_grows_and_shrinks_a_page_scale():
    """A large row raises its page's scale (kept codes round to it); written over by a small one
    the scale falls back, and tokens that stayed normal are what they were."""
    d = dev()
    b = ref.batch([1], [4], 0)
    desc = make_desc(b, 1, 1, rope_rows=64)
    one = torch.ones(HD, dtype=torch.bfloat16, device=d)
    cos, sin = torch.ones((64, 64), device=d), torch.zeros((64, 64), device=d)
    kc, vc, ks, vs = ref.random_cache(b.blocks, 1, 1, d)
    q_out = torch.empty((1, HD), dtype=torch.bfloat16, device=d)
    page = b.tables[0][0]

    def put(offset, v):
        qkv = torch.zeros((1, 3 * HD), dtype=torch.bfloat16, device=d)
        qkv[0, 2 * HD:] = v
        ck.qk_norm_rope_kv_append_kv8(desc, qkv, one, one, cos, sin, i32([offset]), i32([page * PAGE + offset]), kc,
                                      vc, ks, vs, q_out)
    base = torch.randn(HD, generator=torch.Generator(device=d).manual_seed(2), device=d)
    put(0, base)
    put(1, base * 0.5)
    first = ref.values(vc[page, :2]) * vs[page].double()
    scale = vs[page].item()
    put(2, base * 64)
    assert vs[page].item() == scale * 64
    raised = ref.values(vc[page, :2]) * vs[page].double()
    # a value stays unless it became subnormal: below 2^-6 of the new scale it is held to 2^-10 of it
    assert ((raised - first).abs() <= scale * 64 * 2.0 ** -10).all()
    put(2, base)
    assert vs[page].item() == scale
    assert torch.equal(ref.values(vc[page, :2]) * vs[page].double(), raised)


def test_append_is_repeatable():
    """Writing the same rows again changes nothing (a captured step runs twice on its batch)."""
    d = dev()
    b = ref.batch([3, 20], [35, 51], 1)
    desc = make_desc(b, 4, 2, rope_rows=64)
    g = torch.Generator(device=d).manual_seed(0)
    qkv = torch.randn((b.total, 8 * HD), generator=g, device=d).to(torch.bfloat16)
    one = torch.ones(HD, dtype=torch.bfloat16, device=d)
    cos, sin = torch.randn((64, 64), generator=g, device=d), torch.randn((64, 64), generator=g, device=d)
    cache = ref.random_cache(b.blocks, 2, 1, d)
    q_out = torch.empty((b.total, 4 * HD), dtype=torch.bfloat16, device=d)
    states = []
    for _ in range(3):
        ck.qk_norm_rope_kv_append_kv8(desc, qkv, one, one, cos, sin, i32(b.positions), i32(b.slots), *cache, q_out)
        states.append([t.clone() for t in cache])
    for a, c in zip(states[0], states[2]):
        assert torch.equal(a, c)


# ---- attention -------------------------------------------------------------------------------

def attn_case(q_lens, ctxs, nh, nkv, gated=False, window=0, sinks=0, seed=0, scale=1.5, exps=(-7, -4), edit=None,
              tail=0, max_q=None, max_ctx=None):
    d = dev()
    b = ref.batch(q_lens, ctxs, seed)
    g = torch.Generator(device=d).manual_seed(seed)
    T = b.total
    q = (torch.randn((T + tail, nh * HD), generator=g, device=d) * scale).to(torch.bfloat16)
    gate = torch.randn((T + tail, nh * HD), generator=g, device=d).to(torch.bfloat16) if gated else None
    kc, vc, ks, vs = ref.random_cache(b.blocks, nkv, seed + 1, d, exps)
    ref.poison_unused(b, kc, vc, ks, vs)
    if edit:
        edit(b, q, kc, vc, ks, vs)
    desc = make_desc(b, nh, nkv, gated, max_q=max_q, max_ctx=max_ctx)
    desc.total_q = T + tail
    out = torch.full((T + tail, nh * HD), 7.25, dtype=torch.bfloat16, device=d)
    ck.paged_attention_verify_kv8(desc, q, kc, vc, ks, vs, table_of(b), i32(b.cu), i32(ctxs), gate, out, window, sinks)
    torch.cuda.synchronize()
    want, pv, sb = ref.attention(q[:T], kc, vc, ks, vs, b.tables, q_lens, ctxs, nkv,
                                 gate[:T] if gated else None, window, sinks)
    ref.assert_attention(out[:T], want, pv, sb, max(1, max(ctxs)))
    assert (out[T:] == 7.25).all(), "rows behind the last sequence were written"
    return out


@pytest.mark.parametrize("nh,nkv", [(16, 8), (32, 8), (16, 2), (8, 1), (8, 8), (24, 4), (40, 8), (6, 3), (12, 12),
                                    (11, 11), (17, 17), (64, 2), (128, 2)])
def test_attention_decode_heads(nh, nkv):
    attn_case([1, 1, 2, 3], [1, 17, 300, 1025], nh, nkv, seed=nh)


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 13, 16, 17, 31, 33, 64, 100, 129, 300])
def test_attention_row_counts(rows):
    attn_case([rows, max(1, rows // 2), rows], [rows, rows + 15, rows + 777], 8, 2, seed=rows)


@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 2047, 2048, 2049, 9000])
def test_attention_contexts(ctx):
    attn_case([1, min(ctx, 3)], [ctx, ctx], 16, 8, seed=ctx)
    attn_case([min(ctx, 70)], [ctx], 8, 2, seed=ctx)


def test_attention_many_ragged_sequences():
    import random
    rnd = random.Random(7)
    q = [rnd.randint(1, 4) for _ in range(75)]
    attn_case(q, [n + rnd.randint(0, 900) for n in q], 32, 8, seed=8, gated=True)


@pytest.mark.parametrize("seqs,rows,nh,nkv", [(2, 4, 32, 8), (3, 5, 16, 8), (8, 1, 16, 2), (8, 3, 16, 2), (12, 4, 32, 8),
                                              (20, 1, 8, 1), (1, 8, 32, 8), (1, 40, 8, 8), (2, 20, 8, 4), (30, 9, 32, 8)])
def test_attention_sequence_counts(seqs, rows, nh, nkv):
    """From one sequence over all SMs to a few SMs for each: the shares of a row meet in every way."""
    attn_case([rows - (i % 2 and rows > 1) for i in range(seqs)], [2900 - 97 * i for i in range(seqs)], nh, nkv, seed=seqs)


def test_attention_more_sequences_than_one_launch_indexes():
    attn_case([1] * 5000, [1 + (i * 7) % 40 for i in range(5000)], 2, 2, seed=9)


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_attention_gate(rows):
    attn_case([rows, rows], [rows + 30, rows + 500], 16, 2, gated=True, seed=rows)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 33, 100, 128, 129, 1000, 10 ** 9])
@pytest.mark.parametrize("sinks", [0, 1, 16, 33, 5000])
def test_window(window, sinks):
    attn_case([1, 3, 2, 4], [1, 50, 257, 1203], 8, 2, window=window, sinks=sinks, seed=window % 97 + sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 4), (128, 0), (129, 17), (300, 130), (5000, 4)])
def test_window_prompts(window, sinks):
    attn_case([400, 130], [400, 900], 8, 2, window=window, sinks=sinks, seed=window + sinks)
    attn_case([300], [1500], 16, 2, window=window, sinks=sinks, seed=window + sinks, gated=True)


def test_rows_that_see_nothing():
    """Contexts shorter than the rows: rows at negative positions, sequences without context or
    rows between others; their outputs are zeros, and nothing else is disturbed."""
    out = attn_case([3, 2, 0, 5, 1], [1, 0, 100, 3, 40], 8, 2, seed=1, tail=2)
    assert (out[:2] == 0).all() and (out[3:5] == 0).all() and (out[5:7] == 0).all()
    attn_case([90, 80, 0], [50, 0, 300], 8, 2, seed=2, tail=3)
    attn_case([0, 0], [0, 30], 8, 2, seed=3, tail=4)
    attn_case([3, 2, 70], [2, 1, 60], 8, 2, seed=4, tail=2, window=5, sinks=1)


@pytest.mark.parametrize("rows", [2, 150])
def test_invalid_block_ids_read_as_zeros(rows):
    def edit(b, q, kc, vc, ks, vs):
        b.tables[0][3], b.tables[1][0], b.tables[1][-1] = -1, b.blocks, 2 ** 31 - 1
        b.tables[0][5] = -2 ** 31
    attn_case([rows, rows], [rows + 300, rows + 65], 8, 2, seed=rows, edit=edit)


@pytest.mark.parametrize("rows", [2, 12, 150])
def test_pages_outside_the_windows_are_not_looked_at(rows):
    """A serving loop frees pages that have left every row's window: their table entries may be
    anything, another owner's page or one of NaN codes and scales, and no bit changes."""
    d, nh, nkv, window, sinks, ctx = dev(), 16, 2, 300, 20, 2500
    b = ref.batch([rows, 1], [ctx, ctx - 900], rows)
    g = torch.Generator(device=d).manual_seed(rows)
    q = torch.randn((b.total, nh * HD), generator=g, device=d).to(torch.bfloat16)
    kc, vc, ks, vs = ref.random_cache(b.blocks + 1, nkv, 3, d)
    for t, bad in ((kc, 0x7F), (vc, 0xFF), (ks, math.nan), (vs, math.nan)):
        t[b.blocks] = bad
    desc = make_desc(b, nh, nkv)
    desc.num_blocks = b.blocks + 1
    table = table_of(b)
    outs = []
    for freed in (False, True):
        if freed:
            for i, (n, c) in enumerate(zip(b.q_lens, b.ctxs)):
                for pg in range(-(-sinks // PAGE), (c - n - window + 1) // PAGE):
                    table[i, pg] = (b.blocks, -1, 0, 2 ** 31 - 1)[pg % 4]
        out = torch.empty((b.total, nh * HD), dtype=torch.bfloat16, device=d)
        ck.paged_attention_verify_kv8(desc, q, kc, vc, ks, vs, table, i32(b.cu), i32(b.ctxs), None, out, window, sinks)
        outs.append(out)
    assert outs[0].isfinite().all() and torch.equal(*outs)


@pytest.mark.parametrize("rows", [3, 100])
def test_a_nan_query_stays_in_its_row(rows):
    """NaN in one row and head of q: that output is NaN, every other one is as without it."""
    d, nh, nkv = dev(), 8, 2
    b = ref.batch([rows, rows], [700, rows + 40], rows)
    g = torch.Generator(device=d).manual_seed(rows)
    q = torch.randn((b.total, nh * HD), generator=g, device=d).to(torch.bfloat16)
    cache = ref.random_cache(b.blocks, nkv, 5, d)
    desc, outs = make_desc(b, nh, nkv), []
    for bad in (False, True):
        if bad:
            q[1, 5 * HD + 7] = math.nan
        out = torch.empty((b.total, nh * HD), dtype=torch.bfloat16, device=d)
        ck.paged_attention_verify_kv8(desc, q, *cache, table_of(b), i32(b.cu), i32(b.ctxs), None, out)
        outs.append(out)
    assert outs[1][1, 5 * HD:6 * HD].isnan().all()
    outs[1][1, 5 * HD:6 * HD] = outs[0][1, 5 * HD:6 * HD]
    # a NaN score changes the moment at which its group's reference rises, not the values beyond rounding:
    # two orders of the same sum differ by less than a bf16 unit of the largest output
    diff = (outs[0].float() - outs[1].float()).abs().max()
    assert diff <= outs[0].float().abs().max() * 2.0 ** -7


@pytest.mark.parametrize("rows", [1, 50])
def test_sequences_may_share_pages(rows):
    """A common prefix held once: the same page ids in several tables."""
    d, nh, nkv, shared = dev(), 16, 8, 20
    b = ref.batch([rows] * 3, [shared * PAGE + rows + n for n in (0, 40, 700)], rows)
    for t in b.tables[1:]:
        t[:shared] = b.tables[0][:shared]
    g = torch.Generator(device=d).manual_seed(rows)
    q = torch.randn((b.total, nh * HD), generator=g, device=d).to(torch.bfloat16)
    cache = ref.random_cache(b.blocks, nkv, 6, d)
    out = torch.empty((b.total, nh * HD), dtype=torch.bfloat16, device=d)
    ck.paged_attention_verify_kv8(make_desc(b, nh, nkv), q, *cache, table_of(b), i32(b.cu), i32(b.ctxs), None, out)
    want, pv, sb = ref.attention(q, *cache, b.tables, b.q_lens, b.ctxs, nkv)
    ref.assert_attention(out, want, pv, sb, max(b.ctxs))


@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("what", ["wide", "zero", "odd", "huge"])
def test_scales(rows, what):
    """Scales far apart between pages, zero scales, scales that are no powers of two."""
    def edit(b, q, kc, vc, ks, vs):
        g = torch.Generator(device=ks.device).manual_seed(3)
        own = torch.tensor([p for t in b.tables for p in t], device=ks.device)
        n = (len(own), ks.shape[1])
        if what == "wide":
            vs[own] = torch.pow(2.0, torch.randint(-60, 60, n, generator=g, device=ks.device).float())
            ks[own] = torch.pow(2.0, torch.randint(-14, -6, n, generator=g, device=ks.device).float())
        elif what == "zero":
            vs[own[::2]] = 0.0
            ks[own[1::2]] = 0.0
            vs[b.tables[0]] = 0.0
        elif what == "odd":
            vs[own] = torch.rand(n, generator=g, device=ks.device) * 0.01 + 1e-4
            ks[own] = torch.rand(n, generator=g, device=ks.device) * 0.01 + 1e-4
        else:
            vs[own] = 2.0 ** 100
            ks[own] = 2.0 ** -120
    attn_case([rows, rows], [rows + 300, rows + 65], 8, 2, seed=rows, edit=edit)


@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("mag", [0.0, 1e-30, 30.0, 1e4, 1e20])
def test_query_magnitudes(rows, mag):
    attn_case([rows, rows], [rows + 300, rows + 65], 8, 2, seed=rows, scale=mag)


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("where", ["first", "last"])
def test_one_dominant_key_keeps_the_tail(rows, where):
    """One key's probability is 2^16 times each of thousands of others, which together weigh as
    much: small probabilities must not be flushed."""
    def edit(b, q, kc, vc, ks, vs):
        kc.zero_()
        q.fill_(1.0)
        at = 0 if where == "first" else b.ctxs[0] - rows
        # q . k / sqrt(128) = 16 ln 2: 128 elements of 16 ln 2 / sqrt(128) = 0.980...
        ks[b.tables[0]] = 2.0 ** -6
        kc[b.tables[0][at // PAGE], at % PAGE] = torch.full((2, HD), 0.98 * 64, device=kc.device).to(ref.F8).view(
            torch.uint8)
        vs[b.tables[0]] = 2.0 ** -6
        t = torch.tensor(b.tables[0], device=vc.device)
        vc[t] = torch.full((2, HD), 64.0, device=vc.device).to(ref.F8).view(torch.uint8)
        vc[b.tables[0][at // PAGE], at % PAGE] = torch.full((2, HD), -64.0, device=vc.device).to(ref.F8).view(torch.uint8)
    attn_case([rows], [40000], 8, 2, seed=1, edit=edit)


@pytest.mark.parametrize("rows", [2, 150])
def test_bounds_larger_than_the_batch(rows):
    attn_case([rows, 1], [rows + 40, 33], 8, 2, seed=rows, max_q=4 * rows, max_ctx=9000)


def test_block_table_wider_than_needed_and_pages_far_apart():
    """A pool whose byte offsets pass 32 bits: pages at its far end."""
    d = dev()
    nkv, nh = 8, 16
    blocks = (1 << 32) // (PAGE * nkv * HD) + 40     # 4 GiB of codes and a little
    kc = torch.zeros((blocks, PAGE, nkv, HD), dtype=torch.uint8, device=d)
    vc = torch.zeros_like(kc)
    ks = torch.full((blocks, nkv), 2.0 ** -6, device=d)
    vs = torch.full((blocks, nkv), 2.0 ** -6, device=d)
    b = ref.batch([2, 150], [100, 400], 1)
    ids = list(range(blocks - 35, blocks))
    b.tables = [ids[:7], ids[7:32]]
    b.blocks, b.max_pages = blocks, 40
    g = torch.Generator(device=d).manual_seed(0)
    for t in b.tables:
        for p in t:
            for c in (kc, vc):
                c[p] = (torch.randn((PAGE, nkv, HD), generator=g, device=d) * 80).to(ref.F8).view(torch.uint8)
    q = torch.randn((b.total, nh * HD), generator=g, device=d).to(torch.bfloat16)
    out = torch.empty_like(q)
    desc = make_desc(b, nh, nkv)
    ck.paged_attention_verify_kv8(desc, q, kc, vc, ks, vs, table_of(b), i32(b.cu), i32(b.ctxs), None, out)
    want, pv, sb = ref.attention(q, kc, vc, ks, vs, b.tables, b.q_lens, b.ctxs, nkv)
    ref.assert_attention(out, want, pv, sb, 400)
    # and an append there
    qkv = torch.randn((b.total, (nh + 2 * nkv) * HD), generator=g, device=d).to(torch.bfloat16)
    one = torch.ones(HD, dtype=torch.bfloat16, device=d)
    cos, sin = torch.ones((400, 64), device=d), torch.zeros((400, 64), device=d)
    desc = make_desc(b, nh, nkv, rope_rows=400)
    tail = slice(blocks - 40, blocks)
    before = [t[tail].clone() for t in (kc, vc, ks, vs)]
    ck.qk_norm_rope_kv_append_kv8(desc, qkv, one, one, cos, sin, i32(b.positions), i32(b.slots), kc, vc, ks, vs, out)
    v = qkv[:, (nh + nkv) * HD:].double().view(b.total, nkv, HD)
    check_store(v, [s - (blocks - 40) * PAGE for s in b.slots], before[1], before[3], vc[tail], vs[tail])


# ---- the two together, streams, graphs ------------------------------------------------------

@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_append_then_attention_over_steps(window, sinks):
    """A prompt, then verify steps with rejected rows, on the cache as the operators leave it:
    each step's output against the exact attention over the cache's values, and the cache's
    values within half an e4m3 step of the rows that were appended."""
    d = dev()
    nh, nkv = 8, 2
    g = torch.Generator(device=d).manual_seed(11)
    b = ref.batch([1, 1], [200, 200], 3)
    cache = ref.random_cache(b.blocks, nkv, 2, d)
    cos, sin = torch.randn((256, 64), generator=g, device=d), torch.randn((256, 64), generator=g, device=d)
    one = torch.ones(HD, dtype=torch.bfloat16, device=d)
    lens = [0, 0]
    rows = {0: [], 1: []}
    for step, n in enumerate([(70, 37), (3, 2), (3, 3), (1, 4), (2, 1)]):
        b.q_lens, b.ctxs = list(n), [lens[i] + n[i] for i in (0, 1)]
        T = b.total
        qkv = torch.randn((T, (nh + 2 * nkv) * HD), generator=g, device=d).to(torch.bfloat16)
        q = torch.empty((T, nh * HD), dtype=torch.bfloat16, device=d)
        out = torch.empty_like(q)
        desc = make_desc(b, nh, nkv, rope_rows=256)
        ck.qk_norm_rope_kv_append_kv8(desc, qkv, one, one, cos, sin, i32(b.positions), i32(b.slots), *cache, q)
        ck.paged_attention_verify_kv8(desc, q, *cache, table_of(b), i32(b.cu), i32(b.ctxs), None, out, window, sinks)
        want, pv, sb = ref.attention(q, *cache, b.tables, b.q_lens, b.ctxs, nkv, None, window, sinks)
        ref.assert_attention(out, want, pv, sb, 256)
        v = qkv[:, -nkv * HD:].double().view(T, nkv, HD)
        for i in (0, 1):
            start = sum(n[:i])
            rows[i] = rows[i][:lens[i]] + [v[start + j] for j in range(n[i])]
            exact = torch.stack(rows[i])
            at = torch.tensor([b.tables[i][p // PAGE] * PAGE + p % PAGE for p in range(b.ctxs[i])], device=d)
            got = (ref.values(cache[1]) * cache[3].double()[:, None, :, None]).view(-1, nkv, HD)[at]
            sc = cache[3].double()[at // PAGE][:, :, None]
            # one rounding, and one more where the page's scale grew over a value: half a step
            # each; subnormal steps are 2^-9 of the scale
            step_size = ref.e4m3_step(exact / sc) * sc
            assert ((got - exact).abs() <= step_size * (1 + 2.0 ** -8)).all()
            lens[i] = b.ctxs[i] - (1 if step in (1, 2) and n[i] > 1 else 0)  # the last row is rejected


def test_side_stream_and_captured_graphs():
    """Two captured graphs (append + attention each) with workspaces of their own, replayed on
    two streams at once with other inputs and shorter contexts than they were captured with."""
    d = dev()
    nh, nkv = 16, 4
    graphs = []
    for n in (0, 1):
        b = ref.batch([2, 3, 2], [700, 900, 40 + n], 5 + n)
        g = torch.Generator(device=d).manual_seed(n)
        cache = ref.random_cache(b.blocks, nkv, n, d)
        T = b.total
        st = dict(b=b, cache=cache, qkv=torch.randn((T, (nh + 2 * nkv) * HD), generator=g, device=d).to(torch.bfloat16),
                  q=torch.empty((T, nh * HD), dtype=torch.bfloat16, device=d),
                  out=torch.empty((T, nh * HD), dtype=torch.bfloat16, device=d),
                  pos=i32(b.positions), slots=i32(b.slots), ctx=i32(b.ctxs), cu=i32(b.cu), table=table_of(b))
        cos, sin = torch.randn((1000, 64), generator=g, device=d), torch.randn((1000, 64), generator=g, device=d)
        one = torch.ones(HD, dtype=torch.bfloat16, device=d)
        desc = make_desc(b, nh, nkv, rope_rows=1000)
        ws = torch.empty(ck.paged_attention_kv8_workspace_bytes(desc), dtype=torch.uint8, device=d)
        st["hold"] = (cos, sin, one, ws, desc)

        def body(st=st, cos=cos, sin=sin, one=one, desc=desc, ws=ws):
            ck.qk_norm_rope_kv_append_kv8(desc, st["qkv"], one, one, cos, sin, st["pos"], st["slots"], *st["cache"],
                                          st["q"])
            ck.paged_attention_verify_kv8(desc, st["q"], *st["cache"], st["table"], st["cu"], st["ctx"], None,
                                          st["out"], workspace=ws)
        side = torch.cuda.Stream(device=d)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        allocs = abi.alloc_count()
        with torch.cuda.graph(graph):
            body()
        assert abi.alloc_count() == allocs
        graphs.append((graph, st, torch.cuda.Stream(device=d)))
    for ctxs in ([700, 900, 40], [650, 333, 17], [20, 901 - 1, 38]):
        for graph, st, stream in graphs:
            b = st["b"]
            b.ctxs = list(ctxs)
            st["qkv"].copy_(torch.randn(st["qkv"].shape, device=d))
            st["pos"].copy_(i32(b.positions))
            st["slots"].copy_(i32(b.slots))
            st["ctx"].copy_(i32(b.ctxs))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, st, stream in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, st, stream in graphs:
            b = st["b"]
            want, pv, sb = ref.attention(st["q"], *st["cache"], b.tables, b.q_lens, b.ctxs, nkv)
            ref.assert_attention(st["out"], want, pv, sb, 1000)
    for graph, _, _ in graphs:
        graph.reset()


def test_two_runs_agree_bit_for_bit():
    a = attn_case([3] * 9, [1000 + 37 * i for i in range(9)], 32, 8, seed=4)
    c = attn_case([3] * 9, [1000 + 37 * i for i in range(9)], 32, 8, seed=4)
    assert torch.equal(a, c)


def test_workspace_is_checked_and_wrappers_refuse_bad_tensors():
    d = dev()
    b = ref.batch([2, 2], [3000, 3000], 0)
    kc, vc, ks, vs = ref.random_cache(b.blocks, 8, 0, d)
    q = torch.zeros((4, 32 * HD), dtype=torch.bfloat16, device=d)
    out = torch.empty_like(q)
    desc = make_desc(b, 32, 8)
    args = [desc, q, kc, vc, ks, vs, table_of(b), i32(b.cu), i32(b.ctxs), None, out]
    need = ck.paged_attention_kv8_workspace_bytes(desc)
    with pytest.raises(RuntimeError, match="workspace"):
        ck.paged_attention_verify_kv8(*args, workspace=torch.empty(need - 1, dtype=torch.uint8, device=d))
    with pytest.raises(RuntimeError, match="workspace"):
        ck.paged_attention_verify_kv8(*args, workspace=torch.empty(need + 16, dtype=torch.uint8, device=d)[1:])
    with pytest.raises(ValueError, match="window"):
        ck.paged_attention_verify_kv8(*args, window=-1)

    def swapped(i, t):
        a = list(args)
        a[i] = t
        return a
    for i, t in [(1, q.float()), (1, q[:3]), (1, q.cpu()), (2, kc[:-1]), (2, kc.view(torch.int8)), (4, ks.half()),
                 (4, ks.t().contiguous().t()), (6, i32([[0]])), (7, i32([0, 2])), (8, i32([1])),
                 (8, torch.tensor([3000, 3000], device=d)), (10, out[:, ::2]), (10, out[:1])]:
        with pytest.raises(ValueError):
            ck.paged_attention_verify_kv8(*swapped(i, t))
    hold = torch.empty(kc.numel() + 16, dtype=torch.uint8, device=d)
    with pytest.raises(RuntimeError, match="16-byte"):
        ck.paged_attention_verify_kv8(*swapped(2, hold[1:1 + kc.numel()]))
