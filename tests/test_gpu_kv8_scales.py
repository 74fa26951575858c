"""8-bit cache attention where a batch's V scales differ by many powers of two: a row's result keeps
its accuracy whatever the scales of pages that it does not see, or gives no weight."""
import math

import pytest
import torch

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests import _kv8 as ref
from tests._gpu import dev
from tests._kv8 import HD, PAGE
from tests.test_gpu_kv8 import i32, make_desc, table_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    abi.init()
    yield


def restated(q, kc, vc, ks, vs, b, nkv, window, sinks):
    """float64, row by row (all [T, nh, 128]): outputs, sum p |v|, the same over the keys with p below 2^-118
    and, per row and head, the number of keys seen times 448 times the largest p * vs, and the largest
    sum |q k| / sqrt(128)."""
    T, nh = b.total, q.shape[1] // HD
    g, dv = nh // nkv, q.device
    out = torch.zeros((T, nh, HD), dtype=torch.float64, device=dv)
    pv, low, wt, sb = (torch.zeros_like(out) for _ in range(4))
    for i, (n, ctx) in enumerate(zip(b.q_lens, b.ctxs)):
        at = torch.tensor(b.tables[i][:-(-ctx // PAGE)], device=dv)
        k = (ref.values(kc[at]) * ks[at].double()[:, None, :, None]).flatten(0, 1)[:ctx]
        v = (ref.values(vc[at]) * vs[at].double()[:, None, :, None]).flatten(0, 1)[:ctx]
        scale = vs[at].double().repeat_interleave(PAGE, 0)[:ctx]
        for j in range(n):
            p, row = ctx - n + j, b.cu[i] + j
            key = torch.arange(p + 1, device=dv)
            if window:
                key = key[(key > p - window) | (key < sinks)]
            for h in range(nh):
                x = q[row, h * HD:(h + 1) * HD].double()
                kk, vv, sc = k[key, h // g], v[key, h // g], scale[key, h // g]
                w = torch.softmax(kk @ x / math.sqrt(HD), 0)
                out[row, h], pv[row, h] = w @ vv, w @ vv.abs()
                low[row, h] = torch.where(w < 2.0 ** -118, w, 0.0) @ vv.abs()
                wt[row, h] = len(key) * 448 * (w * sc).max()
                sb[row, h] = (kk.abs() @ x.abs()).max() / math.sqrt(HD)
    return out, pv, low, wt, sb


def check(got, want, n_keys, ties=False):
    """|got - out| <= 2^-8 |out|              the output's rounding to bf16
                   + sum p|v| * (2^-11        weights rounded to f16
                                 + 2 e        scores off by e (as tests/_kv8.py derives it); 0 where all
                                              keys are the same: their scores are equal whatever e
                                 + 2^-18      exponentials, logarithms of the scales, division
                                 + n 2^-24)   the fp32 sums
                   + n 448 max(p vs) 2^-34    a weight is held as 2^9 of the row's largest p * vs, or more
                                              (the reference starts at or below it and is a lag behind):
                                              f16 steps of 2^-24 below the normal range are off by 2^-25
                   + sum over p < 2^-118 of p |v|   partials join by l 2^(m - M), 0 in fp32 below 2^-126, and a
                                              partial's m is up to 7.75 below its largest score
                   + 2^-126                   results below the normal range."""
    out, pv, low, wt, sb = want
    e = torch.zeros_like(sb) if ties else (260 * 2.0 ** -24 * sb).clamp(max=1)
    tol = (2.0 ** -8 * out.abs() + pv * (2.0 ** -11 + 2 * e + 2.0 ** -18 + n_keys * 2.0 ** -24) + wt * 2.0 ** -34 +
           low + 2.0 ** -126)
    err = (got.double().view(out.shape) - out).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, in rows "
                           f"{sorted(set(bad.nonzero()[:, 0].tolist()))[:8]}; first "
                           f"{got.view(out.shape)[bad][0].item():.4g} for {out[bad][0].item():.4g}")


def run(q_lens, ctxs, nh, nkv, exponents, window=0, sinks=0, seed=0, edit=None, ties=False, k_exp=-7):
    """exponents(page index, pages of the sequence) -> log2 of the page's V scale (None: a scale of 0)."""
    d = dev()
    b = ref.batch(q_lens, ctxs, seed)
    g = torch.Generator(device=d).manual_seed(seed)
    q = (torch.randn((b.total, nh * HD), generator=g, device=d) * 1.5).to(torch.bfloat16)
    kc, vc, ks, vs = ref.random_cache(b.blocks, nkv, seed + 1, d)
    ks.fill_(2.0 ** k_exp)
    ref.poison_unused(b, kc, vc, ks, vs)
    for t in b.tables:
        for i, page in enumerate(t):
            e = exponents(i, len(t))
            vs[page] = 0.0 if e is None else 2.0 ** e
    if edit:
        edit(b, q, kc, vc, ks, vs)
    out = torch.full((b.total, nh * HD), 7.25, dtype=torch.bfloat16, device=d)
    ck.paged_attention_verify_kv8(make_desc(b, nh, nkv), q, kc, vc, ks, vs, table_of(b), i32(b.cu), i32(ctxs), None, out,
                                  window, sinks)
    torch.cuda.synchronize()
    check(out, restated(q, kc, vc, ks, vs, b, nkv, window, sinks), max(ctxs), ties)


# rows per sequence: on the token kernel (a CTA per sequence, shares of all pages, two row tiles) and,
# past 32 per KV head, on the chunk kernel (one and two tiles, split and not)
SHAPES = [([4, 3], [33, 50], 4, 2), ([4], [2050], 4, 2), ([6, 5], [700, 21], 8, 2), ([40], [40], 2, 2),
          ([70, 33], [90, 400], 2, 1)]


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
@pytest.mark.parametrize("step", [3, 12, 40])
def test_later_pages_of_larger_scales(q_lens, ctxs, nh, nkv, step):
    """Each page's V scale 2^step times that of the one before, up to 2^80: rows that end before the
    last pages must not lose bits to them."""
    run(q_lens, ctxs, nh, nkv, lambda i, n: max(-100, 80 - step * (n - 1 - i)), seed=step)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
@pytest.mark.parametrize("step,window,sinks", [(3, 17, 0), (40, 16, 0), (25, 5, 2), (40, 1, 0)])
def test_pages_behind_the_window_of_larger_scales(q_lens, ctxs, nh, nkv, step, window, sinks):
    """The other way round, through a window: rows that have left the first pages."""
    run(q_lens, ctxs, nh, nkv, lambda i, n: max(-100, min(80, -60 + step * (n - 1 - i))), window, sinks, seed=step)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
def test_seen_pages_without_weight(q_lens, ctxs, nh, nkv):
    """A page whose keys score 2^-100 of the others, with values 2^60 times theirs."""
    def edit(b, q, kc, vc, ks, vs):
        q.abs_()
        for t in b.tables:
            kc[t[0]] = torch.tensor(-448.0).to(ref.F8).view(torch.uint8).item()
            ks[t[0]] = 2.0 ** -6
    run(q_lens, ctxs, nh, nkv, lambda i, n: 40 if i == 0 else -20, seed=3, edit=edit)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
def test_scales_of_zero(q_lens, ctxs, nh, nkv):
    """Pages of zero V scales (no value, but weight), and of zero K scales (scores of zero)."""
    def edit(b, q, kc, vc, ks, vs):
        for t in b.tables:
            ks[t[1::3]] = 0.0
    run(q_lens, ctxs, nh, nkv, lambda i, n: None if i % 2 else -7, seed=4, edit=edit)
    run(q_lens, ctxs, nh, nkv, lambda i, n: None, seed=5)
    run(q_lens, ctxs, nh, nkv, lambda i, n: -30 if i == n - 1 else None, seed=6, edit=edit)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
@pytest.mark.parametrize("e", [-126, -110, 90, 110, 118])
def test_ends_of_the_scales_range(q_lens, ctxs, nh, nkv, e):
    run(q_lens, ctxs, nh, nkv, lambda i, n: e, seed=7)
    run(q_lens, ctxs, nh, nkv, lambda i, n: e if i % 2 else (-126 if e > 0 else -100), seed=8)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_equal_scores_far_from_zero(q_lens, ctxs, nh, nkv, sign):
    """Every key the same, with scores of +-2^32: the weights are equal, whatever the scales of V."""
    def edit(b, q, kc, vc, ks, vs):
        kc[:] = torch.tensor(448.0).to(ref.F8).view(torch.uint8).item()
        q.fill_(sign * 4096.0)
    run(q_lens, ctxs, nh, nkv, lambda i, n: (-7, 0, -3, 4)[i % 4], seed=9, edit=edit, ties=True, k_exp=8)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES)
def test_scales_that_are_no_powers_of_two(q_lens, ctxs, nh, nkv):
    def edit(b, q, kc, vc, ks, vs):
        for i, t in enumerate(b.tables):
            for j, page in enumerate(t):
                vs[page] *= 1.0 + 0.37 * ((5 * i + 3 * j) % 7) / 7
                ks[page] *= 1.0 + 0.41 * ((3 * i + 5 * j) % 5) / 5
    run(q_lens, ctxs, nh, nkv, lambda i, n: -7 + 9 * (i % 3), seed=10, edit=edit)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv", SHAPES + [([2], [9000], 32, 8), ([1] * 3, [4000, 3000, 5000], 64, 4),
                                                         ([12], [9000], 32, 8)])
def test_a_nan_query_gives_nan(q_lens, ctxs, nh, nkv):
    """Also where its row is put together from partials."""
    d = dev()
    b = ref.batch(q_lens, ctxs, 11)
    q = torch.randn((b.total, nh * HD), generator=torch.Generator(device=d).manual_seed(11), device=d).to(torch.bfloat16)
    q[0, HD + 5] = math.nan
    out = torch.empty_like(q)
    ck.paged_attention_verify_kv8(make_desc(b, nh, nkv), q, *ref.random_cache(b.blocks, nkv, 12, d), table_of(b),
                                  i32(b.cu), i32(ctxs), None, out)
    bad = out.isnan().view(b.total, nh, HD)
    assert bad[0, 1].all() and int(bad.sum()) == HD


@pytest.mark.parametrize("tail", [0, 3000])
def test_more_splits_than_lanes(tail):
    """One sequence of 40 rows over many keys takes 64 splits, with rows behind it that are not its own."""
    d, nh, nkv = dev(), 4, 1
    b = ref.batch([10], [5000], 13)
    g = torch.Generator(device=d).manual_seed(13)
    q = (torch.randn((b.total + tail, nh * HD), generator=g, device=d) * 1.5).to(torch.bfloat16)
    cache = ref.random_cache(b.blocks, nkv, 14, d)
    desc = make_desc(b, nh, nkv, max_ctx=5000 * 16)  # a bound: more blocks are planned than there are
    desc.total_q = b.total + tail
    out = torch.full(q.shape, 7.25, dtype=torch.bfloat16, device=d)
    ck.paged_attention_verify_kv8(desc, q, *cache, table_of(b), i32(b.cu), i32(b.ctxs), None, out)
    assert (out[b.total:] == 7.25).all()
    check(out[:b.total], restated(q[:b.total], *cache, b, nkv, 0, 0), 5000)
