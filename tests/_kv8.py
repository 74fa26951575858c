"""The 8-bit KV cache operators restated in float64, and the inputs of their tests.

Layout: codes [num_blocks, 16, n_kv, 128] e4m3 bytes, scales [num_blocks, n_kv] fp32."""
from __future__ import annotations

import math
import random
from dataclasses import dataclass

import torch

HD, PAGE = 128, 16
F8 = torch.float8_e4m3fn


def values(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(F8).double()


def e4m3_step(y: torch.Tensor) -> torch.Tensor:
    """Spacing of e4m3 values at |y| (3 mantissa bits, least exponent -6)."""
    _, top = torch.frexp(y.double())
    top = torch.where(y == 0, torch.full_like(top, -5), top)
    return torch.ldexp(torch.ones_like(y, dtype=torch.float64), (top - 1).clamp(min=-6) - 3)


def scale_exponent(amax: torch.Tensor) -> torch.Tensor:
    """Least e with amax <= 448 * 2^e; 0 where amax is 0."""
    m, e = torch.frexp(amax.double())
    return torch.where(amax > 0, e - 9 + (m > 0.875).int(), torch.zeros_like(e))


def rms_rope(x, w, cos, sin, rot, eps, add_one):
    """x [T, heads, 128] float64 -> RMSNorm * w, then the rotation of the first rot dims."""
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.double() + (1.0 if add_one else 0.0))
    h = rot // 2
    a, b = x[..., :h], x[..., h:rot]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., rot:]], -1)


def store(x, slots, codes, scale):
    """(codes as float64 values, scales) after writing the rows x [T, kv, 128] (float64)."""
    val, scale = values(codes).clone(), scale.double().clone()
    blocks = codes.shape[0]
    pages: dict[int, dict[int, int]] = {}
    for r, s in enumerate(slots):
        if 0 <= s < blocks * PAGE:
            pages.setdefault(s // PAGE, {})[s % PAGE] = r  # the last row of a slot stands
    for pg, put in pages.items():
        lo = min(put)
        new = torch.nan_to_num(x[list(put.values())], nan=0.0, posinf=math.inf, neginf=-math.inf)
        kept = val[pg, :lo] * scale[pg][None, :, None]
        fin = torch.where(new.isfinite(), new, torch.zeros_like(new))
        amax = torch.cat([kept, fin]).abs().amax((0, 2))
        e = scale_exponent(amax)

        def q(v):
            y = torch.ldexp(v, -e[None, :, None]).clamp(-448, 448)
            st = e4m3_step(y)
            return torch.round(y / st) * st
        val[pg, :lo] = q(kept)
        val[pg, list(put)] = q(new)
        scale[pg] = torch.ldexp(torch.ones_like(amax), e)
    return val, scale


def attention(q, codes_k, codes_v, ks, vs, tables, q_lens, ctxs, nkv, gate=None, window=0, sinks=0):
    """float64 outputs [T, nh * 128], and the bound's parts: sum p |v| (same shape), and of each
    row and head [T, nh] the largest sum |q k| / sqrt(128), the largest max|q| sum |k| / sqrt(128), and the number of keys times the
    largest value its V scales allow (448 * scale)."""
    T, nh = q.shape[0], q.shape[1] // HD
    g, dev, blocks = nh // nkv, q.device, codes_k.shape[0]
    out = torch.zeros((T, nh, HD), dtype=torch.float64, device=dev)
    pv = torch.zeros_like(out)
    sb = torch.zeros((T, nh), dtype=torch.float64, device=dev)
    vt, qk = torch.zeros_like(sb), torch.zeros_like(sb)
    r0 = 0
    for b, (n, ctx) in enumerate(zip(q_lens, ctxs)):
        rows, r0 = slice(r0, r0 + n), r0 + n
        if n == 0 or ctx <= 0:
            continue
        pages = torch.tensor(tables[b][:-(-ctx // PAGE)], device=dev)
        ok = (pages >= 0) & (pages < blocks)
        at = torch.where(ok, pages, 0)

        def gather(codes, sc):
            v = values(codes[at]) * sc[at].double()[:, None, :, None]
            v = torch.where(ok[:, None, None, None], v, torch.zeros_like(v))
            return v.flatten(0, 1)[:ctx].transpose(0, 1)                 # [kv, ctx, 128]
        k, v = gather(codes_k, ks), gather(codes_v, vs)
        top = torch.where(ok[:, None], vs[at].double(), 0.0).amax(0)
        vt[rows] = (ctx * 448.0 * top).repeat_interleave(g)
        pos = torch.arange(ctx - n, ctx, device=dev)[:, None]
        key = torch.arange(ctx, device=dev)[None]
        seen = key <= pos
        if window:
            seen &= (key > pos - window) | (key < sinks)
        qq = q[rows].double().view(n, nkv, g, HD)
        s = torch.einsum("nkgd,kcd->nkgc", qq, k) / math.sqrt(HD)
        sa = torch.einsum("nkgd,kcd->nkgc", qq.abs(), k.abs()) / math.sqrt(HD)
        m4 = seen[:, None, None]
        s = torch.where(m4, s, torch.full_like(s, -math.inf))
        ka = torch.where(m4, k.abs().sum(-1)[None, :, None], torch.zeros_like(sa)).amax(-1) / math.sqrt(HD)
        qk[rows] = (qq.abs().amax(-1) * ka).reshape(n, nh)
        mx = s.amax(-1, keepdim=True)
        p = torch.where(m4, torch.exp(s - torch.where(mx.isfinite(), mx, torch.zeros_like(mx))), torch.zeros_like(s))
        tot = p.sum(-1, keepdim=True)
        p = torch.where(tot > 0, p / tot, torch.zeros_like(p))
        out[rows] = torch.einsum("nkgc,kcd->nkgd", p, v).reshape(n, nh, HD)
        pv[rows] = torch.einsum("nkgc,kcd->nkgd", p, v.abs()).reshape(n, nh, HD)
        sb[rows] = torch.where(m4, sa, torch.zeros_like(sa)).amax(-1).reshape(n, nh)
    if gate is not None:
        sg = torch.sigmoid(gate.double()).view(T, nh, HD)
        out, pv = out * sg, pv * sg
    return out.view(T, nh * HD), pv.view(T, nh * HD), (sb, qk, vt)


def assert_attention(got, ref, pv, sb, max_ctx):
    """|got - ref| <= 2^-8 |ref| (the output's rounding to bf16)
                    + sum p|v| * (2^-11          probabilities rounded to f16
                                  + 2 e          a score off by e moves its probability and the
                                                 sum by e each; e = 260 * 2^-24 * sum|q k| (the
                                                 sums of 128 products each, which the tensor
                                                 cores truncate at 2^-23, and their scaling)
                                                 + 2^-39 * max|q| * sum|k| (a query is held in
                                                 f16 with its largest element at least 2^14: the
                                                 steps of 2^-24 below the normal range)
                                  + 2^-18        exp, division, the gate's sigmoid
                                  + ctx 2^-24    the fp32 sum over the keys)
                    + keys * 448 * scale * 2^-34 a probability p (the largest: at least 1) is held
                                                 as 2^9 p in f16: the steps of 2^-24 below the
                                                 normal range leave it at most 2^-34 off
                    + 2^-126                     results below the normal range."""
    sb, qk, vt = sb
    full = lambda x: x[:, :, None].expand(T, nh, HD).reshape(T, nh * HD)  # noqa: E731
    T, nh = sb.shape
    e = 2 * full(260 * 2.0 ** -24 * sb + 2.0 ** -39 * qk)
    tol = 2.0 ** -8 * ref.abs() + pv * (2.0 ** -11 + e.clamp(max=2) + 2.0 ** -18 + max_ctx * 2.0 ** -24) + 2.0 ** -126
    tol = tol + full(vt) * 2.0 ** -34
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {ref[bad][0].item()}")


@dataclass
class Batch:
    q_lens: list
    ctxs: list
    tables: list
    blocks: int
    max_pages: int

    @property
    def total(self):
        return sum(self.q_lens)

    @property
    def cu(self):
        cu = [0]
        for n in self.q_lens:
            cu.append(cu[-1] + n)
        return cu

    @property
    def positions(self):
        return [p for n, c in zip(self.q_lens, self.ctxs) for p in range(c - n, c)]

    @property
    def slots(self):
        return [t[p // PAGE] * PAGE + p % PAGE for n, c, t in zip(self.q_lens, self.ctxs, self.tables)
                for p in range(c - n, c)]


def batch(q_lens, ctxs, seed=0, spare=5) -> Batch:
    """Each sequence's pages drawn without repetition from a pool with `spare` unused ones."""
    rnd = random.Random(seed)
    need = [max(0, -(-c // PAGE)) for c in ctxs]
    blocks = sum(need) + spare
    perm = list(range(blocks))
    rnd.shuffle(perm)
    tables, at = [], 0
    for n in need:
        tables.append(perm[at:at + n])
        at += n
    return Batch(list(q_lens), list(ctxs), tables, blocks, max(1, max(need)))


def random_cache(blocks, nkv, seed, dev, exps=(-7, -4)):
    """(k codes, v codes, k scales, v scales) of normal values under power-of-two scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn((blocks, PAGE, nkv, HD), generator=g, device=dev) * 80
        out.append(x.clamp(-448, 448).to(F8).view(torch.uint8))
    for _ in range(2):
        out.append(torch.pow(2.0, torch.randint(exps[0], exps[1], (blocks, nkv), generator=g, device=dev).float()))
    return out


def poison_unused(b: Batch, codes_k, codes_v, ks, vs):
    """NaN codes past each context in its last page; NaN codes and scales in unowned pages."""
    owned = {p for t in b.tables for p in t}
    for p in range(b.blocks):
        if p not in owned:
            codes_k[p], codes_v[p] = 0x7F, 0xFF
            ks[p], vs[p] = math.nan, math.nan
    for c, t in zip(b.ctxs, b.tables):
        if c > 0 and c % PAGE:
            codes_k[t[-1], c % PAGE:], codes_v[t[-1], c % PAGE:] = 0xFF, 0x7F
