"""Measured cases of the 8-bit paged KV cache operators.

Three operators over one cache: per layer K and V are e4m3 codes [num_blocks, 16, n_kv, 128]
with one fp32 scale for each page and KV head [num_blocks, n_kv]; an element is code * scale.

  append     the q/k/v projection of the pass's rows -> q (RMSNorm, RoPE, bf16), and K (RMSNorm,
             RoPE) and V quantized into their pages.  A page's scale is the smallest power of
             two 2^e with amax <= 448 * 2^e over what the page then holds: the tokens at
             offsets below the first one written now, and the rows written now.
  attention  softmax(q k^T / sqrt(128)) v for the rows at the end of each context (a single
             token, verify rows, a prompt chunk), causal, from the pages of the block table.
  window     the same with a sliding window: a row at position p sees keys in (p - window, p]
             and the first `sinks` keys.
"""
import math

import torch

own = False

HD = 128   # head dim
PAGE = 16  # tokens per page
F8 = torch.float8_e4m3fn


# ---- cases -------------------------------------------------------------------------------

def _case(name, kind, seqs, rows, ctx, heads, kv_heads, gated=False, rot=HD, window=0, sinks=0):
    c = dict(kind=kind, seqs=seqs, rows=rows, ctx=ctx, heads=heads, kv_heads=kv_heads, gated=gated, rot=rot,
             window=window, sinks=sinks)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one sequence's next token at the head layout of Qwen3-0.6B and 1.7B: launch latency
        _case("append-one", "append", 1, 1, 301, 16, 8),
        # the verify pass of a served batch: 32 sequences, two drafts each, Qwen3-8B heads, 8K contexts
        _case("append-verify", "append", 32, 3, 8236, 32, 8),
        # gated attention with partial rotary (Qwen3.5), ragged verify rows
        _case("append-gated", "append", 24, 5, 2517, 16, 2, gated=True, rot=32),
        # five prompts of odd lengths in one pass
        _case("append-prompt", "append", 5, 1733, 1733, 32, 8),
        # one sequence's next token over a short context: launch latency
        _case("decode-one", "attention", 1, 1, 301, 16, 8),
        # the verify pass of the served batch: every page of 32 contexts of about 8K tokens
        _case("verify-8k", "attention", 32, 3, 8236, 32, 8),
        # one long document: a single row over 128K keys, split over the whole GPU
        _case("decode-long", "attention", 1, 1, 131071, 32, 8),
        # more verify rows than one tensor-core tile holds: 5 rows x 8 heads per KV head, gated
        _case("verify-gated", "attention", 24, 5, 2517, 16, 2, gated=True),
        # two prompts from their first token, one of odd length
        _case("prompt-4k", "attention", 2, 4096, 4096, 32, 8),
        # streaming decode of 64 long conversations through a 4K window with 4 sink tokens
        _case("window-decode", "window", 64, 2, 16391, 32, 8, window=4096, sinks=4),
        # a long prompt through a 1K window
        _case("window-prompt", "window", 1, 8192, 8192, 32, 8, window=1024, sinks=4),
        # a window that is no multiple of a page, one sink, as many KV heads as query heads
        _case("window-odd", "window", 8, 3, 1203, 8, 8, window=100, sinks=1),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "window"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (16, 2), (8, 8), (8, 1), (24, 4), (40, 8), (6, 3), (12, 12)])
    gated = rng.random() < 0.25
    rot = rng.choice([128, 128, 128, 64, 32, 96])
    if rng.random() < 0.3:  # a prompt, or a chunk of one over an existing context
        seqs = rng.randint(1, 4)
        rows = _loguniform(rng, 17, 2048 // seqs)
        ctx = rows + (0 if rng.random() < 0.5 else _loguniform(rng, 1, 3000 // seqs))
    else:                   # single tokens and verify rows
        seqs = _loguniform(rng, 1, 64)
        rows = rng.choice([1, 1, 2, 3, 4, 5, 8, 13])
        ctx = rows + _loguniform(rng, 1, min(65536, 2000000 // (kv_heads * seqs)))
    window = sinks = 0
    if kind == "window":
        window = _loguniform(rng, 1, max(2, ctx))
        sinks = rng.choice([0, 1, 4, 16, 33])
    return _case(None, kind, seqs, rows, ctx, heads, kv_heads, gated, rot if kind == "append" else HD, window, sinks)


def _geometry(case):
    """(rows, context) of each sequence: ragged around the case's sizes, the first one full."""
    out = []
    for i in range(case["seqs"]):
        rows = case["rows"] - (i * 5 % 8) * case["rows"] // 16
        ctx = case["ctx"] if case["ctx"] == case["rows"] else case["ctx"] - (i * 11 % 16) * case["ctx"] // 64
        if case["ctx"] == case["rows"]:
            ctx = rows
        out.append((rows, max(rows, ctx)))
    return out


def _visible(case, rows, ctx):
    """(keys that some row of a sequence sees, pairs of a row and a key that it sees)"""
    first = ctx - rows
    if not case["window"]:
        return ctx, sum(range(first + 1, ctx + 1))
    w, s = case["window"], case["sinks"]
    lo = max(0, first - w + 1)
    keys = ctx - lo + min(s, lo)
    pairs = sum(min(p + 1, w) + min(s, max(0, p + 1 - w)) for p in range(first, ctx))
    return keys, pairs


def work(case):
    geo = _geometry(case)
    h, kv = case["heads"], case["kv_heads"]
    rows = sum(r for r, _ in geo)
    if case["kind"] == "append":
        proj = (h * (2 if case["gated"] else 1) + 2 * kv) * HD
        kept = sum((c - r) % PAGE for r, c in geo)
        pages = sum(-(-c // PAGE) - (c - r) // PAGE for r, c in geo)
        b = rows * (proj * 2 + h * HD * 2 * (2 if case["gated"] else 1) + 2 * kv * HD + case["rot"] * 4 + 8)
        b += kept * kv * 2 * HD + pages * kv * 2 * 4 + 2 * HD * 2
        return {"bytes": b, "flops": rows * (h + kv) * HD * 8}
    keys = pairs = pages = 0
    for r, c in geo:
        k, p = _visible(case, r, c)
        keys, pairs, pages = keys + k, pairs + p, pages + -(-k // PAGE)
    b = keys * kv * 2 * HD + pages * (kv * 2 * 4 + 4) + rows * h * HD * 2 * (3 if case["gated"] else 2)
    return {"bytes": b, "flops": 4 * pairs * h * HD}


# ---- inputs ------------------------------------------------------------------------------

def _random_codes(shape, gen, dev):
    """e4m3 codes of normally distributed values, as bytes."""
    out = torch.empty(shape, dtype=torch.uint8, device=dev)
    step = max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, shape[0], step):
        part = torch.randn(out[i:i + step].shape, generator=gen, device=dev)
        out[i:i + step] = part.mul_(80.0).clamp_(-448, 448).to(F8).view(torch.uint8)
    return out


def _random_scales(blocks, kv, gen, dev):
    """Powers of two, so that values are near 0.6, 1.2 and 2.5."""
    return torch.pow(2.0, torch.randint(-7, -4, (blocks, kv), generator=gen, device=dev).float())


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    geo = _geometry(case)
    h, kv = case["heads"], case["kv_heads"]
    s = {"case": case}
    cu, ctx, positions = [0], [], []
    for r, c in geo:
        cu.append(cu[-1] + r)
        ctx.append(c)
        positions += range(c - r, c)
    total = cu[-1]
    i32 = dict(dtype=torch.int32, device=dev)
    s["cu_q"], s["context_lens"] = torch.tensor(cu, **i32), torch.tensor(ctx, **i32)
    s["positions"] = torch.tensor(positions, **i32)
    s["max_rows"], s["max_context"] = max(r for r, _ in geo), max(ctx)
    # pages in random order, some of the pool unused
    if case["kind"] == "append":  # only the pages that the rows fall into are in this pool
        need = [(-(-c // PAGE)) - (c - r) // PAGE for r, c in geo]
        first = [(c - r) // PAGE for r, c in geo]
    else:
        need, first = [-(-c // PAGE) for c in ctx], [0] * len(ctx)
    blocks = sum(need) + 5
    perm, at, tables, slots = torch.randperm(blocks, generator=host).tolist(), 0, [], []
    for (r, c), n, f in zip(geo, need, first):
        pages = perm[at:at + n]
        at += n
        tables.append(pages + [0] * (max(need) - n))
        slots += [pages[p // PAGE - f] * PAGE + p % PAGE for p in range(c - r, c)]
    s["block_table"], s["slots"] = torch.tensor(tables, **i32), torch.tensor(slots, **i32)
    s["blocks"] = blocks
    shape = (blocks, PAGE, kv, HD)
    s["k_cache"], s["v_cache"] = _random_codes(shape, gen, dev), _random_codes(shape, gen, dev)
    s["k_scale"], s["v_scale"] = _random_scales(blocks, kv, gen, dev), _random_scales(blocks, kv, gen, dev)
    bf = dict(dtype=torch.bfloat16, device=dev)
    proj = (h * (2 if case["gated"] else 1) + 2 * kv) * HD
    if case["kind"] == "append":
        s["qkv"] = torch.randn(total, proj, generator=gen, device=dev).mul_(1.5).to(torch.bfloat16)
        s["q_norm"] = torch.randn(HD, generator=gen, device=dev).mul_(0.1).add_(1).to(torch.bfloat16)
        s["k_norm"] = torch.randn(HD, generator=gen, device=dev).mul_(0.1).add_(1).to(torch.bfloat16)
        half = case["rot"] // 2
        freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        angle = torch.arange(max(ctx), dtype=torch.float64, device=dev)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.empty(total, h * HD, **bf)
        s["gate_out"] = torch.empty(total, h * HD, **bf) if case["gated"] else None
    else:
        s["q"] = torch.randn(total, h * HD, generator=gen, device=dev).mul_(1.5).to(torch.bfloat16)
        s["gate"] = torch.randn(total, h * HD, generator=gen, device=dev).to(torch.bfloat16) if case["gated"] else None
        s["out"] = torch.empty(total, h * HD, **bf)
    if own:  # what a serving program keeps across passes: the batch descriptor and the workspace
        from pilm_b200 import bindings, ckernel
        bindings.init()
        s["desc"] = ckernel.attn_desc(
            num_seqs=len(geo), total_q=total, max_q_len=s["max_rows"], n_heads=h, n_kv_heads=kv, head_dim=HD,
            block_size=PAGE, num_blocks=blocks, max_blocks_per_seq=max(need), max_context=s["max_context"],
            qkv_stride=proj, rope_rows=max(ctx), rot_dim=case["rot"], eps=1e-6, add_one=False,
            output_gate=case["gated"])
        if case["kind"] != "append":
            n = ckernel.paged_attention_kv8_workspace_bytes(s["desc"], case["window"], case["sinks"])
            s["workspace"] = torch.empty(n, dtype=torch.uint8, device=dev)
    return s


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    if s["case"]["kind"] == "append":
        if own:
            from pilm_b200 import ckernel
            ckernel.qk_norm_rope_kv_append_kv8(
                s["desc"], s["qkv"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], s["positions"], s["slots"],
                s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["q_out"], s["gate_out"])
        else:
            _plain_append(s)
        out = {"q": s["q_out"], "k": s["k_cache"].view(F8), "v": s["v_cache"].view(F8), "k_scale": s["k_scale"],
               "v_scale": s["v_scale"]}
        if s["gate_out"] is not None:
            out["gate"] = s["gate_out"]
        return out
    if own:
        from pilm_b200 import ckernel
        ckernel.paged_attention_verify_kv8(
            s["desc"], s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["cu_q"],
            s["context_lens"], s["gate"], s["out"], window=s["case"]["window"], sinks=s["case"]["sinks"],
            workspace=s["workspace"])
        return s["out"]
    return _plain_attention(s)


def _norm_rope(x, weight, cos, sin, rot):
    """RMSNorm over the last axis, then the rotation of the first `rot` dims (pairs d, d + rot/2)."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)


def _plain_store(rows, slots, cache, scale):
    """Quantizes rows [T, kv, 128] into their pages, one power-of-two scale for a page and head."""
    blocks, kv = scale.shape
    page, off = slots // PAGE, slots % PAGE
    first = torch.full((blocks,), PAGE, device=slots.device).scatter_reduce(0, page, off, "amin")
    kept = (torch.arange(PAGE, device=slots.device) < first[:, None]) & (first < PAGE)[:, None]
    old = torch.where(kept[:, :, None, None], cache.view(F8).float() * scale[:, None, :, None], 0.0)
    amax = old.abs().amax((1, 3)).scatter_reduce(0, page[:, None].expand(-1, kv), rows.abs().amax(-1), "amax")
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875), 0)
    new_scale = torch.where((first < PAGE)[:, None], torch.ldexp(torch.ones_like(amax), e), scale)
    codes = (old / new_scale[:, None, :, None]).to(F8).view(torch.uint8)
    codes = torch.where(kept[:, :, None, None], codes, cache)
    codes.view(blocks * PAGE, kv, HD)[slots] = (rows / new_scale[page][:, :, None]).to(F8).view(torch.uint8)
    cache.copy_(codes)
    scale.copy_(new_scale)


def _plain_append(s):
    c = s["case"]
    h, kv, rot, t = c["heads"], c["kv_heads"], c["rot"], s["qkv"].shape[0]
    q, k, v = s["qkv"].split([s["qkv"].shape[1] - 2 * kv * HD, kv * HD, kv * HD], 1)
    q = q.view(t, h, -1)  # [q_h | gate_h] per head when gated
    if c["gated"]:
        s["gate_out"].copy_(q[..., HD:].reshape(t, h * HD))
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["q_out"].copy_(_norm_rope(q[..., :HD], s["q_norm"], cos, sin, rot).view(t, h * HD))
    slots = s["slots"].long()
    _plain_store(_norm_rope(k.view(t, kv, HD), s["k_norm"], cos, sin, rot), slots, s["k_cache"], s["k_scale"])
    _plain_store(v.view(t, kv, HD).float(), slots, s["v_cache"], s["v_scale"])


def _plain_attention(s):
    c = s["case"]
    h, kv, b, n = c["heads"], c["kv_heads"], c["seqs"], s["max_rows"]
    g, dev = h // kv, s["q"].device
    table, lens, cu = s["block_table"].long(), s["context_lens"].long(), s["cu_q"].long()
    rows = cu[1:] - cu[:-1]
    # [b, kv, keys, 128] and [b, kv, n * g, 128], rows padded to the longest pass
    k = (s["k_cache"].view(F8)[table].float() * s["k_scale"][table][:, :, None, :, None]).flatten(1, 2).transpose(1, 2)
    v = (s["v_cache"].view(F8)[table].float() * s["v_scale"][table][:, :, None, :, None]).flatten(1, 2).transpose(1, 2)
    j = torch.arange(n, device=dev)
    real = j < rows[:, None]
    at = torch.where(real, cu[:-1, None] + j, 0)
    q = s["q"].float()[at].view(b, n, kv, g, HD).permute(0, 2, 1, 3, 4).reshape(b, kv, n * g, HD)
    scores = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(HD)).view(b, kv, n, g, -1)
    pos = (lens - rows)[:, None] + j                      # [b, n]
    key = torch.arange(k.shape[2], device=dev)
    seen = key <= pos[..., None]
    if c["window"]:
        seen = seen & ((key > pos[..., None] - c["window"]) | (key < c["sinks"]))
    scores = scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(b, kv, n * g, -1)
    o = (p @ v).view(b, kv, n, g, HD).permute(0, 2, 1, 3, 4).reshape(b, n, h * HD)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())[at]
    s["out"][at[real]] = o[real].to(torch.bfloat16)
    return s["out"]


# ---- the definitions in 64 bits ------------------------------------------------------------

def _exact_codes(x, e):
    """x / 2^e rounded to the nearest e4m3 value, ties to even: 3 mantissa bits, least exponent -6."""
    y = torch.ldexp(x, -e)
    _, top = torch.frexp(y)
    ulp = torch.ldexp(torch.ones_like(y), (top - 1).clamp(min=-6) - 3)
    return torch.round(y / ulp) * ulp


def _exact_store(rows, slots, cache, scale):
    cache, scale = cache.view(F8).double(), scale.double().clone()
    by_page = {}
    for r, slot in enumerate(slots):
        by_page.setdefault(slot // PAGE, []).append((slot % PAGE, r))
    for page, put in by_page.items():
        lo = min(o for o, _ in put)
        new = rows[[r for _, r in put]]                                # [n, kv, 128]
        held = cache[page, :lo] * scale[page][None, :, None]
        amax = torch.cat([held, new]).abs().amax((0, 2))
        e = torch.ceil(torch.log2(amax / 448)).to(torch.int32)
        e = torch.where(torch.ldexp(torch.full_like(amax, 448.0), e - 1) >= amax, e - 1, e)
        e = torch.where(amax > 0, e, 0)
        cache[page, :lo] = _exact_codes(held, e[None, :, None])
        cache[page, [o for o, _ in put]] = _exact_codes(new, e[None, :, None])
        scale[page] = torch.ldexp(torch.ones_like(amax), e)
    return cache, scale


def _exact_append(s, c):
    h, kv, half, t = c["heads"], c["kv_heads"], c["rot"] // 2, s["qkv"].shape[0]
    x = s["qkv"].double()
    width = HD * (2 if c["gated"] else 1)
    pos = s["positions"].long()
    cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]

    def rotated(u, w):
        u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        z = torch.complex(u[..., :half], u[..., half:2 * half]) * torch.complex(cos, sin)[:, None]
        return torch.cat([z.real, z.imag, u[..., 2 * half:]], -1)

    heads = x[:, :h * width].reshape(t, h, width)
    k = x[:, h * width:h * width + kv * HD].reshape(t, kv, HD)
    v = x[:, h * width + kv * HD:].reshape(t, kv, HD)
    slots = s["slots"].tolist()
    k_cache, k_scale = _exact_store(rotated(k, s["k_norm"]), slots, s["k_cache"], s["k_scale"])
    v_cache, v_scale = _exact_store(v, slots, s["v_cache"], s["v_scale"])
    out = {"q": rotated(heads[..., :HD], s["q_norm"]).reshape(t, h * HD), "k": k_cache, "v": v_cache,
           "k_scale": k_scale, "v_scale": v_scale}
    if c["gated"]:
        out["gate"] = heads[..., HD:].reshape(t, h * HD)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s, case)
    h, kv = case["heads"], case["kv_heads"]
    g = h // kv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    cu, table = s["cu_q"].tolist(), s["block_table"].long()
    for b, n in enumerate(s["context_lens"].tolist()):
        pages = table[b, :-(-n // PAGE)]
        pos = torch.arange(n - (cu[b + 1] - cu[b]), n, device=out.device)[:, None]
        key = torch.arange(n, device=out.device)[None]
        hidden = key > pos
        if case["window"]:
            hidden |= (pos - key >= case["window"]) & (key >= case["sinks"])
        for i in range(kv):
            k = (s["k_cache"][pages, :, i].view(F8).double() * s["k_scale"][pages, i].double()[:, None, None])
            v = (s["v_cache"][pages, :, i].view(F8).double() * s["v_scale"][pages, i].double()[:, None, None])
            k, v = k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]
            for j in range(i * g, (i + 1) * g):
                q = s["q"][cu[b]:cu[b + 1], j * HD:(j + 1) * HD].double()
                logit = torch.where(hidden, -math.inf, torch.einsum("qd,kd->qk", q, k) / math.sqrt(HD))
                out[cu[b]:cu[b + 1], j * HD:(j + 1) * HD] = torch.softmax(logit, 1) @ v
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].double()))
    return out
