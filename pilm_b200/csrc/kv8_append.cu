// QK-RMSNorm + RoPE of a pass's rows, K and V quantized into the pages of an 8-bit cache.
//
// Cache: e4m3 codes [num_blocks, 16, n_kv, 128] for K and for V, and one fp32 scale per page
// and KV head [num_blocks, n_kv]; an element is code * scale.  The rows that one call writes
// into a page join the tokens at offsets below the first of them (the page's kept tokens; what
// lies above is stale: rejected drafts, an earlier owner's tokens).  With
//   amax = max |x| over the kept tokens (as stored) and the new rows,
//   e    = the least integer with amax <= 448 * 2^e   (0 for an all-zero page)
// the page's scale becomes 2^e, the kept codes are rounded to it and the new rows stored as
// rne_e4m3(x * 2^-e).  A power of two costs an e4m3 value nothing (its exponent moves), so
// requantizing kept tokens is exact except where a code becomes subnormal, and a page holds
// the same values whatever rows were written and rejected in between, except for those.
//
// The reference's rows are FullAttention.forward's (src/models/qwen3/attention.py:79-97,
// layers.py:122-176); the reference has no 8-bit cache.  Everything here is fp32 with one
// rounding at the end (q to bf16, K and V to e4m3), not the bf16 module rounding of the
// bf16-cache prologue: there is no reference result to reproduce, and each rounding left out
// is error left out.
#include "fp8.cuh"

using namespace pilm;

namespace {

constexpr int kHD = kKv8HD;
constexpr int kAppendWarps = 4;

struct AppendParams {
    const __nv_bfloat16 *qkv;  // [total_q, qkv_stride], or null
    const float *part;         // [splits][total_q][qkv_stride] split-K partial sums, or null
    int splits;
    size_t plane;              // elements of one split
    const __nv_bfloat16 *qnw, *knw;
    const float *cos_t, *sin_t;  // [rope_rows, rot_dim / 2]
    const int32_t *positions, *slots;
    uint8_t *kc, *vc;
    float *ks, *vs;
    __nv_bfloat16 *q_out, *gate_out;
    long long num_slots;
    size_t stride;
    float eps;
    int total_q, nh, nkv, gated, add_one, rope_rows, nf;
    int q_blocks, band;  // blocks of query items; rows per K/V warp
};

// Four consecutive projection values as bf16 bits.  Split-K partials are summed in split order
// and rounded: the value that the projection's own combine pass writes.
template <bool VEC>
__device__ __forceinline__ uint2 load4(const AppendParams &p, size_t off) {
    if (p.part) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.splits; ++k) {
            const float *pl = p.part + (size_t)k * p.plane + off;
            if constexpr (VEC) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(pl));
                s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += __ldcs(pl + j);
            }
        }
        const __nv_bfloat162 a = __floats2bfloat162_rn(s[0], s[1]), b = __floats2bfloat162_rn(s[2], s[3]);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    if constexpr (VEC) {
        return *reinterpret_cast<const uint2 *>(p.qkv + off);
    } else {
        const uint16_t *x = reinterpret_cast<const uint16_t *>(p.qkv) + off;
        return make_uint2(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16);
    }
}
__device__ __forceinline__ void unpack4(uint2 v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}

template <bool VEC>
__device__ __forceinline__ void store4(__nv_bfloat16 *dst, uint2 v) {
    if constexpr (VEC) {
        *reinterpret_cast<uint2 *>(dst) = v;
    } else {
        uint16_t *d = reinterpret_cast<uint16_t *>(dst);
        d[0] = (uint16_t)v.x, d[1] = (uint16_t)(v.x >> 16), d[2] = (uint16_t)v.y, d[3] = (uint16_t)(v.y >> 16);
    }
}
__device__ __forceinline__ uint2 pack4(const float (&x)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// Lane l's dims 4l .. 4l + 3 of the norm weight (1 + w for Gemma norms).
template <bool VEC>
__device__ __forceinline__ void norm_weight(const __nv_bfloat16 *w, int add_one, float (&out)[4]) {
    const int d = 4 * (threadIdx.x & 31);
    if constexpr (VEC) {
        const uint2 v = *reinterpret_cast<const uint2 *>(w + d);
        out[0] = __uint_as_float(v.x << 16), out[1] = __uint_as_float(v.x & 0xffff0000u);
        out[2] = __uint_as_float(v.y << 16), out[3] = __uint_as_float(v.y & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = bf2f(w[d + j]);
    }
    if (add_one)
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] += 1.f;
}

// The norm weight and the rotation of a position as one pair of factors for each of lane l's dims:
//   y[d] = (x[d] * a[d] + x[partner(d)] * b[d]) * rsqrt(mean x^2 + eps)
// first half: (a cos - b sin), second: (a sin + b cos) (layers.py:161-164).  A dim that is not
// rotated, as all are at positions outside the table, is its own partner with b = 0.
struct Rotation {
    float a[4], b[4];
};
template <bool VEC>
__device__ __forceinline__ Rotation rotation(const AppendParams &p, const float (&w)[4], int pos, float *buf) {
    Rotation r;
    const int lane = threadIdx.x & 31, d = 4 * lane, nf = p.nf;
    const bool ok = pos >= 0 && pos < p.rope_rows;
    if constexpr (VEC) {  // nf is a multiple of 4: a lane's dims are all in one half
        const bool rot = ok && d < 2 * nf;
        float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (rot) {
            const size_t at = (size_t)pos * nf + (d < nf ? d : d - nf);
            c = *reinterpret_cast<const float4 *>(p.cos_t + at);
            s = *reinterpret_cast<const float4 *>(p.sin_t + at);
        }
        const float sign = d < nf ? -1.f : 1.f;
        const int partner = d >= 2 * nf ? lane : (d < nf ? lane + nf / 4 : lane - nf / 4);
        const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            r.a[j] = w[j] * cv[j];
            r.b[j] = sign * sv[j] * __shfl_sync(0xffffffffu, w[j], partner);
        }
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) buf[d + j] = w[j];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = d + j;
            const bool rot = ok && e < 2 * nf;
            const size_t at = rot ? (size_t)pos * nf + (e < nf ? e : e - nf) : 0;
            r.a[j] = rot ? w[j] * p.cos_t[at] : w[j];
            r.b[j] = rot ? (e < nf ? -p.sin_t[at] * buf[e + nf] : p.sin_t[at] * buf[e - nf]) : 0.f;
        }
    }
    return r;
}

// x -> rope(rmsnorm(x) * w) of one head held 4 dims per lane; buf: 128 floats of the warp.
template <bool VEC>
__device__ __forceinline__ void norm_rope(float (&x)[4], const Rotation &r, int nf, float eps, float *buf) {
    const int lane = threadIdx.x & 31, d = 4 * lane;
    const float ss = warp_sum(x[0] * x[0] + x[1] * x[1] + (x[2] * x[2] + x[3] * x[3]));
    float o[4];  // the partners
    if constexpr (VEC) {
        const int partner = d >= 2 * nf ? lane : (d < nf ? lane + nf / 4 : lane - nf / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __shfl_sync(0xffffffffu, x[j], partner);
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) buf[d + j] = x[j];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = d + j;
            o[j] = e < nf ? buf[e + nf] : (e < 2 * nf ? buf[e - nf] : x[j]);
        }
    }
    const float inv = rsqrtf(ss * (1.f / kHD) + eps);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (x[j] * r.a[j] + o[j] * r.b[j]) * inv;
}

// The exponent e of a page's scale: the least with amax <= 448 * 2^e (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_exponent(float amax) {
    if (!(amax > 0.f)) return 0;
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// One page's share of one KV head, K (is_k) or V: the run of rows that starts at row `lead`.  Warp
// w of the block takes the offsets w, w + 4, w + 8, w + 12; s_amax: one slot per warp.
template <bool VEC>
__device__ void append_run(const AppendParams &p, int lead, long long page, int head, bool is_k, float *buf,
                           float *s_amax) {
    constexpr int N = kKv8Page / kAppendWarps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the row that writes each offset (lane o < 16)
    int my_row = -1;
    for (int base = lead;; base += 32) {
        const int r = base + lane;
        const long long slot = r < p.total_q ? p.slots[r] : -1;
        const bool valid = slot >= 0 && slot < p.num_slots;
        const uint32_t vm = __ballot_sync(0xffffffffu, valid);
        const uint32_t other = __ballot_sync(0xffffffffu, valid && (slot >> 4) != page);
        const int limit = other ? __ffs((int)other) - 1 : 32;
        const bool in = valid && lane < limit;
        const int off = (int)(slot & 15), off0 = __shfl_sync(0xffffffffu, off, 0);
        const uint32_t inm = vm & (limit == 32 ? ~0u : (1u << limit) - 1u);
        if (base == lead && __popc(inm) <= 16 && inm == (1u << __popc(inm)) - 1u && __all_sync(0xffffffffu, !in || off == off0 + lane)) {
            if (lane >= off0 && lane < off0 + __popc(inm)) my_row = lead + lane - off0;  // slots in order
        } else {
#pragma unroll 1
            for (int o = 0; o < 16; ++o) {  // the last row, where rows repeat a slot
                const uint32_t m = __ballot_sync(0xffffffffu, in && off == o);
                if (m && lane == o) my_row = base + 31 - __clz((int)m);
            }
        }
        if (other || base + 32 >= p.total_q) break;
    }
    const uint32_t wmask = __ballot_sync(0xffffffffu, my_row >= 0);
    const int lo = __ffs((int)wmask) - 1;  // the first offset written: tokens below it are kept

    uint8_t *cache = (is_k ? p.kc : p.vc) + (((size_t)page * kKv8Page) * p.nkv + head) * kHD + 4 * lane;
    const size_t tok = (size_t)p.nkv * kHD;  // bytes from one token to the next
    float *scale = (is_k ? p.ks : p.vs) + (size_t)page * p.nkv + head;
    const float old_scale = lo > 0 ? *scale : 0.f;
    const size_t src = (size_t)(p.nh * (p.gated ? 2 : 1) + (is_k ? 0 : p.nkv) + head) * kHD + 4 * lane;
    uint32_t kept[N];
    uint2 raw[N];
    int row[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int o = warp + kAppendWarps * i;
        kept[i] = o < lo ? *reinterpret_cast<const uint32_t *>(cache + o * tok) : 0u;
        row[i] = __shfl_sync(0xffffffffu, my_row, o);
        raw[i] = row[i] >= 0 ? load4<VEC>(p, (size_t)row[i] * p.stride + src) : make_uint2(0u, 0u);
    }
    float w[4] = {1.f, 1.f, 1.f, 1.f};
    if (is_k) norm_weight<VEC>(p.knw, p.add_one, w);
    float x[N][4], amax = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unpack4(raw[i], x[i]);
        if (is_k && row[i] >= 0) norm_rope<VEC>(x[i], rotation<VEC>(p, w, p.positions[row[i]], buf), p.nf, p.eps, buf);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            amax = fmaxf(amax, fabsf(x[i][j]));
            odd |= !(fabsf(x[i][j]) < INFINITY);
        }
    }
    if (odd) {  // NaN is stored as 0, infinities saturate at what the finite values need
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!(x[i][j] == x[i][j])) x[i][j] = 0.f;
                if (fabsf(x[i][j]) < INFINITY) amax = fmaxf(amax, fabsf(x[i][j]));
            }
    }
    // e4m3 magnitudes order like their codes: the kept tokens' largest is their largest code
    // (0x7f is NaN, which this call never writes; taken as the largest finite one)
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = __vmaxu4(top, kept[i] & 0x7f7f7f7fu);
    uint32_t code = max(max(top & 0xffu, (top >> 8) & 0xffu), max((top >> 16) & 0xffu, top >> 24));
    code = min(__reduce_max_sync(0xffffffffu, code), 0x7eu);
    amax = fmaxf(warp_max(amax), f16x2_to_f32x2(e4m3x2_to_f16x2(code)).x * old_scale);
    if (lane == 0) s_amax[warp] = amax;
    __syncthreads();  // and every warp has read the old scale
#pragma unroll
    for (int i = 0; i < kAppendWarps; ++i) amax = fmaxf(amax, s_amax[i]);
    const int e = scale_exponent(amax);
    const float new_scale = pow2f(e), inv = pow2f(-e);
    const bool rescale = lo > 0 && new_scale != old_scale;
    const float f = old_scale * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int o = warp + kAppendWarps * i;
        uint32_t *dst = reinterpret_cast<uint32_t *>(cache + o * tok);
        if (row[i] >= 0) {
            *dst = f32x4_to_e4m3x4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv);
        } else if (rescale && o < lo) {
            const float2 a = f16x2_to_f32x2(e4m3x2_to_f16x2(kept[i]));
            const float2 b = f16x2_to_f32x2(e4m3x2hi_to_f16x2(kept[i]));
            *dst = f32x4_to_e4m3x4(a.x * f, a.y * f, b.x * f, b.y * f);
        }
    }
    if (threadIdx.x == 0) *scale = new_scale;
}

// Blocks [0, q_blocks): a warp takes QH query heads of one row, all loaded before the first is
// worked on.  The others: a block takes K or V of one KV head for `band` consecutive rows, and of
// those rows the ones that begin a page's run (the row before them, rows without a slot aside,
// writes another page).  So one block alone reads and writes a page's scale and codes for a head,
// and needs no other's amax.  Bound by HBM for prompts and by latency (slot -> page -> codes) for
// single tokens; one launch for both parts, since a token's whole call is a few microseconds.
template <bool VEC, int QH>
__global__ void __launch_bounds__(kAppendWarps * 32) kv8_append(const AppendParams p) {
    pdl_trigger();
    __shared__ float s_buf[kAppendWarps][kHD];
    __shared__ float s_amax[2][kAppendWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *buf = s_buf[warp];
    pdl_wait();
    if ((int)blockIdx.x < p.q_blocks) {
        const int groups = (p.nh + QH - 1) / QH;
        const long long item = (long long)blockIdx.x * kAppendWarps + warp;
        if (item >= (long long)p.total_q * groups) return;
        const int row = (int)(item / groups), h0 = (int)(item % groups) * QH;
        const int width = kHD * (p.gated ? 2 : 1);
        const size_t src = (size_t)row * p.stride + (size_t)h0 * width + 4 * lane;
        const size_t dst = ((size_t)row * p.nh + h0) * kHD + 4 * lane;
        const int pos = p.positions[row];
        uint2 raw[QH];
#pragma unroll
        for (int i = 0; i < QH; ++i)
            raw[i] = h0 + i < p.nh ? load4<VEC>(p, src + (size_t)i * width) : make_uint2(0u, 0u);
        if (p.gated)
#pragma unroll
            for (int i = 0; i < QH; ++i)
                if (h0 + i < p.nh) store4<VEC>(p.gate_out + dst + i * kHD, load4<VEC>(p, src + (size_t)i * width + kHD));
        float w[4];
        norm_weight<VEC>(p.qnw, p.add_one, w);
        const Rotation r = rotation<VEC>(p, w, pos, buf);
#pragma unroll
        for (int i = 0; i < QH; ++i)
            if (h0 + i < p.nh) {
                float x[4];
                unpack4(raw[i], x);
                norm_rope<VEC>(x, r, p.nf, p.eps, buf);
                store4<VEC>(p.q_out + dst + i * kHD, pack4(x));
            }
        return;
    }
    const int combos = 2 * p.nkv;
    const int item = (int)blockIdx.x - p.q_blocks;
    const long long row0 = (long long)(item / combos) * p.band;
    const int combo = item % combos;
    // lanes 16 .. 16 + band - 1 are the block's rows, lanes 0 .. 15 the rows before them
    const long long r = row0 - 16 + lane;
    const long long slot = r >= 0 && r < p.total_q && lane < 16 + p.band ? p.slots[r] : -1;
    const bool valid = slot >= 0 && slot < p.num_slots;
    const long long page = valid ? slot >> 4 : -1;
    const uint32_t vmask = __ballot_sync(0xffffffffu, valid);
    const uint32_t below = vmask & ((1u << lane) - 1u);
    long long prev = __shfl_sync(0xffffffffu, page, below ? 31 - __clz((int)below) : 0);
    if (!below) prev = -1;
    // rows without a slot may fill the window: look further back for the first of the band
    if (!(vmask & 0xffffu) && (vmask >> 16) && row0 > 16) {
        long long far = -1;
        for (long long base = row0 - 17; base >= 0 && far < 0; base -= 32) {
            const long long q = base - lane;
            const long long sl = q >= 0 ? p.slots[q] : -1;
            const bool v = sl >= 0 && sl < p.num_slots;
            const uint32_t m = __ballot_sync(0xffffffffu, v);
            if (m) far = __shfl_sync(0xffffffffu, sl >> 4, __ffs((int)m) - 1);
        }
        if (!below) prev = far;
    }
    uint32_t lead = __ballot_sync(0xffffffffu, valid && lane >= 16 && prev != page);
    for (int n = 0; lead; ++n, lead &= lead - 1) {
        const int l = __ffs((int)lead) - 1;
        append_run<VEC>(p, (int)(row0 - 16 + l), __shfl_sync(0xffffffffu, page, l), combo >> 1, !(combo & 1), buf,
                        s_amax[n & 1]);
    }
}

bool aligned(const void *ptr, size_t to) { return ((uintptr_t)ptr & (to - 1)) == 0; }

int append(const ekernel_paged_attn_desc_t *d, const uint16_t *qkv, const float *part, int splits,
           const uint16_t *q_norm_w, const uint16_t *k_norm_w, const float *rope_cos, const float *rope_sin,
           const int32_t *positions, const int32_t *slot_mapping, uint8_t *k_cache, uint8_t *v_cache, float *k_scale,
           float *v_scale, uint16_t *q_out, uint16_t *gate_out, const char *what) {
    int rc = kv8_check_desc(d, what);
    if (rc != ECPU_OK) return rc;
    if (d->total_q == 0) return ECPU_OK;
    const bool tables = d->rot_dim > 0 && d->rope_rows > 0;  // without them none is read
    PILM_REQUIRE((qkv || part) && q_norm_w && k_norm_w && ((rope_cos && rope_sin) || !tables) && positions &&
                     slot_mapping && k_cache && v_cache && k_scale && v_scale && q_out,
                 ECPU_ERR_PARAM, "%s: null argument", what);
    PILM_REQUIRE(!d->output_gate || gate_out, ECPU_ERR_PARAM, "%s: gate_out required when output_gate", what);
    PILM_REQUIRE(aligned(k_cache, 16) && aligned(v_cache, 16), ECPU_ERR_PARAM,
                 "%s: the K and V caches must be 16-byte aligned", what);
    const size_t width = (d->n_heads * (d->output_gate ? 2 : 1) + 2 * d->n_kv_heads) * kHD;
    PILM_REQUIRE(d->qkv_stride >= width, ECPU_ERR_PARAM, "%s: qkv_stride %zu is below the row's %zu values", what,
                 d->qkv_stride, width);
    AppendParams p;
    p.qkv = (const __nv_bfloat16 *)qkv;
    p.part = part;
    p.splits = splits;
    p.plane = d->total_q * d->qkv_stride;
    p.qnw = (const __nv_bfloat16 *)q_norm_w;
    p.knw = (const __nv_bfloat16 *)k_norm_w;
    p.cos_t = rope_cos;
    p.sin_t = rope_sin;
    p.positions = positions;
    p.slots = slot_mapping;
    p.kc = k_cache;
    p.vc = v_cache;
    p.ks = k_scale;
    p.vs = v_scale;
    p.q_out = (__nv_bfloat16 *)q_out;
    p.gate_out = (__nv_bfloat16 *)gate_out;
    p.num_slots = (long long)d->num_blocks * kKv8Page;
    p.stride = d->qkv_stride;
    p.eps = d->eps;
    p.total_q = (int)d->total_q;
    p.nh = (int)d->n_heads;
    p.nkv = (int)d->n_kv_heads;
    p.gated = d->output_gate ? 1 : 0;
    p.add_one = d->add_one;
    p.rope_rows = (int)d->rope_rows;
    p.nf = (int)d->rot_dim / 2;
    // Rows per K/V block.  Verify passes have a few rows per sequence, each a page's first: one
    // row per block runs them side by side.  A prompt's pages take 16 rows each, and a block for
    // every row would mostly start, find another's run and leave.
    p.band = d->max_q_len >= kKv8Page ? kKv8Page : 1;
    // Query heads per warp: two where all the warps fit on the GPU at once (a short call's time is
    // one warp's), eight, with their loads in flight together, where they do not.
    const int qh = (long long)p.total_q * p.nh > (long long)num_sms() * 16 * 2 * kAppendWarps ? 8 : 2;
    const long long q_items = (long long)p.total_q * ((p.nh + qh - 1) / qh);
    const long long qb = (q_items + kAppendWarps - 1) / kAppendWarps;
    const long long blocks = qb + ((long long)p.total_q + p.band - 1) / p.band * 2 * p.nkv;
    PILM_REQUIRE(blocks <= 0x7fffffffLL, ECPU_ERR_PARAM, "%s: too many rows", what);
    p.q_blocks = (int)qb;
    // 8- and 16-byte accesses where every base and row allows them, and a lane's four dims are
    // rotated alike; single elements otherwise
    const bool vec = (d->qkv_stride & 3) == 0 && aligned(qkv, 8) && aligned(part, 16) && aligned(q_norm_w, 8) &&
                     aligned(k_norm_w, 8) && aligned(rope_cos, 16) && aligned(rope_sin, 16) && aligned(q_out, 8) &&
                     aligned(gate_out, 8) && (p.nf & 3) == 0;
    launch_pdl(vec ? (qh == 8 ? kv8_append<true, 8> : kv8_append<true, 2>)
                   : (qh == 8 ? kv8_append<false, 8> : kv8_append<false, 2>),
               dim3((unsigned)blocks), dim3(kAppendWarps * 32), 0, p);
    return check_launch(what);
}

}  // namespace

namespace pilm {

int kv8_check_desc(const ekernel_paged_attn_desc_t *d, const char *what) {
    PILM_REQUIRE(d, ECPU_ERR_PARAM, "%s: null descriptor", what);
    PILM_REQUIRE(d->head_dim == kKv8HD, ECPU_ERR_UNSUPPORTED, "%s: head_dim must be 128", what);
    PILM_REQUIRE(d->block_size == kKv8Page, ECPU_ERR_UNSUPPORTED, "%s: block_size must be 16", what);
    PILM_REQUIRE(d->n_kv_heads > 0 && d->n_heads > 0 && d->n_heads % d->n_kv_heads == 0, ECPU_ERR_PARAM,
                 "%s: n_heads must be a multiple of n_kv_heads", what);
    PILM_REQUIRE(d->total_q <= 0x7fffff && d->num_seqs <= 0xffff && d->n_heads <= 1024, ECPU_ERR_PARAM,
                 "%s: sizes out of range", what);
    PILM_REQUIRE(d->num_blocks > 0 && d->num_blocks < (1u << 27), ECPU_ERR_PARAM,
                 "%s: num_blocks must be in [1, 2^27)", what);
    PILM_REQUIRE(d->rot_dim <= kKv8HD && (d->rot_dim & 1) == 0 && d->rope_rows <= 0x7fffffff, ECPU_ERR_PARAM,
                 "%s: bad rot_dim or rope_rows", what);
    return ECPU_OK;
}

}  // namespace pilm

extern "C" {

int ekernel_qk_norm_rope_kv_append_kv8(const ekernel_paged_attn_desc_t *desc, const uint16_t *qkv,
                                       const uint16_t *q_norm_w, const uint16_t *k_norm_w, const float *rope_cos,
                                       const float *rope_sin, const int32_t *positions, const int32_t *slot_mapping,
                                       uint8_t *k_cache, uint8_t *v_cache, float *k_scale, float *v_scale,
                                       uint16_t *q_out, uint16_t *gate_out) {
    return append(desc, qkv, nullptr, 0, q_norm_w, k_norm_w, rope_cos, rope_sin, positions, slot_mapping, k_cache,
                  v_cache, k_scale, v_scale, q_out, gate_out, "ekernel_qk_norm_rope_kv_append_kv8");
}

int ekernel_qk_norm_rope_kv_append_kv8_splitk(const ekernel_paged_attn_desc_t *desc, const float *partials,
                                              int32_t splits, const uint16_t *q_norm_w, const uint16_t *k_norm_w,
                                              const float *rope_cos, const float *rope_sin, const int32_t *positions,
                                              const int32_t *slot_mapping, uint8_t *k_cache, uint8_t *v_cache,
                                              float *k_scale, float *v_scale, uint16_t *q_out, uint16_t *gate_out) {
    const char *what = "ekernel_qk_norm_rope_kv_append_kv8_splitk";
    PILM_REQUIRE(splits > 0, ECPU_ERR_PARAM, "%s: splits must be positive", what);
    return append(desc, nullptr, partials, splits, q_norm_w, k_norm_w, rope_cos, rope_sin, positions, slot_mapping,
                  k_cache, v_cache, k_scale, v_scale, q_out, gate_out, what);
}

}  // extern "C"
