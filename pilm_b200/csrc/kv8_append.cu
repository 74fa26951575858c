// QK-RMSNorm + RoPE of a pass's rows, K and V quantized into the pages of an 8-bit cache.
//
// Cache: e4m3 codes [num_blocks, 16, n_kv, 128] for K and for V, and one fp32 scale per page
// and KV head [num_blocks, n_kv]; an element is code * scale.  The rows that one call writes
// into a page join the tokens at offsets below the first of them (the page's kept tokens; what
// lies above is stale: rejected drafts, an earlier owner's tokens).  With
//   amax = max |x| over the kept tokens (as stored) and the new rows,
//   e    = the least integer from -126 on with amax <= 448 * 2^e   (0 for an all-zero page)
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
    uint32_t num_slots;  // at most 2^31 - 16
    size_t stride;
    float eps;
    int total_q, nh, nkv, gated, add_one, rope_rows, nf;
    int kv_blocks, band;  // blocks of K/V, the first of the grid; rows of each
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

// Sixteen lanes hold a head, eight dims each: four from d0 on and four from d1 on.  For vectors the
// two are each other's partners in the rotation, which then needs no exchange between lanes (dims
// that are not rotated pair up among themselves); nf is a multiple of 4 there.
struct Dims {
    int d0, d1;
};
template <bool VEC>
__device__ __forceinline__ Dims lane_dims(int nf) {
    const int l = threadIdx.x & 15, n = nf / 4;
    if (!VEC) return {4 * l, 64 + 4 * l};
    return l < n ? Dims{4 * l, 4 * l + nf} : Dims{4 * (l + n), 4 * (l + n) + 64 - nf};
}

template <bool VEC>
__device__ __forceinline__ void load8(const AppendParams &p, size_t off, const Dims &d, uint2 (&r)[2]) {
    r[0] = load4<VEC>(p, off + d.d0), r[1] = load4<VEC>(p, off + d.d1);
}

// The norm weight of the lane's dims (1 + w for Gemma norms).
template <bool VEC>
__device__ __forceinline__ void norm_weight(const __nv_bfloat16 *w, int add_one, const Dims &d, float (&out)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const __nv_bfloat16 *at = w + (h ? d.d1 : d.d0);
        if constexpr (VEC) {
            unpack4(*reinterpret_cast<const uint2 *>(at), *reinterpret_cast<float (*)[4]>(&out[4 * h]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * h + j] = bf2f(at[j]);
        }
    }
    if (add_one)
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] += 1.f;
}

// The norm weight and the rotation of a position as one pair of factors for each of the lane's dims:
//   y[d] = (x[d] * a[d] + x[partner(d)] * b[d]) * rsqrt(mean x^2 + eps)
// first half: (a cos - b sin), second: (a sin + b cos) (layers.py:161-164).  Dims that are not
// rotated, as all are at positions outside the table, have b = 0.  Two dims per 64-bit word.
struct Rotation {
    uint64_t a[4], b[4];
};
// buf: 128 floats of the half warp
template <bool VEC>
__device__ __forceinline__ Rotation rotation(const AppendParams &p, const float (&w)[8], int pos, const Dims &d, float *buf) {
    Rotation r;
    const int nf = p.nf;
    const bool ok = pos >= 0 && pos < p.rope_rows;
    float a[8], b[8];
    if constexpr (VEC) {
        float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ok && d.d0 < nf) {
            const size_t at = (size_t)pos * nf + d.d0;
            c = *reinterpret_cast<const float4 *>(p.cos_t + at);
            s = *reinterpret_cast<const float4 *>(p.sin_t + at);
        }
        const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = w[j] * cv[j], b[j] = -(w[4 + j] * sv[j]);
            a[4 + j] = w[4 + j] * cv[j], b[4 + j] = w[j] * sv[j];
        }
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) buf[(j < 4 ? d.d0 : d.d1 - 4) + j] = w[j];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = (j < 4 ? d.d0 : d.d1 - 4) + j;
            const bool rot = ok && e < 2 * nf;
            const size_t at = rot ? (size_t)pos * nf + (e < nf ? e : e - nf) : 0;
            a[j] = rot ? w[j] * p.cos_t[at] : w[j];
            b[j] = rot ? (e < nf ? -p.sin_t[at] * buf[e + nf] : p.sin_t[at] * buf[e - nf]) : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) r.a[j] = f2_pack(a[2 * j], a[2 * j + 1]), r.b[j] = f2_pack(b[2 * j], b[2 * j + 1]);
    return r;
}

// x -> rope(rmsnorm(x) * w) of one head per half warp.
template <bool VEC>
__device__ __forceinline__ void norm_rope(const uint2 (&raw)[2], const Rotation &r, const Dims &d, int nf, float eps,
                                          float *buf, float (&y)[8]) {
    float x[8];
    unpack4(raw[0], *reinterpret_cast<float (*)[4]>(&x[0]));
    unpack4(raw[1], *reinterpret_cast<float (*)[4]>(&x[4]));
    uint64_t v[4], o[4], sq = 0ull;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2_pack(x[2 * j], x[2 * j + 1]), sq = f2_fma(v[j], v[j], sq);
    const float2 s2 = f2_unpack(sq);
    float ss = s2.x + s2.y;
#pragma unroll
    for (int i = 8; i; i >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, i);
    if constexpr (VEC) {
        o[0] = v[2], o[1] = v[3], o[2] = v[0], o[3] = v[1];
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) buf[(j < 4 ? d.d0 : d.d1 - 4) + j] = x[j];
        __syncwarp();
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = (j < 4 ? d.d0 : d.d1 - 4) + j;
            t[j] = e < nf ? buf[e + nf] : (e < 2 * nf ? buf[e - nf] : x[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f2_pack(t[2 * j], t[2 * j + 1]);
    }
    const float inv = rsqrtf(ss * (1.f / kHD) + eps);
    const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 z = f2_unpack(f2_mul(f2_fma(v[j], r.a[j], f2_mul(o[j], r.b[j])), inv2));
        y[2 * j] = z.x, y[2 * j + 1] = z.y;
    }
}

// the largest magnitude, NaN if one is NaN
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The exponent e of a page's scale: the least from -126 on with amax <= 448 * 2^e (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_exponent(float amax) {
    if (!(amax > 0.f)) return 0;
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}

// One page's share of one KV head: the run of rows that starts at row `lead`.  The first two warps of
// the block take K, the others V (is_k); half warp h of those four takes the offsets h, h + 4, h + 8
// and h + 12.  s_amax: one slot per warp.
template <bool VEC>
__device__ __forceinline__ void append_run(const AppendParams &p, int lead, int page, int head, bool is_k, float *buf, float *s_amax) {
    constexpr int N = kKv8Page / 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Dims d = lane_dims<VEC>(p.nf);
    // the row that writes each offset (lane o < 16)
    int my_row = -1;
    for (int base = lead;; base += 32) {
        const int r = base + lane;
        const int slot = r < p.total_q ? p.slots[r] : -1;
        const bool valid = (uint32_t)slot < p.num_slots;
        const uint32_t vm = __ballot_sync(0xffffffffu, valid);
        const uint32_t other = __ballot_sync(0xffffffffu, valid && (slot >> 4) != page);
        const int limit = other ? __ffs((int)other) - 1 : 32;
        const bool in = valid && lane < limit;
        const int off = slot & 15, off0 = __shfl_sync(0xffffffffu, off, 0);
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

    const size_t tok = (size_t)p.nkv * kHD;  // bytes from one token to the next
    uint8_t *cache = (is_k ? p.kc : p.vc) + ((size_t)page * kKv8Page) * tok + (size_t)head * kHD;
    float *scale = (is_k ? p.ks : p.vs) + (size_t)page * p.nkv + head;
    const float old_scale = lo > 0 ? *scale : 0.f;
    const size_t src = (size_t)(p.nh * (p.gated ? 2 : 1) + (is_k ? 0 : p.nkv) + head) * kHD;
    const int o0 = 2 * (warp & 1) + (lane >> 4);
    uint32_t kept[N][2];
    uint2 raw[N][2];
    int row[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int o = o0 + 4 * i;
        const uint8_t *at = cache + o * tok;
        kept[i][0] = o < lo ? *reinterpret_cast<const uint32_t *>(at + d.d0) : 0u;
        kept[i][1] = o < lo ? *reinterpret_cast<const uint32_t *>(at + d.d1) : 0u;
        row[i] = __shfl_sync(0xffffffffu, my_row, o);
        raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
        if (row[i] >= 0) load8<VEC>(p, (size_t)row[i] * p.stride + src, d, raw[i]);
    }
    float x[N][8], amax = 0.f;
    if (is_k) {
        int pos[N];
#pragma unroll
        for (int i = 0; i < N; ++i) pos[i] = row[i] >= 0 ? p.positions[row[i]] : -1;
        float w[8];
        norm_weight<VEC>(p.knw, p.add_one, d, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (__any_sync(0xffffffffu, row[i] >= 0)) {  // (a half without a row: zeros)
                norm_rope<VEC>(raw[i], rotation<VEC>(p, w, pos[i], d, buf), d, p.nf, p.eps, buf, x[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            unpack4(raw[i][0], *reinterpret_cast<float (*)[4]>(&x[i][0]));
            unpack4(raw[i][1], *reinterpret_cast<float (*)[4]>(&x[i][4]));
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) amax = max3_abs_nan(amax, x[i][j], x[i][j + 1]);
    if (!(amax < INFINITY)) {  // NaN is stored as 0, infinities saturate at what the finite values need
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (!(x[i][j] == x[i][j])) x[i][j] = 0.f;
                if (fabsf(x[i][j]) < INFINITY) amax = fmaxf(amax, fabsf(x[i][j]));
            }
    }
    // e4m3 magnitudes order like their codes: the kept tokens' largest is their largest code
    // (0x7f is NaN, which this call never writes; taken as the largest finite one)
    float kept_max = 0.f;
    if (lo > 0) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) top = __vmaxu4(top, __vmaxu4(kept[i][0] & 0x7f7f7f7fu, kept[i][1] & 0x7f7f7f7fu));
        uint32_t code = max(max(top & 0xffu, (top >> 8) & 0xffu), max((top >> 16) & 0xffu, top >> 24));
        code = min(__reduce_max_sync(0xffffffffu, code), 0x7eu);
        kept_max = f16x2_to_f32x2(e4m3x2_to_f16x2(code)).x * old_scale;
    }
    // a finite magnitude: its bits order like it
    amax = fmaxf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax))), kept_max);
    if (lane == 0) s_amax[warp] = amax;
    __syncthreads();  // and every warp has read the old scale
    amax = fmaxf(s_amax[warp & ~1], s_amax[warp | 1]);
    const int e = scale_exponent(amax);
    const float new_scale = pow2f(e), inv = pow2f(-e);
    // kept zeros stay as they are: the ratio of the scales may be infinite there (elsewhere it is at most
    // 2^18: the largest kept value, at least 2^-9 * old_scale, is at most 448 * new_scale)
    const bool rescale = kept_max > 0.f && new_scale != old_scale;
    const float f = old_scale * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int o = o0 + 4 * i;
        uint8_t *at = cache + o * tok;
        if (row[i] >= 0) {
            *reinterpret_cast<uint32_t *>(at + d.d0) = f32x4_to_e4m3x4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv);
            *reinterpret_cast<uint32_t *>(at + d.d1) = f32x4_to_e4m3x4(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv);
        } else if (rescale && o < lo) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 a = f16x2_to_f32x2(e4m3x2_to_f16x2(kept[i][h]));
                const float2 b = f16x2_to_f32x2(e4m3x2hi_to_f16x2(kept[i][h]));
                *reinterpret_cast<uint32_t *>(at + (h ? d.d1 : d.d0)) = f32x4_to_e4m3x4(a.x * f, a.y * f, b.x * f, b.y * f);
            }
        }
    }
    if ((warp & 1) == 0 && lane == 0) *scale = new_scale;
}

// The first kv_blocks blocks take one KV head for `band` consecutive rows, and of those rows the ones
// that begin a page's run (the row before them, rows without a slot aside, writes another page).  So
// one block alone reads and writes a page's scale and codes for a head, and needs no other's amax.
// In the others a warp takes QH query heads of one row, all loaded before the first is worked on.
// One launch for both parts, since a token's whole call is a few microseconds: 2.9 us for one row of
// 16 + 2 x 8 heads and 4.0 for 96 rows of 32 + 2 x 8, a chain of loads (slot -> row -> position ->
// rotation, page -> codes).  6880 rows of prompts of 32 + 2 x 8 heads: 45 us, 3.4 TB/s, where the
// query heads alone take 26 and K and V alone 25: a warp waits 11 cycles between instructions
// (loads, instruction fetch, the barrier), so for prompts (QH = 8) the registers are held to eight
// blocks per SM (48 us with five); a head per whole warp, whose rotation exchanges values between lanes,
// took 55.
template <bool VEC, int QH>
__global__ void __launch_bounds__(kAppendWarps * 32, QH == 8 ? 8 : 1) kv8_append(const AppendParams p) {
    pdl_trigger();
    __shared__ float s_buf[VEC ? 1 : kAppendWarps][2][kHD];
    __shared__ float s_amax[2][kAppendWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4;
    float *buf = s_buf[VEC ? 0 : warp][half];
    pdl_wait();
    if ((int)blockIdx.x >= p.kv_blocks) {
        const int groups = (p.nh + QH - 1) / QH;
        const uint32_t item = (blockIdx.x - p.kv_blocks) * kAppendWarps + warp, row = item / (uint32_t)groups;
        if (row >= (uint32_t)p.total_q) return;
        const int h0 = (int)(item - row * groups) * QH + half, width = kHD * (p.gated ? 2 : 1);
        const Dims d = lane_dims<VEC>(p.nf);
        const size_t src = (size_t)row * p.stride + (size_t)h0 * width;
        const size_t dst = ((size_t)row * p.nh + h0) * kHD;
        const int pos = p.positions[row];
        uint2 raw[QH / 2][2];
#pragma unroll
        for (int i = 0; i < QH / 2; ++i) {  // the half's heads h0, h0 + 2 ..
            raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
            if (h0 + 2 * i < p.nh) load8<VEC>(p, src + (size_t)(2 * i) * width, d, raw[i]);
        }
        if (p.gated)
#pragma unroll
            for (int i = 0; i < QH / 2; ++i)
                if (h0 + 2 * i < p.nh) {
                    uint2 g[2];
                    load8<VEC>(p, src + (size_t)(2 * i) * width + kHD, d, g);
                    store4<VEC>(p.gate_out + dst + 2 * i * kHD + d.d0, g[0]);
                    store4<VEC>(p.gate_out + dst + 2 * i * kHD + d.d1, g[1]);
                }
        float w[8];
        norm_weight<VEC>(p.qnw, p.add_one, d, w);
        const Rotation r = rotation<VEC>(p, w, pos, d, buf);
#pragma unroll
        for (int i = 0; i < QH / 2; ++i) {
            float y[8];
            norm_rope<VEC>(raw[i], r, d, p.nf, p.eps, buf, y);
            if (h0 + 2 * i < p.nh) {
                store4<VEC>(p.q_out + dst + 2 * i * kHD + d.d0, pack4(*reinterpret_cast<const float (*)[4]>(&y[0])));
                store4<VEC>(p.q_out + dst + 2 * i * kHD + d.d1, pack4(*reinterpret_cast<const float (*)[4]>(&y[4])));
            }
        }
        return;
    }
    const int row0 = (int)blockIdx.x / p.nkv * p.band, head = (int)blockIdx.x % p.nkv;
    // lanes 16 .. 16 + band - 1 are the block's rows, lanes 0 .. 15 the rows before them
    const int r = row0 - 16 + lane;
    const int slot = r >= 0 && r < p.total_q && lane < 16 + p.band ? p.slots[r] : -1;
    const bool valid = (uint32_t)slot < p.num_slots;
    const int page = valid ? slot >> 4 : -1;
    const uint32_t vmask = __ballot_sync(0xffffffffu, valid);
    const uint32_t below = vmask & ((1u << lane) - 1u);
    int prev = __shfl_sync(0xffffffffu, page, below ? 31 - __clz((int)below) : 0);
    if (!below) prev = -1;
    // rows without a slot may fill the window: look further back for the first of the band
    if (!(vmask & 0xffffu) && (vmask >> 16) && row0 > 16) {
        int far = -1;
        for (int base = row0 - 17; base >= 0 && far < 0; base -= 32) {
            const int sl = base >= lane ? p.slots[base - lane] : -1;
            const uint32_t m = __ballot_sync(0xffffffffu, (uint32_t)sl < p.num_slots);
            if (m) far = __shfl_sync(0xffffffffu, sl >> 4, __ffs((int)m) - 1);
        }
        if (!below) prev = far;
    }
    uint32_t lead = __ballot_sync(0xffffffffu, valid && lane >= 16 && prev != page);
    for (int n = 0; lead; ++n, lead &= lead - 1) {
        const int l = __ffs((int)lead) - 1;
        append_run<VEC>(p, row0 - 16 + l, __shfl_sync(0xffffffffu, page, l), head, warp < 2, buf, s_amax[n & 1]);
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
    PILM_REQUIRE(d->qkv_stride >= width && d->qkv_stride <= 0x7fffffff, ECPU_ERR_PARAM,
                 "%s: qkv_stride %zu is not in [%zu, 2^31), from the row's values on", what, d->qkv_stride, width);
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
    p.num_slots = (uint32_t)d->num_blocks * kKv8Page;
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
    const long long kvb = ((long long)p.total_q + p.band - 1) / p.band * p.nkv, blocks = qb + kvb;
    PILM_REQUIRE(blocks <= 0x7fffffffLL, ECPU_ERR_PARAM, "%s: too many rows", what);
    p.kv_blocks = (int)kvb;
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
    PILM_REQUIRE(d->max_blocks_per_seq <= 0x7fffffff, ECPU_ERR_PARAM, "%s: max_blocks_per_seq must be below 2^31", what);
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
