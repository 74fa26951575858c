// Paged attention over an 8-bit KV cache (e4m3 codes, one scale per page and KV head).
//
// out = softmax(q k^T / sqrt(128)) v for rows at the end of each sequence's context; a row at
// position p sees keys <= p, or with a window the keys in (p - window, p] and the first sinks.
// With k = ks * K8 and v = vs * V8 of a page, codes K8 and V8 being f16 values exactly:
//   s = (q . K8) * (ks / sqrt(128))      the scale of a page multiplies 16 scores, not 2048 codes
//   o = 2^d / sum 2^(s - m) * sum_pages (2^(s - m + log2 vs - d) . V8)
// in base 2.  Each row has two running references: m for its scores, m + d for s + log2 vs over the keys
// that it sees.  What goes into the product with V is thus held relative to the row's own largest
// p * vs, and no page that it does not see, or gives no weight, takes bits from the others.
// m is a whole number.  So is d in the token kernel: with power-of-two scales every exponent's constant
// is exact and O is rescaled exactly, so that a row's result hardly depends on when its references moved
// or on which power of two a page's scale is, and a verified row nearly always repeats what decoding it
// gave (drafts from a model's own continuation over 8K contexts: 59 of a hundred accepted, 2 with d a
// multiple of 2^-14).  In the chunk kernel, whose rows no decoding repeats, it is such a multiple: the
// weight that sets it is then exact in f16 to 2^-15, and 5.6 of a hundred outputs of prompts are not the
// nearest bf16, 7.1 with whole numbers (in the token kernel 4 to 6, and 7 to 8 as it is).
//
// The reference's attention is FullAttention.forward (src/models/qwen3/attention.py:98-139);
// it caches in the model's dtype, so there is no reference result to reproduce here: scores
// stay in fp32.
#include "fp8.cuh"

using namespace pilm;

// Set when a bounded wait gave up (read and cleared in synchronous mode).
static __device__ int g_kv8_error;

namespace {

constexpr int kHD = kKv8HD;
// Polls, of about two microseconds each, before a wait gives up (ekernel_set_wait_limit's instead where
// set; the waits for what is in flight at the end keep this one).
constexpr uint32_t kWaitLimit = 1u << 20;

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t *b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_test(uint64_t *b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait; false once it has polled `limit` times (0: if it is not met now) or another warp gave up.
__device__ __forceinline__ bool mbar_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag, uint32_t limit) {
    if (mbar_test(b, parity)) return true;
    for (uint32_t i = 0; i < limit; ++i) {
        if (mbar_try_wait(b, parity)) return true;
        if ((i & 255) == 255 && *abort_flag) return false;
    }
    return false;
}
// A wait for what always completes, before the CTA may exit.
__device__ __forceinline__ void mbar_drain(uint64_t *b, uint32_t parity) {
    for (uint32_t i = 0; i < kWaitLimit; ++i)
        if (mbar_try_wait(b, parity)) return;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            dst),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// The barrier's phase also waits for this thread's cp.async so far (one of its expected arrivals).
__device__ __forceinline__ void cp_async_arrive(uint64_t *b) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// log2 of a page's scale, -inf for 0 and below 2^-126.  Exact for powers of two, which lg2.approx below 1
// is not: the exponent (as a float: 2^23 + its bits) plus the logarithm of the significand, 0 at 1.
__device__ __forceinline__ float log2_scale(float x) {
    const uint32_t b = __float_as_uint(x);
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__uint_as_float((b & 0x7fffffu) | 0x3f800000u)));
    y += __uint_as_float((b >> 23) | 0x4b000000u) - 8388735.f;
    return b < 0x800000u ? -INFINITY : y;
}

constexpr float kScoreScale = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)
// The weights p * vs are held as 2^9 p vs / 2^M in f16 for a reference M = m + d at most kLag below
// their running maximum (in base 2): below 2^16, with 11 bits down to 2^-23 of that maximum and
// steps of 2^-33 below, so a long tail of small ones still counts.  The lag, which m has too, spares
// most of the rescalings of O: a new maximum within it leaves the references where they are.
constexpr float kProbBits = 9.f, kLag = 6.75f;
// A page's log2 vs - d is held to this: below, its weights are nothing in f16, while its scores, which
// come from the same exponentials, still count in the sum of p.
constexpr float kLogFloor = -60.f;
__device__ __forceinline__ float finite_or_0(float x) { return x == -INFINITY ? 0.f : x; }
__device__ __forceinline__ float floor_2m14(float x) { return floorf(x * 0x1p14f) * 0x1p-14f; }
// O -> out: 2^d / l as two factors, neither of which leaves the normal range (g is 1 but near its ends)
struct OutScale {
    float f, g;
};
__device__ __forceinline__ OutScale out_scale(float d, float l) {
    const bool lo = d < -100.f, hi = d > 100.f;
    const float e = lo ? d + 64.f : (hi ? d - 64.f : d);
    return {l > 0.f ? __fdiv_rn(ex2(e), l) : 0.f, lo ? 0x1p-64f : (hi ? 0x1p64f : 1.f)};
}
// Partials of a row (reference m, sum l, output o of four dims) join by their shares of the sum so far, so
// that o stays a convex combination of the values, in their range; a NaN partial gives NaN.
struct Joined {
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    // U more (-inf and 0 where there is none)
    template <int U>
    __device__ __forceinline__ void add(const float (&m2)[U], const float (&l2)[U], const float4 (&o2)[U]) {
        float mx = m, w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, m2[u]);
        const float mb = finite_or_0(mx), had = l * ex2(m - mb);
        m = mx, l = had;
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = l2[u] * ex2(m2[u] - mb), l += w[u];
        const float inv = l > 0.f ? __frcp_rn(l) : 0.f, keep = had * inv;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= keep;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float x = w[u] * inv;
            o[0] += x * o2[u].x, o[1] += x * o2[u].y, o[2] += x * o2[u].z, o[3] += x * o2[u].w;
        }
    }
};

// x / (1 + exp(-gate)) of eight outputs
__device__ __forceinline__ void apply_gate(float (&e)[8], const __nv_bfloat16 *gate) {
    const uint4 gw = *reinterpret_cast<const uint4 *>(gate);
    const uint32_t wd[4] = {gw.x, gw.y, gw.z, gw.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float gt = __uint_as_float((j & 1) ? (wd[j >> 1] & 0xffff0000u) : (wd[j >> 1] << 16));
        e[j] = __fdividef(e[j], 1.f + __expf(-gt));
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16 *out, const float (&e)[8]) {
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(e[2 * j], e[2 * j + 1]);
        r[j] = *reinterpret_cast<const uint32_t *>(&t);
    }
    *reinterpret_cast<uint4 *>(out) = make_uint4(r[0], r[1], r[2], r[3]);
}
// four merged outputs at element `at`
__device__ __forceinline__ void finish4(__nv_bfloat16 *out, const __nv_bfloat16 *gate, size_t at, const float (&o)[4]) {
    uint2 gw = make_uint2(0u, 0u);
    if (gate) gw = *reinterpret_cast<const uint2 *>(gate + at);
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[i] = o[i];
        if (gate) {
            const uint32_t w = i < 2 ? gw.x : gw.y;
            const float gt = __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
            e[i] = __fdividef(e[i], 1.f + __expf(-gt));
        }
    }
    const __nv_bfloat162 lo = __floats2bfloat162_rn(e[0], e[1]), hi = __floats2bfloat162_rn(e[2], e[3]);
    *reinterpret_cast<uint2 *>(out + at) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}

// ---------------------------------------------------------------------------------
// Geometry shared by the kernels.  rho = j * gsz + g numbers a sequence's rows, for query row j and
// head g of a KV head's group.  The token kernel takes a sequence's rows together; the keys that
// they see are a list of nv pages: the first n_sink pages of the sequence, then those from lo_page
// on.
// ---------------------------------------------------------------------------------
struct Geometry {
    const int32_t *cu_q, *ctx;
    int gsz;            // query heads per KV head
    int window, sinks;  // window 0: none
};
struct Group {
    int q0, rows, p0, ctx;  // first row, rows (rho) of the sequence, position of row j = 0
    int n_sink, lo_page, nv;
};

__device__ __forceinline__ Group group_of(const Geometry &g, int rpg, int b) {  // rpg: rows at most
    Group r;
    r.q0 = g.cu_q[b];
    const int q_len = g.cu_q[b + 1] - r.q0;
    r.ctx = g.ctx[b];
    r.rows = min(q_len * g.gsz, rpg);
    r.p0 = r.ctx - q_len;
    r.n_sink = r.lo_page = r.nv = 0;
    if (r.rows <= 0) return r;
    const int pmin = r.p0, pmax = r.p0 + (r.rows - 1) / g.gsz;
    if (pmax < 0) return r;
    const int end = (pmax >> 4) + 1;
    if (g.window > 0) {
        r.lo_page = pmin - g.window + 1 > 0 ? (pmin - g.window + 1) >> 4 : 0;
        r.n_sink = min((g.sinks + 15) >> 4, r.lo_page);
    }
    r.nv = r.n_sink + end - r.lo_page;
    return r;
}
__device__ __forceinline__ int page_of(const Group &g, int v) { return v < g.n_sink ? v : v - g.n_sink + g.lo_page; }

// Shares of T units among G CTAs: CTA c has [share(c), share(c + 1)).  32-bit divisions where the
// products fit (64-bit ones are subroutines, and took most of the merge kernel's time).
__device__ __forceinline__ int share_of(int c, int T, int G) {
    const unsigned long long n = (unsigned long long)c * (unsigned)T;
    return (n >> 32) == 0 ? (int)((unsigned)n / (unsigned)G) : (int)(n / (unsigned)G);
}
// the CTA whose share holds unit x
__device__ __forceinline__ int cta_of(int x, int T, int G) {
    const unsigned long long n = (unsigned long long)x * (unsigned)G;
    int c = (n >> 32) == 0 ? (int)((unsigned)n / (unsigned)T) : (int)(n / (unsigned)T);
    if (c >= G) c = G - 1;
    while (c + 1 < G && share_of(c + 1, T, G) <= x) ++c;
    while (c > 0 && share_of(c, T, G) > x) --c;
    return c;
}

// ---------------------------------------------------------------------------------
// Token kernel: calls of at most 32 rows per KV head (decode, verify), bound by reading the cache.
//
// One CTA per SM.  The sequences' pages, in blocks of `pps`, form one list that the CTAs of a head
// group share evenly: a producer warp streams whole blocks (K and V of `hg` KV heads) through a
// TMA ring, and consumer warp (h, c, k) takes head h, row tile c (16 rows) and pages 2k, 2k + 1
// of each block, so every byte is read from HBM once and 8 warps share the conversions.  A sequence
// that a boundary cuts leaves partial sums for the merge kernel; with few sequences and short
// contexts a CTA takes a whole sequence and there is nothing to merge.
//
// Per pair of pages a warp computes S = Q K8^T and O += P V8 with mma.sync m16n8k16 on f16, the
// codes converted in registers as they leave shared memory (e4m3 operands run no faster: sm_100 has
// no e4m3 mma.sync of its own).  Both products sum over an index whose order is free, and each order
// is chosen so that a thread's operand is contiguous in the cache as it lies there: thread (g, c) =
// (lane / 4, lane % 4) holds dims 32c .. 32c + 31 of a key for S, and dims 16g .. 16g + 15 of its
// four keys for O, where four byte permutes pair the keys.  With the TMA's 128-byte swizzle all these
// 16-byte shared-memory loads are free of bank conflicts.
//
// The tcgen05 pipe does not fit these shapes: one token's rows (gsz = 4, say) would fill 4 of its
// 128 rows.  mma.sync at 16 rows keeps up with HBM.
//
// Measured, in a captured graph: 96 verify rows over 32 x 8236 keys, 32 + 8 heads: 93.5 us with the
// merge, 5.1 TB/s of cache, where the copy of as many bytes takes 74 us and this kernel with its
// arithmetic left out 89 (sums of pages differ by up to a block of 0.8 us between the CTAs, and the
// first bytes arrive 5 us after the start).  One row over 131071 keys 54.4 us, 4.9 TB/s; one row over 301
// keys 8.2 us, a chain of loads (lengths and page ids -> pages), two rounds of products and a join.
// ---------------------------------------------------------------------------------
constexpr int kTokWarps = 8;      // consumer warps at most
// Three warpgroups: two of consumers, and one whose first warp is the producer.  Launched with
// 168 registers a thread (64512 in all), the producer's group keeps 40 and the consumers take 232:
// 256 * 232 + 128 * 40 = 64512.
constexpr int kTokThreads = 384;
constexpr int kTokGroups = 4096;  // groups per launch (their prefix is kept in shared memory)
constexpr int kTokStages = 8;     // ring stages at most
constexpr int kMergeScan = 128;   // groups up to which the merge works out the prefix itself
constexpr int kRec = kHD + 4;     // a partial: O[128] normalised, max (base 2), sum, two pad floats

struct TokParams {
    Geometry geo;
    const __nv_bfloat16 *q, *gate;
    const float *ks, *vs;
    const int32_t *block_table;
    __nv_bfloat16 *out;
    float *part;      // [head groups][G][2][hg * rpg][kRec]
    int *prefix_out;  // [groups + 1]: blocks before each group, for the merge
    int nh, nkv, max_blocks, num_blocks;
    int groups, hg, ch, kw, pps, rpg, stages, G;  // groups: sequences; rpg = 16 ch rows of each
    int whole;  // a CTA per group (and head group) instead of equal shares of all pages
    uint32_t wait_limit;
};

// Rows of a group that sees no key.
__device__ void zero_rows(const TokParams &p, const Group &g, int head0, int heads) {
    for (int i = threadIdx.x; i < g.rows * heads * (kHD / 8); i += blockDim.x) {
        const int d = i % (kHD / 8), h = i / (kHD / 8) % heads, rho = i / (kHD / 8) / heads;
        if (head0 + h >= p.nkv) continue;
        const size_t row = (size_t)(g.q0 + rho / p.geo.gsz) * p.nh + (head0 + h) * p.geo.gsz + rho % p.geo.gsz;
        *reinterpret_cast<uint4 *>(p.out + row * kHD + 8 * d) = make_uint4(0u, 0u, 0u, 0u);
    }
}

__global__ void __launch_bounds__(kTokThreads, 1) kv8_attn_tokens(const __grid_constant__ CUtensorMap kmap,
                                                                           const __grid_constant__ CUtensorMap vmap,
                                                                           const TokParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_prefix[kTokGroups + 1];
    __shared__ __align__(8) uint64_t full_bar[kTokStages], empty_bar[kTokStages], meet_bar;
    __shared__ float s_scale[kTokStages][2][16];  // [stage][K, V][page of the block * hg + head]
    __shared__ uint32_t s_valid[kTokStages];      // bit i: page i of the block has a valid id
    __shared__ float2 s_ml[2][kTokWarps][16];     // [segment parity][warp][row]: max, sum
    __shared__ int s_abort;
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int consumers = p.hg * p.ch * p.kw;
    const int cta = blockIdx.x, head0 = blockIdx.y * p.hg;
    const uint32_t page_bytes = (uint32_t)p.hg * 2048;        // K (or V) of one page, hg heads
    const uint32_t stage_bytes = 2 * page_bytes * p.pps;      // K pages, then V pages
    if (threadIdx.x == 0) {
        for (int st = 0; st < p.stages; ++st) {
            mbar_init(&full_bar[st], 1 + 32);
            mbar_init(&empty_bar[st], (uint32_t)consumers);
        }
        mbar_init(&meet_bar, (uint32_t)consumers);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTokWarps && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? &vmap : &kmap) : "memory");
    pdl_wait();
    // only now: the merge kernel reads the batch's geometry before it waits for this one, and what
    // came before this one (which may have written it) is complete here
    pdl_trigger();
    int x0, x1;  // this CTA's blocks
    int v_first;       // the group of block x0
    Group own;         // and its geometry
    int early = -1;    // the producer's first page ids, where they can be asked for beside the lengths
    if (p.whole) {     // (s_prefix: only the CTA's own group, from 0)
        if (warp == kTokWarps && p.geo.window == 0 && lane < min(p.pps, p.max_blocks))
            early = p.block_table[(size_t)cta * p.max_blocks + lane];
        own = group_of(p.geo, p.rpg, cta);
        v_first = cta;
        x0 = 0, x1 = (own.nv + p.pps - 1) / p.pps;
        __syncthreads();
        if (x1 == 0) {
            zero_rows(p, own, head0, p.hg);
            return;
        }
    } else {
        if (warp == 0) {  // blocks before each group
            int carry = 0;
            if (lane == 0) s_prefix[0] = 0;
            for (int v0 = 0; v0 < p.groups; v0 += 32) {
                const int v = v0 + lane;
                int n = v < p.groups ? (group_of(p.geo, p.rpg, v).nv + p.pps - 1) / p.pps : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, n, o);
                    if (lane >= o) n += up;
                }
                if (v < p.groups) s_prefix[v + 1] = carry + n;
                carry += __shfl_sync(0xffffffffu, n, 31);
            }
        }
        __syncthreads();
        if (cta == 0 && blockIdx.y == 0 && p.groups > kMergeScan)
            for (int v = threadIdx.x; v <= p.groups; v += blockDim.x) p.prefix_out[v] = s_prefix[v];
        for (int v = cta; v < p.groups; v += p.G)
            if (s_prefix[v] == s_prefix[v + 1]) zero_rows(p, group_of(p.geo, p.rpg, v), head0, p.hg);
        const int T = s_prefix[p.groups];
        x0 = share_of(cta, T, p.G), x1 = share_of(cta + 1, T, p.G);
        if (x0 >= x1) return;
        int lo = 0, hi = p.groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_prefix[mid] <= x0) lo = mid; else hi = mid - 1;
        }
        v_first = lo;
        own = group_of(p.geo, p.rpg, v_first);
    }
    auto start = [&](int v) { return p.whole ? (v == v_first ? 0 : x1) : s_prefix[v]; };
    const uint32_t ring = smem_u32(smem);

    if (warp >= kTokWarps) {
        // ---- producer ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp > kTokWarps) return;
        int v = v_first, issued = 0;
        Group g = own;
        bool ok = true;
        // a block's page ids are fetched one block ahead (lane i: page i of the block)
        auto fetch = [&](int x, int &vv, Group &gg) {
            if (x >= x1) return -1;
            while (x >= start(vv + 1)) gg = group_of(p.geo, p.rpg, ++vv);
            const int vp = (x - start(vv)) * p.pps + lane;
            int blk = -1;
            if (lane < p.pps && vp < gg.nv) {
                const int pg = page_of(gg, vp);
                if (pg < p.max_blocks) blk = p.block_table[(size_t)vv * p.max_blocks + pg];
            }
            return blk;  // as it comes: a look at it here would wait for the load
        };
        int next = p.whole && p.geo.window == 0 ? (lane < g.nv ? early : -1) : fetch(x0, v, g);
        for (int x = x0; x < x1; ++x, ++issued) {
            const int blk = (uint32_t)next < (uint32_t)p.num_blocks ? next : -1;
            next = fetch(x + 1, v, g);
            const int st = issued % p.stages;
            if (issued >= p.stages)
                ok = mbar_wait(&empty_bar[st], (uint32_t)(issued / p.stages - 1) & 1u, &s_abort, p.wait_limit);
            if (!__all_sync(0xffffffffu, ok)) break;
            const uint32_t valid = __ballot_sync(0xffffffffu, blk >= 0);
            if (lane == 0) {
                s_valid[st] = valid;  // published by the arrive
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_expect_tx(&full_bar[st], (uint32_t)__popc(valid) * 2 * page_bytes);
            }
            __syncwarp();
            if (blk >= 0) {
                const uint32_t dst = ring + st * stage_bytes + lane * page_bytes;
                tma_load_3d(dst, &kmap, &full_bar[st], 0, blk * kKv8Page, head0);
                tma_load_3d(dst + p.pps * page_bytes, &vmap, &full_bar[st], 0, blk * kKv8Page, head0);
            }
            const int pg = lane / p.hg, h = lane % p.hg;  // pps * hg <= 16 scales of each kind
            const int src = __shfl_sync(0xffffffffu, blk, pg & 31);
            if (pg < p.pps && src >= 0 && head0 + h < p.nkv) {
                const size_t at = (size_t)src * p.nkv + head0 + h;
                cp_async_4(smem_u32(&s_scale[st][0][lane]), p.ks + at);
                cp_async_4(smem_u32(&s_scale[st][1][lane]), p.vs + at);
            }
            cp_async_arrive(&full_bar[st]);
        }
        if (!__all_sync(0xffffffffu, ok) && lane == 0) {
            s_abort = 1;
            atomicExch(&g_kv8_error, 1);
        }
        // every copy issued lands before the CTA may exit
        for (int j = issued > p.stages ? issued - p.stages : 0; j < issued; ++j)
            mbar_drain(&full_bar[j % p.stages], (uint32_t)(j / p.stages) & 1u);
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    if (warp >= consumers) return;

    // ---- consumer warp (h, c, k) ----
    const int k_of = warp % p.kw, c_of = warp / p.kw % p.ch, h_of = warp / (p.kw * p.ch);
    const int g4 = lane >> 2, c4 = lane & 3;
    const int head = head0 + h_of;
    const bool head_ok = head < p.nkv;
    // byte offsets of this thread's loads in one head's 2 KB tile (rows of 128 B, 16-byte chunk i
    // of row r at i ^ (r & 7))
    const uint32_t k_off = g4 * 128 + ((2 * c4 ^ g4) << 4);                    // key g4; its second chunk: ^ 16
    const uint32_t v_off = 2 * c4 * 128 + ((g4 ^ (2 * c4)) << 4);              // key 2 c4
    const uint32_t v_off1 = (2 * c4 + 1) * 128 + ((g4 ^ (2 * c4 + 1)) << 4);   // key 2 c4 + 1; both: + 8 rows
    // all consumer warps meet (bounded, unlike a hardware barrier whose partner has given up)
    int met = 0;
    auto meet = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet_bar);
        const bool w = __all_sync(0xffffffffu, mbar_wait(&meet_bar, (uint32_t)met++ & 1u, &s_abort, p.wait_limit));
        if (!w && lane == 0) {
            s_abort = 1;
            atomicExch(&g_kv8_error, 1);
        }
        return w;
    };
    int done = 0;  // blocks consumed
    int v = v_first;
    bool ok = true;
    int segs = 0;
    for (int x = x0; x < x1 && ok; ++segs) {
        while (x >= start(v + 1)) ++v;
        const Group g = v == v_first ? own : group_of(p.geo, p.rpg, v);
        const int seg1 = min(x1, start(v + 1));
        const bool whole = x == start(v) && seg1 == start(v + 1);
        const int slot = x == x0 ? 0 : 1;
        const int tile0 = 16 * c_of;
        const bool active = head_ok && tile0 < g.rows;
        const int tile1 = min(g.rows, tile0 + 16);

        // queries in f16 as q * 2^k, the largest magnitude of the row in [2^14, 2^15): exact for bf16
        // elements down to 2^-28 of the largest; 2^-k goes into the row's score factor
        uint32_t qf[8][4];
        float rowf[2];
        int qpos[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const int rho = tile0 + g4 + 8 * hh;
            const bool in = active && rho < tile1;
            qpos[hh] = in ? g.p0 + rho / p.geo.gsz : -1;
            const __nv_bfloat16 *qr =
                p.q + ((size_t)(g.q0 + rho / p.geo.gsz) * p.nh + head * p.geo.gsz + rho % p.geo.gsz) * kHD + 32 * c4;
            uint4 w[4];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = in ? *reinterpret_cast<const uint4 *>(qr + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t wd[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(wd[j] << 16)), fabsf(__uint_as_float(wd[j] & 0xffff0000u))));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            int sh = 14 - ((int)(__float_as_uint(mx) >> 23) - 127);
            sh = sh > 126 ? 126 : sh;
            const float up = pow2f(sh);
            rowf[hh] = pow2f(-sh) * kScoreScale;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t wd[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    qf[2 * i + (j >> 1)][2 * (j & 1) + hh] =
                        pack_f16(__uint_as_float(wd[j] << 16) * up, __uint_as_float(wd[j] & 0xffff0000u) * up);
            }
        }
        // The pages [plain0, plain1) of the list need no mask: every row of the tile sees them whole.
        const int pmin = g.p0 + tile0 / p.geo.gsz, pmax = g.p0 + (tile1 - 1) / p.geo.gsz;
        int plain0 = 0, plain1 = pmin + 1 > 0 ? (pmin + 1) >> 4 : 0;  // ends at or before pmin
        if (p.geo.window > 0) {
            const int first = pmax - p.geo.window + 1;  // the last row's first key
            plain0 = g.n_sink + max(0, (first > 0 ? (first + 15) >> 4 : 0) - g.lo_page);
            plain1 = plain1 - g.lo_page + g.n_sink;
        }

        float o[16][4], m[2] = {-INFINITY, -INFINITY}, d[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float base[2] = {kProbBits, kProbBits}, dz[2] = {0.f, 0.f};  // kProbBits - m and d, with 0 for -inf
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        for (; x < seg1; ++x, ++done) {
            const int st = done % p.stages;
            ok = mbar_wait(&full_bar[st], (uint32_t)(done / p.stages) & 1u, &s_abort, p.wait_limit);
            if (!__all_sync(0xffffffffu, ok)) {
                if (lane == 0) {
                    s_abort = 1;
                    atomicExch(&g_kv8_error, 1);
                }
                ok = false;
                break;
            }
            const int vp = (x - start(v)) * p.pps + 2 * k_of;
            if (active && vp < g.nv) {
                const uint32_t kb = ring + st * stage_bytes + (2 * k_of) * page_bytes + h_of * 2048;
                const uint32_t vb = kb + p.pps * page_bytes;
                const uint32_t valid = s_valid[st] >> (2 * k_of) & 3u;
                const bool masked = vp < plain0 || vp + 2 > plain1 || valid != 3u;
                float kf[2], lv[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int at = (2 * k_of + i) * p.hg + h_of;
                    kf[i] = s_scale[st][0][at];
                    lv[i] = log2_scale(s_scale[st][1][at]);
                }
                // ---- S = Q K8^T: two pages of two 8-key tiles, four independent chains ----
                float s[2][2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[i][t][j] = 0.f;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint4 w[2][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            w[i][t] = lds128(kb + i * page_bytes + t * 1024 + (hf ? k_off ^ 16u : k_off));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const uint32_t c = k == 0 ? w[i][t].x : (k == 1 ? w[i][t].y : (k == 2 ? w[i][t].z : w[i][t].w));
                                mma_f16(s[i][t], qf[4 * hf + k], e4m3x2_to_f16x2(c), e4m3x2hi_to_f16x2(c));
                            }
                }
                // ---- scores in base 2, masks, online softmax ----
                // A page's K scale is a factor of its raw products, applied with the reference in one
                // fma; its V scale is an addend there (p' = p * vs / 2^d), taken out of the sum again.
                float f[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i) f[i][0] = rowf[0] * kf[i], f[i][1] = rowf[1] * kf[i];
                int key0[2] = {0, 0};
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const bool ok_page = (valid >> i) & 1u;
                        if (!ok_page) lv[i] = -INFINITY;
                        key0[i] = page_of(g, vp + i) * 16;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int key = key0[i] + 8 * t + 2 * c4 + (j & 1), qp = qpos[j >> 1];
                                const bool see = vp + i < g.nv && key <= qp &&
                                                 (p.geo.window == 0 || key > qp - p.geo.window || key < p.geo.sinks);
                                // a page with no valid id is one of zeros
                                s[i][t][j] = see ? (ok_page ? s[i][t][j] : 0.f) : -INFINITY;
                            }
                        // -inf must not meet a factor of 0 (nor what lies in the place of a missing page's): with
                        // the least normal number there a product is still nothing beside the exponents
                        f[i][0] = fmaxf(ok_page ? f[i][0] : 0.f, 1.17549435e-38f);
                        f[i][1] = fmaxf(ok_page ? f[i][1] : 0.f, 1.17549435e-38f);
                    }
                }
                // this thread's largest score of each page, and whether any thread's moves a reference
                float top[2][2];
                bool rise = false, huge = false;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    const int e = 2 * hh;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        top[i][hh] = fmaxf(max3(s[i][0][e], s[i][0][e + 1], s[i][1][e]), s[i][1][e + 1]) * f[i][hh];
                    const float mx = fmaxf(top[0][hh], top[1][hh]), w = fmaxf(top[0][hh] + lv[0], top[1][hh] + lv[1]);
                    rise |= mx > m[hh] + kLag || w > m[hh] + d[hh] + kLag;
                    huge |= fabsf(mx) > 65536.f && mx > -INFINITY;
                }
                // The exponents below add a page's log2 vs - d to -m, which past 2^16 would lose bits of
                // it, and -m to an unrounded product: such scores are rounded and made relative to m first.
                huge = __any_sync(0xffffffffu, huge);
                if (huge || __any_sync(0xffffffffu, rise)) {
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        float mx = fmaxf(top[0][hh], top[1][hh]), w = fmaxf(top[0][hh] + lv[0], top[1][hh] + lv[1]);
#pragma unroll
                        for (int x = 1; x <= 2; x *= 2) {
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                            w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, x));
                        }
                        // (a row's references move by its own scores alone: its bits do not depend on the
                        // rows beside it)
                        const float mn = mx > m[hh] + kLag ? fmaxf(m[hh], floorf(mx)) : m[hh], mz = finite_or_0(mn);
                        w -= mz;
                        if (__builtin_expect(huge, 0)) {
                            w = fmaxf((top[0][hh] - mz) + lv[0], (top[1][hh] - mz) + lv[1]);
                            w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 1));
                            w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 2));
                        }
                        const float dm = m[hh] - mz, dd = d[hh] + dm;  // first keys: -inf
                        const float dn = w > dd + kLag ? fmaxf(dd, floorf(w)) : dd;
                        const float fo = dn == -INFINITY ? 1.f : ex2(dd - dn);
                        m[hh] = mn, d[hh] = dn;
                        base[hh] = kProbBits - mz, dz[hh] = finite_or_0(dn);
                        l[hh] *= ex2(dm);
#pragma unroll
                        for (int n = 0; n < 16; ++n) o[n][2 * hh] *= fo, o[n][2 * hh + 1] *= fo;
                        if (__builtin_expect(huge, 0))
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
#pragma unroll
                                for (int t = 0; t < 2; ++t)
#pragma unroll
                                    for (int j = 2 * hh; j < 2 * hh + 2; ++j)
                                        s[i][t][j] = __fmul_rn(s[i][t][j], f[i][hh]) - mz;
                                f[i][hh] = 1.f;
                            }
                    }
                }
                uint32_t pa[2][4];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    const float at = huge ? kProbBits : base[hh];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float lr = fmaxf(lv[i] - dz[hh], kLogFloor);
                        const uint64_t ff = f2_pack(f[i][hh], f[i][hh]), cc = f2_pack(at + lr, at + lr);
                        float2 x[2];
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            x[t] = f2_unpack(f2_fma(f2_pack(s[i][t][2 * hh], s[i][t][2 * hh + 1]), ff, cc));
                            x[t].x = ex2(x[t].x), x[t].y = ex2(x[t].y);
                            pa[i][2 * t + hh] = pack_f16(x[t].x, x[t].y);
                        }
                        l[hh] = fmaf((x[0].x + x[0].y) + (x[1].x + x[1].y), ex2(-lr), l[hh]);
                    }
                }
                // ---- O += P V8 ----
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint4 w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = lds128(vb + i * page_bytes + (k >> 1) * 1024 + (k & 1 ? v_off1 : v_off));
                    if (masked) {  // bytes of keys that no row sees may be NaN codes: P = 0 there
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (key0[i] + 2 * c4 + (k & 1) + 8 * (k >> 1) > pmax || !((valid >> i) & 1u))
                                w[k] = make_uint4(0u, 0u, 0u, 0u);
                    }
                    const uint32_t a[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, b[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
                    const uint32_t c[4] = {w[2].x, w[2].y, w[2].z, w[2].w}, d[4] = {w[3].x, w[3].y, w[3].z, w[3].w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const uint32_t ab0 = __byte_perm(a[n], b[n], 0x5140), ab1 = __byte_perm(a[n], b[n], 0x7362);
                        const uint32_t cd0 = __byte_perm(c[n], d[n], 0x5140), cd1 = __byte_perm(c[n], d[n], 0x7362);
                        mma_f16(o[4 * n], pa[i], e4m3x2_to_f16x2(ab0), e4m3x2_to_f16x2(cd0));
                        mma_f16(o[4 * n + 1], pa[i], e4m3x2hi_to_f16x2(ab0), e4m3x2hi_to_f16x2(cd0));
                        mma_f16(o[4 * n + 2], pa[i], e4m3x2_to_f16x2(ab1), e4m3x2_to_f16x2(cd1));
                        mma_f16(o[4 * n + 3], pa[i], e4m3x2hi_to_f16x2(ab1), e4m3x2hi_to_f16x2(cd1));
                    }
                }
            }
            // the segment's last stage stays held: the warps that share its rows meet there
            if (x + 1 < seg1 || p.kw == 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[st]);
            }
        }
        if (!ok) break;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
            l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
            // O in its own units: a convex combination of the values
            const OutScale os = out_scale(d[hh], l[hh]);
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n][2 * hh] *= os.f, o[n][2 * hh + 1] *= os.f;
            if (__any_sync(0xffffffffu, os.g != 1.f))
#pragma unroll
                for (int n = 0; n < 16; ++n) o[n][2 * hh] *= os.g, o[n][2 * hh + 1] *= os.g;
        }
        if (p.kw > 1) {
            // The kw warps of each (head, tile) hold different pages' shares.  They leave them in
            // shared memory (the last stage's, which has room for one row tile and is free once all
            // have read it; with more tiles, or a single segment and so no need of a long ring, in a
            // buffer behind the ring) and each finishes every kw-th row.  16-byte chunk 8 c + i of
            // a row lies at 8 c + (i ^ (c | (row & 1) << 2)): free of bank conflicts both ways.
            const int st = (done - 1) % p.stages;
            const bool own_buf = p.ch > 1 || p.whole;
            float *buf = reinterpret_cast<float *>(smem + (size_t)(own_buf ? p.stages : st) * stage_bytes) +
                         (size_t)(h_of * p.ch + c_of) * p.kw * 16 * kHD;
            if (!own_buf) ok = meet();  // every warp has read the stage
            if (!ok) break;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int r = g4 + 8 * hh;
                float *row = buf + (k_of * 16 + r) * kHD;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = 2 * hh + (i >> 2), n = 4 * (i & 3);
                    *reinterpret_cast<float4 *>(row + 4 * (8 * c4 + (i ^ (c4 | (r & 1) << 2)))) =
                        make_float4(o[n][e], o[n + 1][e], o[n + 2][e], o[n + 3][e]);
                }
                if (c4 == 0) s_ml[segs & 1][warp][r] = make_float2(m[hh], l[hh]);
            }
            ok = meet();
            if (!ok) break;
            if (active)
                for (int r = k_of; r < tile1 - tile0; r += p.kw) {
                    Joined sum;
                    float m2[kTokWarps], l2[kTokWarps];
                    float4 o2[kTokWarps];
#pragma unroll
                    for (int k = 0; k < kTokWarps; ++k) {
                        m2[k] = -INFINITY, l2[k] = 0.f, o2[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (k < p.kw) {
                            const float2 ml = s_ml[segs & 1][warp - k_of + k][r];
                            m2[k] = ml.x, l2[k] = ml.y;
                            o2[k] = *reinterpret_cast<const float4 *>(
                                buf + (k * 16 + r) * kHD + 4 * ((lane & 24) + ((lane & 7) ^ (lane >> 3 | (r & 1) << 2))));
                        }
                    }
                    sum.add(m2, l2, o2);
                    const int rho = tile0 + r;
                    if (whole) {
                        finish4(p.out, p.gate, ((size_t)(g.q0 + rho / p.geo.gsz) * p.nh + head * p.geo.gsz + rho % p.geo.gsz) * kHD + 4 * lane, sum.o);
                    } else {
                        float *rec = p.part + ((((size_t)blockIdx.y * p.G + cta) * 2 + slot) * p.hg * p.rpg +
                                               (size_t)h_of * p.rpg + rho) * kRec;
                        *reinterpret_cast<float4 *>(rec + 4 * lane) = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
                        if (lane == 0) rec[kHD] = sum.m, rec[kHD + 1] = sum.l;
                    }
                }
            if (p.ch > 1 && !p.whole) ok = meet();  // before the buffer's next use
            // reads and writes here come before the copies into this stage
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[st]);
            continue;
        }
        if (!active) continue;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const int rho = tile0 + g4 + 8 * hh;
            if (rho >= tile1) continue;
            if (whole) {
                const size_t ob = ((size_t)(g.q0 + rho / p.geo.gsz) * p.nh + head * p.geo.gsz + rho % p.geo.gsz) * kHD;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const size_t at = ob + 32 * c4 + 16 * half + 8 * i;
                        float e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) e[j] = o[8 * i + j][2 * hh + half];
                        if (p.gate) apply_gate(e, p.gate + at);
                        store8(p.out + at, e);
                    }
            } else {
                float *rec = p.part + ((((size_t)blockIdx.y * p.G + cta) * 2 + slot) * p.hg * p.rpg +
                                       (size_t)h_of * p.rpg + rho) * kRec;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4 *>(rec + 32 * c4 + 16 * half + 4 * i) =
                            make_float4(o[4 * i][2 * hh + half], o[4 * i + 1][2 * hh + half],
                                        o[4 * i + 2][2 * hh + half], o[4 * i + 3][2 * hh + half]);
                if (c4 == 0) rec[kHD] = m[hh], rec[kHD + 1] = l[hh];
            }
        }
    }
}

// Combines the partials that CTA range boundaries cut.  A block's WPB warps take one (row, query
// head) each, or wpi of them share one's partials (many CTAs on one sequence) and join through
// shared memory; U partials in flight per warp, lane l takes dims 4l .. 4l + 3.  The shares follow
// from the contexts, which the token kernel only reads: for up to kMergeScan groups they are worked
// out before the wait for it, and one round of loads remains.
template <int WPB, int U>
__global__ void __launch_bounds__(WPB * 32) kv8_attn_merge(const TokParams p, int wpi) {
    __shared__ __align__(16) float s_o[WPB][kHD];
    __shared__ float s_ml[WPB][2];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % wpi;
    const int per = WPB / wpi, hb = (p.nh + per - 1) / per;
    const int head = blockIdx.x % hb * per + warp / wpi;
    const int j = blockIdx.x / hb, b = blockIdx.y;
    const int q0 = p.geo.cu_q[b], q_len = p.geo.cu_q[b + 1] - q0;
    const bool in = head < p.nh && j < q_len;
    const int kvh = in ? head / p.geo.gsz : 0, rho = j * p.geo.gsz + (in ? head % p.geo.gsz : 0);
    int T = 0, P0 = 0, P1 = 0;
    if (p.groups <= kMergeScan) {
        for (int v0 = 0; v0 < p.groups; v0 += 32) {
            const int x = v0 + lane, n = x < p.groups ? (group_of(p.geo, p.rpg, x).nv + p.pps - 1) / p.pps : 0;
            T += __reduce_add_sync(0xffffffffu, n);
            P0 += __reduce_add_sync(0xffffffffu, x < b ? n : 0);
            P1 += __reduce_add_sync(0xffffffffu, x <= b ? n : 0);
        }
    } else {
        pdl_wait();
        T = p.prefix_out[p.groups], P0 = p.prefix_out[b], P1 = p.prefix_out[b + 1];
    }
    int c0 = 0, c1 = -1;
    if (in && P1 > P0) {
        const int c = cta_of(lane == 0 ? P0 : P1 - 1, T, p.G);
        c0 = __shfl_sync(0xffffffffu, c, 0), c1 = __shfl_sync(0xffffffffu, c, 1);
    }
    pdl_wait();
    const bool cut = c1 > c0;  // else its one CTA wrote the output
    const size_t rows = (size_t)p.hg * p.rpg;
    const float *base = p.part + ((size_t)(kvh / p.hg) * p.G * 2) * rows * kRec +
                        ((size_t)(kvh % p.hg) * p.rpg + rho) * kRec;
    Joined sum;
    if (cut)
        for (int cb = c0 + sub * U; cb <= c1; cb += wpi * U) {
            float m[U], l[U];
            float4 o[U];
            // lane u: the slot of CTA cb + u's partial (0 where the group starts in its range or
            // fills its beginning), or none where its range is empty
            int sl = -1;
            if (lane < U && cb + lane <= c1) {
                const int lo = share_of(cb + lane, T, p.G), hi = share_of(cb + lane + 1, T, p.G);
                if (hi > lo) sl = lo >= P0 ? 0 : 1;
            }
            // unconditional loads (of the group's first partial where there is none): all in flight
            float4 ml[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int slot = __shfl_sync(0xffffffffu, sl, u);
                const float *rec = base + ((size_t)(slot < 0 ? c0 : cb + u) * 2 + max(slot, 0)) * rows * kRec;
                ml[u] = __ldcg(reinterpret_cast<const float4 *>(rec + kHD));
                o[u] = __ldcg(reinterpret_cast<const float4 *>(rec + 4 * lane));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool none = __shfl_sync(0xffffffffu, sl, u) < 0;
                m[u] = none ? -INFINITY : ml[u].x, l[u] = none ? 0.f : ml[u].y;
                if (none) o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            sum.add(m, l, o);
        }
    if (wpi > 1) {
        *reinterpret_cast<float4 *>(&s_o[warp][4 * lane]) = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
        if (lane == 0) s_ml[warp][0] = sum.m, s_ml[warp][1] = sum.l;
        __syncthreads();
        if (sub) return;
        float m[WPB - 1], l[WPB - 1];  // the others' sums
        float4 o[WPB - 1];
#pragma unroll
        for (int u = 0; u < WPB - 1; ++u) {
            const int at = warp + min(u + 1, wpi - 1);
            m[u] = u + 1 < wpi ? s_ml[at][0] : -INFINITY, l[u] = u + 1 < wpi ? s_ml[at][1] : 0.f;
            o[u] = *reinterpret_cast<const float4 *>(&s_o[at][4 * lane]);
        }
        sum.add(m, l, o);
    }
    if (!cut) return;
    const size_t ob = ((size_t)(q0 + j) * p.nh + head) * kHD + 4 * lane;
    finish4(p.out, p.gate, ob, sum.o);
}

// ---------------------------------------------------------------------------------
// Chunk kernel: prompts and other calls with many rows per KV head, bound by the tensor cores.
//
// A CTA owns 256 rows (two tiles of 128) of one KV head of one sequence and a share of the pages that
// they see, in blocks of eight (128 keys): with a window, the sinks' pages and the window's follow
// one another in a block.  Four converter warps read a block's codes from the cache, write them to shared
// memory as f16 (K and V each into two 32 KB stages; the code-to-f16 step is shared by both tiles),
// and one thread issues, per block and tile,
//   S = Q K8^T    8 x tcgen05.mma M=128 N=128 K=16 (kind::f16), both operands in shared memory
//   O += P V8     8 x the same, P from TMEM, V as it lies (keys x dims, an MN-major operand)
// Two groups of four softmax warps, a thread per row, turn S into P in place (P's 64 columns lie
// over S's 128), so S, P and O of both tiles fill the 512 TMEM columns, and while one tile's
// softmax runs the tensor cores work on the other tile.  The softmax takes the row maximum page by
// page on the raw products (a page's scale is one factor) and folds the page's V scale into the
// exponent: p' = 2^(s f + c), c = bits - m + log2 vs - d, one fma and one exp2 per score.
// Register split of the 512 threads (128 each at launch, 65536): 176 for the softmax warps, 120 for
// the converters, 40 for the issuer's group: 256 * 176 + 128 * 120 + 128 * 40 = 65536.  (With fewer the
// converters spill, and a spilled load in flight waits for itself.)
//
// Measured: two prompts of 4096 rows, 32 + 8 heads: 275 us, 737 TFLOP/s (the products alone at the
// card's f16 rate: 118); 8192 rows through a 1024-key window with 4 sinks 231 us, 560 TFLOP/s.  A
// block of both tiles takes 2.0 to 2.4 us, of which the tensor cores work 1.5 (an M = 128, N = 128
// product takes 88 cycles of the ideal 64) and the exponentials 1.04; a tile's next scores wait for its
// P to be used: with two tiles TMEM is full (a CTA with one tile takes the same turns, although the
// other's columns are idle).  A CTA's first scores come 6 us after its start, its last stores 4 us
// after the last P.
// Measured and left out: 64-key blocks with two score buffers (349 us: N = 64 products cost nearly what N = 128
// ones do, twice the hand-overs), 16 softmax warps (348), scores held in registers, and blocks that take over
// the next group as they finish (355: more registers than there are).
// ---------------------------------------------------------------------------------
constexpr int kChThreads = 512;
constexpr int kChTile = 128, kChRows = 2 * kChTile;  // rows per tile and per CTA
constexpr int kChKeys = 128, kChPages = kChKeys / kKv8Page;  // keys and pages per block
constexpr int kChHalf = kChKeys * 128;               // 64 dims of a 128-row f16 operand: 16 KB
constexpr int kChOperand = 2 * kChHalf;              // 32 KB
constexpr size_t kChSmemK = 2 * (size_t)kChOperand, kChSmemV = kChSmemK + 2 * (size_t)kChOperand;
constexpr size_t kChSmem = kChSmemV + 2 * (size_t)kChOperand + 1024;
constexpr int kChScales = 4;  // blocks whose scales are kept: the softmax may be two behind the copies

struct ChunkParams {
    Geometry geo;
    const __nv_bfloat16 *q, *gate;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *block_table;
    __nv_bfloat16 *out;
    float *part;  // [splits][total_q][nh][kRec], when splits > 1
    int nh, nkv, max_blocks, num_blocks, total_q, rgs, splits;  // rgs: groups of kChRows rows per sequence
    uint32_t wait_limit;
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// SWIZZLE_128B operand, 1024 bytes between groups of 8 rows (of 8 keys, for the MN-major V).  The
// upper word of its descriptor is constant; the lower one holds the address / 16 and, for V, the
// distance / 16 of the two halves of the dims.  An operand's next 16 columns (or keys) are an
// addition to the lower word, so the issuing thread spends a few instructions per MMA.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tc_desc(uint32_t saddr, uint32_t lead) { return ((saddr & 0x3FFFF) >> 4) | (lead << 16); }
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// the lowest n of 16 bits, none for n <= 0, all for n >= 16
__device__ __forceinline__ uint32_t low16(int n) { return (1u << min(max(n, 0), 16)) - 1u; }
// the largest of 16 floats
__device__ __forceinline__ float max16(const uint32_t *s) {
    float a = max3(__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[2]));
    float b = max3(__uint_as_float(s[3]), __uint_as_float(s[4]), __uint_as_float(s[5]));
    float c = max3(__uint_as_float(s[6]), __uint_as_float(s[7]), __uint_as_float(s[8]));
    float d = max3(__uint_as_float(s[9]), __uint_as_float(s[10]), __uint_as_float(s[11]));
    a = max3(a, __uint_as_float(s[12]), __uint_as_float(s[13]));
    b = max3(b, __uint_as_float(s[14]), __uint_as_float(s[15]));
    return fmaxf(max3(a, b, c), d);
}
struct __align__(8) ChunkBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], o_done[2], drain;
};

// grid: groups of rows (the last first) x sequences x KV heads x splits
__global__ void __launch_bounds__(kChThreads, 1) kv8_attn_chunk(const ChunkParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ ChunkBars bar;
    __shared__ __align__(16) float s_scale[kChScales][2][8];  // [block][K scale, log2 of the V scale][page]
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.k_full[i], 4);
            mbar_init(&bar.k_empty[i], 1);
            mbar_init(&bar.v_full[i], 4);
            mbar_init(&bar.v_empty[i], 1);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i][0], 4);
            mbar_init(&bar.p_full[i][1], 4);
            mbar_init(&bar.o_done[i], 1);
        }
        mbar_init(&bar.drain, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_wait();

    // the last positions see the most keys: their groups first
    const int per = (int)gridDim.x / p.rgs, rg = p.rgs - 1 - blockIdx.x / per, in_rg = blockIdx.x % per;
    const int split = in_rg % p.splits, kvh = in_rg / p.splits % p.nkv, b = in_rg / (p.splits * p.nkv);
    const int q0 = p.geo.cu_q[b], q_len = p.geo.cu_q[b + 1] - q0, ctx = p.geo.ctx[b];
    const int gsz = p.geo.gsz, p0 = ctx - q_len;
    const int rho0 = rg * kChRows, rho1 = min(q_len * gsz, rho0 + kChRows);
    const int tiles = rho1 - rho0 > kChTile ? 2 : (rho1 > rho0 ? 1 : 0);
    // the group's pages: n_sink from the sequence's first on, then those from lo_page on, nv in all;
    // block j holds the pages 8 j .. 8 j + 7 of this list
    int n_sink = 0, lo_page = 0, nv = 0;
    if (tiles > 0) {
        const int pmin = p0 + rho0 / gsz, pmax = p0 + (rho1 - 1) / gsz;
        if (pmax >= 0) {
            if (p.geo.window > 0) {
                lo_page = max(0, pmin - p.geo.window + 1) / kKv8Page;
                n_sink = min((p.geo.sinks + kKv8Page - 1) / kKv8Page, lo_page);
            }
            nv = n_sink + pmax / kKv8Page + 1 - lo_page;
        }
    }
    const int nb = (nv + kChPages - 1) / kChPages;
    const int j0 = (int)((long long)nb * split / p.splits), j1 = (int)((long long)nb * (split + 1) / p.splits);
    auto key_of = [&](int i) { return (i < n_sink ? i : i - n_sink + lo_page) * kKv8Page; };  // page i's first
    // a wait of the whole warp; false once any lane gave up
    auto wait = [&](uint64_t *m, uint32_t parity) {
        const bool ok = __all_sync(0xffffffffu, mbar_wait(m, parity, &s_abort, p.wait_limit));
        if (!ok) *(volatile int *)&s_abort = 1;
        return ok;
    };

    if (warp >= 12) {
        // ---- issuer ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 12 && j0 < j1) {
            const uint32_t idesc_s = (1u << 4) | ((uint32_t)(kChKeys >> 3) << 17) | ((uint32_t)(kChTile >> 4) << 24);
            const uint32_t idesc_pv = idesc_s | (1u << 16);  // B MN-major
            const uint32_t base = smem_u32(smem);
            auto issue_s = [&](int t, int n) {  // block n of this CTA
                if (lane == 0) {
                    const uint32_t qa = tc_desc(base + t * kChOperand, 1);
                    const uint32_t ka = tc_desc(base + (uint32_t)kChSmemK + (n & 1) * kChOperand, 1);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        tc_mma_ss(tmem + 128 * t, qa + (k >> 2) * (kChHalf >> 4) + 2 * (k & 3),
                                  ka + (k >> 2) * (kChHalf >> 4) + 2 * (k & 3), idesc_s, k > 0 ? 1u : 0u);
                    tc_commit(&bar.s_full[t]);
                    if (t == tiles - 1) tc_commit(&bar.k_empty[n & 1]);
                }
                __syncwarp();
            };
            const int total = j1 - j0;
            bool ok = wait(&bar.q_full, 0) && wait(&bar.k_full[0], 0);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < tiles; ++t) issue_s(t, 0);
            }
            for (int n = 0; ok && n < total; ++n) {
                ok = wait(&bar.v_full[n & 1], (uint32_t)(n >> 1) & 1u);
                for (int t = 0; ok && t < tiles; ++t) {
                    ok = wait(&bar.p_full[t][0], (uint32_t)n & 1u);
                    if (ok && n + 1 < total && t == 0) ok = wait(&bar.k_full[(n + 1) & 1], (uint32_t)((n + 1) >> 1) & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t va = tc_desc(base + (uint32_t)kChSmemV + (n & 1) * kChOperand, kChHalf >> 4);
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // 16 keys: 8 columns of P, 16 rows of V
                            tc_mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, va + k * (2048 >> 4),
                                      idesc_pv, n > 0 || k > 0 ? 1u : 0u);
                    }
                    __syncwarp();
                    ok = wait(&bar.p_full[t][1], (uint32_t)n & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t va = tc_desc(base + (uint32_t)kChSmemV + (n & 1) * kChOperand, kChHalf >> 4);
#pragma unroll
                        for (int k = 4; k < 8; ++k)  // 16 keys: 8 columns of P, 16 rows of V
                            tc_mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, va + k * (2048 >> 4),
                                      idesc_pv, n > 0 || k > 0 ? 1u : 0u);
                        if (t == tiles - 1) tc_commit(&bar.v_empty[n & 1]);
                        if (n + 1 == total) tc_commit(&bar.o_done[t]);
                    }
                    __syncwarp();
                    if (n + 1 < total) issue_s(t, n + 1);  // after PV: S lies over P
                }
            }
            // everything issued has completed (also when a wait gave up)
            if (lane == 0) tc_commit(&bar.drain);
            __syncwarp();
            mbar_drain(&bar.drain, 0);
            if (!ok && lane == 0) atomicExch(&g_kv8_error, 1);
            __syncwarp();
        }
    } else if (warp >= 8) {
        // ---- converters: thread (row, ch) takes 16 codes of token `row` of each of a block's pages ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        // Eight lanes (a phase of 16-byte accesses) have one half of two neighbouring rows, whose swizzle
        // puts their chunks on all banks.
        const int row = 4 * (warp - 8) + (lane >> 2 & 1) + 2 * (lane >> 4), ch = (lane & 3) | (lane >> 1 & 4);
        // page ids of block j: lane i holds page i's
        auto fetch_ids = [&](int j) {
            int blk = -1;
            if (j < j1 && lane < 8) {
                const int i = j * kChPages + lane, pg = key_of(i) / kKv8Page;
                if (i < nv && pg < p.max_blocks && pg * kKv8Page < ctx) blk = p.block_table[(size_t)b * p.max_blocks + pg];
                if (blk < 0 || blk >= p.num_blocks) blk = -1;
            }
            return blk;
        };
        // unconditional loads (of page 0 where there is none), so that all eight are in flight;
        // what must not count is zeroed when it is converted
        auto fetch = [&](const uint8_t *cache, int ids, uint4 (&r)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int blk = max(__shfl_sync(0xffffffffu, ids, i), 0);
                r[i] = ldg_nc_v4(cache + (((size_t)blk * kKv8Page + row) * p.nkv + kvh) * kHD + 16 * ch);
            }
        };
        // dims 16 ch ..: two 16-byte chunks of the half ch / 4
        const uint32_t dst0 = (ch >> 2) * kChHalf + row * 128 + ((2 * (ch & 3) ^ (row & 7)) << 4), dst1 = dst0 ^ 16u;
        // live: bit i: this thread's token of page i counts (the page has a valid id, the token is one
        // of the context's)
        auto convert = [&](uint32_t at, uint32_t live, const uint4 (&r)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
                if (live != 0xffu && !((live >> i) & 1u)) w[0] = w[1] = w[2] = w[3] = 0u;
                const uint32_t x[4] = {e4m3x2_to_f16x2(w[0]), e4m3x2hi_to_f16x2(w[0]), e4m3x2_to_f16x2(w[1]), e4m3x2hi_to_f16x2(w[1])};
                const uint32_t y[4] = {e4m3x2_to_f16x2(w[2]), e4m3x2hi_to_f16x2(w[2]), e4m3x2_to_f16x2(w[3]), e4m3x2hi_to_f16x2(w[3])};
                sts128(at + i * 2048 + dst0, x);
                sts128(at + i * 2048 + dst1, y);
            }
        };
        auto publish = [&](uint64_t *m) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(m);
        };
        const uint32_t base = smem_u32(smem);
        uint4 kr[8], vr[8];
        int ids = fetch_ids(j0);
        fetch(p.kc, ids, kr);
        fetch(p.vc, ids, vr);
        bool ok = true;
        for (int j = j0, n = 0; j < j1 && ok; ++j, ++n) {
            const int st = n & 1;
            const uint32_t parity = (uint32_t)((n >> 1) - 1) & 1u;
            // scales of the block's pages (warp 8: lanes 0..7 K, 8..15 log2 of V); zero without a valid id
            float sc = 0.f;
            const bool cut = key_of(j * kChPages + lane) + kKv8Page > ctx;  // the context ends in the page
            uint32_t live = __ballot_sync(0xffffffffu, ids >= 0 && !cut);
            const uint32_t last = __ballot_sync(0xffffffffu, ids >= 0 && cut);
            if (row < (ctx & (kKv8Page - 1))) live |= last;
            if (warp == 8) {
                const int blk = __shfl_sync(0xffffffffu, ids, lane & 7);
                sc = (lane < 8 ? p.ks : p.vs)[(size_t)max(blk, 0) * p.nkv + kvh];
                if (blk < 0) sc = 0.f;
                if (lane >= 8) sc = log2_scale(sc);
            }
            const int next = fetch_ids(j + 1);
            if (n >= 2) ok = wait(&bar.k_empty[st], parity);
            if (!ok) break;
            if (warp == 8 && lane < 16) s_scale[n % kChScales][lane >> 3][lane & 7] = sc;
            convert(base + (uint32_t)kChSmemK + st * kChOperand, live, kr);
            publish(&bar.k_full[st]);
            fetch(p.kc, next, kr);
            if (n >= 2) ok = wait(&bar.v_empty[st], parity);
            if (!ok) break;
            convert(base + (uint32_t)kChSmemV + st * kChOperand, live, vr);
            publish(&bar.v_full[st]);
            fetch(p.vc, next, vr);
            ids = next;
        }
    } else {
        // ---- softmax: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const int t = warp >> 2, r = threadIdx.x & 127;
        const int rho = rho0 + t * kChTile + r;
        const bool in = rho < rho1;
        const size_t qrow = ((size_t)(q0 + (in ? rho / gsz : 0)) * p.nh + (size_t)kvh * gsz + (in ? rho % gsz : 0));
        const int qp = in ? p0 + rho / gsz : -1;
        float rowf;
        {   // the row in f16 as q * 2^k, its largest magnitude in [2^14, 2^15), into the Q operand
            uint4 w[16];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = in ? *reinterpret_cast<const uint4 *>(p.q + qrow * kHD + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t wd[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(wd[k] << 16)), fabsf(__uint_as_float(wd[k] & 0xffff0000u))));
            }
            int sh = 14 - ((int)(__float_as_uint(mx) >> 23) - 127);
            sh = sh > 126 ? 126 : sh;
            const float up = pow2f(sh);
            rowf = pow2f(-sh) * kScoreScale;
            const uint32_t dst = smem_u32(smem) + t * kChOperand + r * 128;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t wd[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                uint32_t h[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    h[k] = pack_f16(__uint_as_float(wd[k] << 16) * up, __uint_as_float(wd[k] & 0xffff0000u) * up);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (i >> 3) * kChHalf +
                                                                             (((i & 7) ^ (r & 7)) << 4)),
                             "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3])
                             : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.q_full);
        }
        float m = -INFINITY, d = -INFINITY, l = 0.f;
        bool ok = true;
        if (t < tiles) {
            // positions of the warp's rows: pages [plain0, plain1) of the list, which all of them see
            // whole, need no mask
            const int w0 = rho0 + t * kChTile + (warp & 3) * 32, w1 = min(rho1, w0 + 32) - 1;
            const int pmin = p0 + w0 / gsz, pmax = p0 + (w1 >= w0 ? w1 : w0) / gsz;
            int plain0 = 0, plain1 = max(pmin + 1, 0) / kKv8Page;
            if (p.geo.window > 0) {
                plain0 = n_sink + max(0, (max(0, pmax - p.geo.window + 1) + kKv8Page - 1) / kKv8Page - lo_page);
                plain1 += n_sink - lo_page;
            }
            const uint32_t s_at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 128 * t, o_at = s_at + 256;
            for (int j = j0, n = 0; j < j1; ++j, ++n) {
                ok = wait(&bar.s_full[t], (uint32_t)n & 1u);
                if (!ok) break;
                tc_fence_after();
                float f[8], lv[8];
                {
                    const float *sc = &s_scale[n % kChScales][0][0];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = rowf * sc[i], lv[i] = sc[8 + i];
                }
                const bool plain = j * kChPages >= plain0 && (j + 1) * kChPages <= plain1;
                if (!plain) {
                    // in pages that some row does not see whole, which at 128 keys a block are few, the
                    // others' scores become -inf, which must not meet a factor of 0 (with the least
                    // normal number in its place a product is still nothing beside the exponents)
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) {
                        const int at = j * kChPages + i, k0 = key_of(at);
                        if (at >= plain0 && at < plain1) continue;
                        uint32_t s[16], see = at < nv ? low16(qp + 1 - k0) : 0u;
                        if (p.geo.window) see &= ~low16(qp - p.geo.window + 1 - k0) | low16(p.geo.sinks - k0);
                        tc_ld16(s_at + 16 * i, s);
                        tc_ld_wait();
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (!((see >> k) & 1u)) s[k] = 0xff800000u;
                        tc_st16(s_at + 16 * i, s);
                    }
                    tc_st_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = fmaxf(f[i], 1.17549435e-38f);
                }
                float mx = -INFINITY, top = -INFINITY;  // of s and s + log2 vs, page by page on the raw products
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t s[64];
                    tc_ld32(s_at + 64 * c, s);
                    tc_ld32(s_at + 64 * c + 32, s + 32);
                    tc_ld_wait();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = max16(s + 16 * i) * f[4 * c + i];
                        mx = fmaxf(mx, a), top = fmaxf(top, a + lv[4 * c + i]);
                    }
                }
                // The exponents below add a page's log2 vs - d to -m, which past 2^16 would lose bits of
                // it, and -m to an unrounded product: such scores are rounded and made relative to m first.
                const bool huge = __any_sync(0xffffffffu, fabsf(mx) > 65536.f && mx > -INFINITY);
                if (huge || __any_sync(0xffffffffu, mx > m + kLag || top > m + d + kLag)) {
                    // (all rows of the warp move where one has to, which they will have to anyway: 275 us for
                    // two 4K prompts, 280 where each moves by its own scores alone, as in the token kernel)
                    const float mn = fmaxf(m, floorf(mx)), mz = finite_or_0(mn);
                    float w = top - mz;
                    if (huge) {
                        w = -INFINITY;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t s[32];
                            tc_ld32(s_at + 32 * c, s);
                            tc_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                s[i] = __float_as_uint(__fmul_rn(__uint_as_float(s[i]), f[2 * c + (i >> 4)]) - mz);
                            w = max3(w, max16(s) + lv[2 * c], max16(s + 16) + lv[2 * c + 1]);
                            tc_st32(s_at + 32 * c, s);
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = 1.f;
                        tc_st_wait();
                    }
                    // s_full of this block came after the products of the last one: O is complete
                    const float dm = m - mz, dd = d + dm, dn = fmaxf(dd, floor_2m14(w));  // first keys: dm, dd = -inf
                    const float fo = dn == -INFINITY ? 1.f : ex2(dd - dn);
                    m = mn, d = dn;
                    l *= ex2(dm);
                    if (n > 0) {
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            uint32_t u[16];
                            tc_ld16(o_at + 16 * c, u);
                            tc_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(__uint_as_float(u[k]) * fo);
                            tc_st16(o_at + 16 * c, u);
                        }
                    }
                }
                const float base = huge ? kProbBits : kProbBits - finite_or_0(m), dz = finite_or_0(d);
                // P over S, 32 scores at a time (their 16 columns of P lie over columns read before):
                // two scores per fma, the sum of a page's with its V scale taken out again
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t s[32], h[16];
                    tc_ld32(s_at + 32 * c, s);
                    tc_ld_wait();
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float lr = fmaxf(lv[2 * c + i] - dz, kLogFloor);
                        const uint64_t ff = f2_pack(f[2 * c + i], f[2 * c + i]), cc = f2_pack(base + lr, base + lr);
                        uint64_t sum = 0ull;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint32_t *x2 = s + 16 * i + 2 * k;
                            float2 x = f2_unpack(f2_fma((uint64_t)x2[0] | ((uint64_t)x2[1] << 32), ff, cc));
                            x.x = ex2(x.x), x.y = ex2(x.y);
                            sum = f2_add(sum, f2_pack(x.x, x.y));
                            h[8 * i + k] = pack_f16(x.x, x.y);
                        }
                        const float2 y = f2_unpack(sum);
                        l = fmaf(y.x + y.y, ex2(-lr), l);
                    }
                    tc_st16(s_at + 16 * c, h);
                    if (c & 1) {
                        tc_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.p_full[t][c >> 1]);
                    }
                }
            }
            if (ok && j0 < j1) ok = wait(&bar.o_done[t], 0);
            if (ok) {
                tc_fence_after();
                const OutScale os = out_scale(d, l);
                const size_t ob = qrow * kHD;
                float *rec = p.splits > 1 ? p.part + ((size_t)split * p.total_q * p.nh + qrow) * kRec : nullptr;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t u[32];
                    __syncwarp();
                    if (j0 < j1) {
                        tc_ld32(o_at + 32 * c, u);
                        tc_ld_wait();
                    }
                    if (!in) continue;
#pragma unroll
                    for (int k = 0; k < 32; ++k) u[k] = j0 < j1 ? __float_as_uint(__uint_as_float(u[k]) * os.f) : 0u;
                    if (os.g != 1.f)
#pragma unroll
                        for (int k = 0; k < 32; ++k) u[k] = __float_as_uint(__uint_as_float(u[k]) * os.g);
                    if (rec) {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            *reinterpret_cast<uint4 *>(rec + 32 * c + 4 * k) =
                                make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
                        continue;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float e[8];
#pragma unroll
                        for (int x = 0; x < 8; ++x) e[x] = __uint_as_float(u[8 * k + x]);
                        if (p.gate) apply_gate(e, p.gate + ob + 32 * c + 8 * k);
                        store8(p.out + ob + 32 * c + 8 * k, e);
                    }
                }
                if (rec && in) rec[kHD] = m, rec[kHD + 1] = l;
            }
        }
    }
    // ---- teardown ----
    tc_fence_before();
    __syncthreads();
    if (s_abort && threadIdx.x == 0) atomicExch(&g_kv8_error, 1);
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Adds the splits of the chunk kernel.  WPI warps per (row, query head), each over every WPI-th
// split, lane l: dims 4l .. 4l + 3; the first one adds their sums.
template <int WPI>
__global__ void __launch_bounds__(256) kv8_attn_join(const ChunkParams p, int num_seqs) {
    __shared__ float4 s_o[8][32];
    __shared__ float2 s_ml[8];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPI;
    const long long item = (long long)blockIdx.x * (8 / WPI) + warp / WPI;
    // rows of the batch only: those behind the last sequence are not written
    const bool in = item < (long long)p.geo.cu_q[num_seqs] * p.nh && item >= (long long)p.geo.cu_q[0] * p.nh;
    Joined sum;
    float m[4], l[4];
    float4 o[4];
    if (in)
        for (int s = part; s < p.splits; s += 4 * WPI) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool is = s + u * WPI < p.splits;
                const float *rec = p.part + ((size_t)(is ? s + u * WPI : part) * p.total_q * p.nh + item) * kRec;
                const float2 ml = *reinterpret_cast<const float2 *>(rec + kHD);
                m[u] = is ? ml.x : -INFINITY, l[u] = is ? ml.y : 0.f;
                o[u] = is ? *reinterpret_cast<const float4 *>(rec + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            sum.add(m, l, o);
        }
    if (WPI > 1) {
        s_o[warp][lane] = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
        if (lane == 0) s_ml[warp] = make_float2(sum.m, sum.l);
        __syncthreads();
        if (part) return;
        float m7[WPI], l7[WPI];  // the others' sums
        float4 o7[WPI];
        m7[0] = -INFINITY, l7[0] = 0.f, o7[0] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 1; i < WPI; ++i) m7[i] = s_ml[warp + i].x, l7[i] = s_ml[warp + i].y, o7[i] = s_o[warp + i][lane];
        sum.add(m7, l7, o7);
    }
    if (!in) return;
    finish4(p.out, p.gate, (size_t)item * kHD + 4 * lane, sum.o);
}

// ---------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------
long long max_keys(const ekernel_paged_attn_desc_t *d) {  // a larger bound bounds no more: contexts are int32
    return d->max_context < 0x7fffffff ? (long long)d->max_context : 0x7fffffff;
}

struct TokPlan {
    int hg, ngroups, ch, kw, pps, G, whole, stages;
    size_t stage_bytes, smem, part_bytes, prefix_bytes;
};

constexpr size_t kTokSmem = 200 * 1024;  // ring; with the static arrays below the 227 KB of an SM

TokPlan plan_tokens(const ekernel_paged_attn_desc_t *d, size_t window, size_t sinks) {
    TokPlan t;
    const int nkv = (int)d->n_kv_heads, gsz = (int)(d->n_heads / d->n_kv_heads), sms = num_sms();
    const long long max_q = (long long)(d->max_q_len < 1 ? 1 : (d->max_q_len < d->total_q ? d->max_q_len : d->total_q));
    t.ch = (int)(max_q * gsz + 15) / 16;  // 1 or 2 row tiles share the pages that a CTA reads
    long long keys = max_keys(d);
    if (window > 0 && window < (1u << 30) && sinks < (1u << 30)) {
        const long long seen = (long long)window + (long long)sinks + max_q + 32;
        if (seen < keys) keys = seen;
    }
    const long long pages = (keys + 15) / 16, groups = (long long)d->num_seqs;
    auto shape = [&](int heads) {  // KV heads per CTA, the rest of the warps on different pages
        t.ngroups = (nkv + heads - 1) / heads;
        t.hg = (nkv + t.ngroups - 1) / t.ngroups;
        t.kw = kTokWarps / (t.hg * t.ch);
        t.pps = 2 * t.kw;
    };
    // Equal shares of all pages: as many KV heads per CTA as fill the warps (long contiguous reads),
    // one CTA per SM over the head groups, at least one block of pages each.
    shape(kTokWarps / t.ch);
    const long long per = sms / t.ngroups < 1 ? 1 : sms / t.ngroups;
    const long long blocks = groups * ((pages + t.pps - 1) / t.pps);
    t.whole = 0;
    t.G = (int)(blocks < 1 ? 1 : (blocks < per ? blocks : per));
    const long long share = (blocks + t.G - 1) / t.G;
    // Or a CTA for each sequence and as few heads as the SMs allow: no partials, no second launch, whose
    // time is that of about four blocks (measured: 3 us, 0.8 us a block; one row over 301 keys 14.2 us
    // with shares, 8.2 whole; 8 sequences in a 100-key window 18.7 and 7.0).
    for (int heads = 1; heads <= kTokWarps / t.ch; heads *= 2) {
        if (groups * ((nkv + heads - 1) / heads) > sms) continue;
        const TokPlan shares = t;
        shape(heads);
        if ((pages + t.pps - 1) / t.pps <= share + 4) {
            t.whole = 1;
            t.G = (int)groups;
        } else {
            t = shares;
        }
        break;
    }
    t.stage_bytes = (size_t)t.pps * t.hg * 4096;
    const size_t join = t.kw > 1 && (t.ch > 1 || t.whole) ? (size_t)t.hg * t.ch * t.kw * 16 * kHD * sizeof(float) : 0;
    t.stages = (int)((kTokSmem - join) / t.stage_bytes);
    if (t.stages > kTokStages) t.stages = kTokStages;
    t.smem = t.stages * t.stage_bytes + join + 1024;
    t.part_bytes = t.whole ? 0 : (size_t)t.ngroups * t.G * 2 * t.hg * 16 * t.ch * kRec * sizeof(float);
    t.prefix_bytes = (size_t)(kTokGroups + 4) * sizeof(int);
    return t;
}

struct ChunkPlan {
    int rgs, splits;
    long long ctas;
    size_t part_bytes;
};

// Calls of more than 32 rows per KV head run on the chunk kernel.  Its 128-row tiles cost the same
// however few of their rows are used; the token kernel converts the cache anew for every 16-row tile
// and reads it anew for every eight.  Measured (us, token against chunk): 32 sequences over 8K keys,
// 8 KV heads, 32 rows 167 against 239, 40 rows 309 against 240; 24 sequences over 2.5K keys, 2 KV
// heads, 40 rows 31 against 24; one sequence of 40 rows over 8K keys 14.6 against 15.9, which is what a
// rule on rows alone costs there.
constexpr long long kChunkRows = 33;

bool plan_chunks(const ekernel_paged_attn_desc_t *d, size_t window, size_t sinks, ChunkPlan &c) {
    const int gsz = (int)(d->n_heads / d->n_kv_heads);
    const long long max_q = (long long)(d->max_q_len < 1 ? 1 : (d->max_q_len < d->total_q ? d->max_q_len : d->total_q));
    if (max_q * gsz < kChunkRows) return false;
    c.rgs = (int)((max_q * gsz + kChRows - 1) / kChRows);
    const long long ctas = (long long)d->num_seqs * c.rgs * (long long)d->n_kv_heads;
    long long keys = max_keys(d);
    if (window > 0 && window < (1u << 30) && sinks < (1u << 30)) {
        const long long seen = (long long)window + (long long)sinks + max_q + 2 * kChKeys;
        if (seen < keys) keys = seen;
    }
    const long long blocks = (keys + kChKeys - 1) / kChKeys;
    // fewer CTAs than SMs: split the keys as far as one wave of CTAs goes (1000 rows over 8K keys, 2 KV
    // heads: 96 us; one split more, of two waves, 126), at least three blocks each
    long long s = num_sms() / ctas;
    if (s > blocks / 3) s = blocks / 3;
    c.splits = (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
    c.part_bytes = c.splits > 1 ? (size_t)c.splits * d->total_q * d->n_heads * kRec * sizeof(float) : 0;
    c.ctas = ctas * c.splits;
    return true;
}

int encode_pages(const uint8_t *kc, const uint8_t *vc, int nkv, int num_blocks, int hg, CUtensorMap (&maps)[2],
                 const char *what) {
    TensorMapEncodeTiledFn enc = tensor_map_encoder();
    PILM_REQUIRE(enc, ECPU_ERR_UNSUPPORTED, "%s: cuTensorMapEncodeTiled is unavailable", what);
    const uint8_t *src[2] = {kc, vc};
    for (int i = 0; i < 2; ++i) {
        // (dim, slot, head): a box of 128 x 16 x hg lands as [head][slot][128 B], each head's 2 KB
        // a SWIZZLE_128B tile
        cuuint64_t dims[3] = {(cuuint64_t)kHD, (cuuint64_t)num_blocks * kKv8Page, (cuuint64_t)nkv};
        cuuint64_t strides[2] = {(cuuint64_t)nkv * kHD, (cuuint64_t)kHD};
        cuuint32_t box[3] = {(cuuint32_t)kHD, (cuuint32_t)kKv8Page, (cuuint32_t)hg};
        cuuint32_t es[3] = {1, 1, 1};
        const CUresult r = enc(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, (void *)src[i], dims, strides, box, es,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        PILM_REQUIRE(r == CUDA_SUCCESS, ECPU_ERR_PARAM, "%s: the cache's tensor map was rejected (error %d)", what,
                     (int)r);
    }
    return ECPU_OK;
}

int check_error(const char *what) {
    if (!sync_mode() || capturing()) return ECPU_OK;
    int *word = nullptr;
    if (cudaGetSymbolAddress((void **)&word, g_kv8_error) != cudaSuccess) return ECPU_OK;
    return check_error_word_at(word, what, "a wait for a page did not complete");
}

}  // namespace

extern "C" {

size_t ekernel_paged_attention_kv8_workspace_bytes(const ekernel_paged_attn_desc_t *desc, size_t window,
                                                   size_t sinks) {
    if (kv8_check_desc(desc, "ekernel_paged_attention_kv8_workspace_bytes") != ECPU_OK) return 0;
    if (desc->total_q == 0 || desc->num_seqs == 0) return 256;  // nothing to plan; 0 is a refusal
    ChunkPlan c;
    if (plan_chunks(desc, window, sinks, c)) return c.part_bytes + 256;
    const TokPlan t = plan_tokens(desc, window, sinks);
    return t.part_bytes + t.prefix_bytes;
}

int ekernel_paged_attention_verify_kv8(const ekernel_paged_attn_desc_t *desc, const uint16_t *q,
                                       const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scale,
                                       const float *v_scale, const int32_t *block_table, const int32_t *cu_q,
                                       const int32_t *context_lens, const uint16_t *gate, size_t window, size_t sinks,
                                       void *workspace, size_t workspace_bytes, uint16_t *out) {
    const char *what = "ekernel_paged_attention_verify_kv8";
    int rc = kv8_check_desc(desc, what);
    if (rc != ECPU_OK) return rc;
    if (desc->total_q == 0 || desc->num_seqs == 0) return ECPU_OK;
    PILM_REQUIRE(q && k_cache && v_cache && k_scale && v_scale && block_table && cu_q && context_lens && out,
                 ECPU_ERR_PARAM, "%s: null argument", what);
    PILM_REQUIRE(!desc->output_gate || gate, ECPU_ERR_PARAM, "%s: gate required when output_gate", what);
    PILM_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)q | (uintptr_t)out | (uintptr_t)gate) & 15) == 0,
                 ECPU_ERR_PARAM, "%s: the caches, q, gate and out must be 16-byte aligned", what);
    const size_t need = ekernel_paged_attention_kv8_workspace_bytes(desc, window, sinks);
    PILM_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, ECPU_ERR_PARAM,
                 "%s: workspace must be 16-byte aligned and hold %zu bytes, got %zu", what, need, workspace_bytes);
    const size_t cap = 1u << 30;  // positions stay below it: a larger window is none
    Geometry geo;
    geo.cu_q = cu_q;
    geo.ctx = context_lens;
    geo.gsz = (int)(desc->n_heads / desc->n_kv_heads);
    geo.window = window >= cap ? 0 : (int)window;
    geo.sinks = (int)(sinks < cap ? sinks : cap);
    const uint32_t limit = wait_limit_override() >= 0 ? (uint32_t)wait_limit_override() : kWaitLimit;
    ChunkPlan c;
    if (plan_chunks(desc, window, sinks, c)) {
        PILM_REQUIRE(c.ctas <= 0x7fffffffLL, ECPU_ERR_PARAM, "%s: too many rows", what);
        ChunkParams p;
        p.geo = geo;
        p.rgs = c.rgs;
        p.q = (const __nv_bfloat16 *)q;
        p.gate = desc->output_gate ? (const __nv_bfloat16 *)gate : nullptr;
        p.kc = k_cache;
        p.vc = v_cache;
        p.ks = k_scale;
        p.vs = v_scale;
        p.block_table = block_table;
        p.out = (__nv_bfloat16 *)out;
        p.part = (float *)workspace;
        p.nh = (int)desc->n_heads;
        p.nkv = (int)desc->n_kv_heads;
        p.max_blocks = (int)desc->max_blocks_per_seq;
        p.num_blocks = (int)desc->num_blocks;
        p.total_q = (int)desc->total_q;
        p.splits = c.splits;
        p.wait_limit = limit;
        cudaFuncSetAttribute(kv8_attn_chunk, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kChSmem);
        launch_pdl(kv8_attn_chunk, dim3((unsigned)c.ctas), dim3(kChThreads),
                   kChSmem, p);
        rc = check_launch(what);
        if (rc == ECPU_OK) rc = check_error(what);
        if (rc != ECPU_OK || c.splits == 1) return rc;
        const size_t items = desc->total_q * desc->n_heads;
        if (c.splits > 4 && items <= (size_t)num_sms() * 8)  // few rows of many splits: 8 warps share a row's
            launch_pdl(kv8_attn_join<8>, dim3((unsigned)items), dim3(256), 0, p, (int)desc->num_seqs);
        else
            launch_pdl(kv8_attn_join<1>, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, p, (int)desc->num_seqs);
        return check_launch(what);
    }
    const TokPlan t = plan_tokens(desc, window, sinks);
    CUtensorMap maps[2];
    rc = encode_pages(k_cache, v_cache, (int)desc->n_kv_heads, (int)desc->num_blocks, t.hg, maps, what);
    if (rc != ECPU_OK) return rc;
    cudaFuncSetAttribute(kv8_attn_tokens, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kTokSmem + 1024));
    for (size_t b0 = 0; b0 < desc->num_seqs; b0 += (size_t)kTokGroups) {
        const int seqs = (int)(desc->num_seqs - b0 < (size_t)kTokGroups ? desc->num_seqs - b0 : (size_t)kTokGroups);
        TokParams p;
        p.geo = geo;
        p.geo.cu_q += b0;
        p.geo.ctx += b0;
        p.rpg = 16 * t.ch;
        p.q = (const __nv_bfloat16 *)q;
        p.gate = desc->output_gate ? (const __nv_bfloat16 *)gate : nullptr;
        p.ks = k_scale;
        p.vs = v_scale;
        p.block_table = block_table + b0 * desc->max_blocks_per_seq;
        p.out = (__nv_bfloat16 *)out;
        p.part = (float *)workspace;
        p.prefix_out = (int *)((char *)workspace + t.part_bytes);
        p.nh = (int)desc->n_heads;
        p.nkv = (int)desc->n_kv_heads;
        p.max_blocks = (int)desc->max_blocks_per_seq;
        p.num_blocks = (int)desc->num_blocks;
        p.groups = seqs;
        p.hg = t.hg;
        p.ch = t.ch;
        p.kw = t.kw;
        p.pps = t.pps;
        p.stages = t.stages;
        p.G = t.G;
        p.whole = t.whole;
        p.wait_limit = limit;
        launch_pdl(kv8_attn_tokens, dim3((unsigned)t.G, (unsigned)t.ngroups), dim3(kTokThreads), t.smem,
                   maps[0], maps[1], p);
        rc = check_launch(what);
        if (rc != ECPU_OK) return rc;
        rc = check_error(what);
        if (rc != ECPU_OK) return rc;
        if (t.G == 1 || t.whole) continue;  // every group whole
        // a row of the batch is the longest a sequence can have
        const int max_q = (int)(desc->max_q_len < 1 ? 1 : (desc->max_q_len < desc->total_q ? desc->max_q_len : desc->total_q));
        // A group's partials lie in span CTAs at most.  As many warps share a row and head as load them
        // in one round (8 sequences of 5 rows over 4K keys: 38.0 us with 16 warps, 24.6 with 4); 16
        // with 10 loads each where one wave of blocks holds them all (8 rows over 8K: 20.2 against 21.1).
        const int span = t.G / seqs + 2;
        const bool wide = span > 8 && (long long)max_q * p.nh * seqs <= num_sms();
        int wpi = wide ? 16 : 1;
        while (!wide && wpi < 8 && 8 * wpi < span) wpi *= 2;
        const int per = wide ? 1 : 8 / wpi;
        launch_pdl(wide ? kv8_attn_merge<16, 10> : kv8_attn_merge<8, 8>,
                   dim3((unsigned)((p.nh + per - 1) / per * max_q), (unsigned)seqs), dim3(wide ? 512 : 256), 0, p, wpi);
        rc = check_launch(what);
        if (rc != ECPU_OK) return rc;
    }
    return ECPU_OK;
}

}  // extern "C"
