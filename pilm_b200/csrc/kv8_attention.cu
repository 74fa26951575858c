// Paged attention over an 8-bit KV cache (e4m3 codes, one scale per page and KV head).
//
// out = softmax(q k^T / sqrt(128)) v for rows at the end of each sequence's context; a row at
// position p sees keys <= p, or with a window the keys in (p - window, p] and the first sinks.
#include "fp8.cuh"

using namespace pilm;

namespace {

constexpr int kHD = kKv8HD;

struct AttnParams {
    const __nv_bfloat16 *q, *gate;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *block_table, *cu_q, *ctx;
    __nv_bfloat16 *out;
    int nh, nkv, num_seqs, max_blocks, num_blocks;
    long long window, sinks;
    float scale;
};

// One warp per (row, head), 4 dims per lane, one key at a time: online softmax in fp32.
__global__ void kv8_attn_simple(const AttnParams p, int total_q) {
    pdl_entry();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int row = (int)(item / p.nh), h = (int)(item % p.nh);
    if (row >= total_q || row >= p.cu_q[p.num_seqs]) return;
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {  // the last sequence that starts at or before the row
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const int b = lo, kvh = h / (p.nh / p.nkv);
    const int q_end = p.cu_q[b + 1], ctx = p.ctx[b];
    if (row >= q_end) return;
    const int pos = ctx - (q_end - row);
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    const size_t base = ((size_t)row * p.nh + h) * kHD + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = bf2f(p.q[base + j]) * p.scale;
    const long long first = p.window > 0 ? (long long)pos - p.window + 1 : 0;
    for (int key = 0; key <= pos; ++key) {
        if (key < first && key >= p.sinks) {
            key = (int)first - 1;
            continue;
        }
        const int blk = (key >> 4) < p.max_blocks ? p.block_table[(size_t)b * p.max_blocks + (key >> 4)] : -1;
        const bool ok = blk >= 0 && blk < p.num_blocks;
        float s = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
        if (ok) {
            const size_t at = (((size_t)blk * kKv8Page + (key & 15)) * p.nkv + kvh) * kHD + 4 * lane;
            const float ks = p.ks[(size_t)blk * p.nkv + kvh], vs = p.vs[(size_t)blk * p.nkv + kvh];
            const uint32_t kw = *reinterpret_cast<const uint32_t *>(p.kc + at);
            const uint32_t vw = *reinterpret_cast<const uint32_t *>(p.vc + at);
            const float2 k0 = f16x2_to_f32x2(e4m3x2_to_f16x2(kw)), k1 = f16x2_to_f32x2(e4m3x2hi_to_f16x2(kw));
            const float2 v0 = f16x2_to_f32x2(e4m3x2_to_f16x2(vw)), v1 = f16x2_to_f32x2(e4m3x2hi_to_f16x2(vw));
            s = (q[0] * k0.x + q[1] * k0.y + q[2] * k1.x + q[3] * k1.y) * ks;
            v[0] = v0.x * vs, v[1] = v0.y * vs, v[2] = v1.x * vs, v[3] = v1.y * vs;
        }
        s = warp_sum(s);
        const float mn = fmaxf(m, s), a = __expf(m - mn), pr = __expf(s - mn);
        m = mn;
        l = l * a + pr;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = o[j] * a + pr * v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float r = l > 0.f ? o[j] / l : 0.f;
        if (p.gate) r = r / (1.f + __expf(-bf2f(p.gate[base + j])));
        p.out[base + j] = f2bf(r);
    }
}

}  // namespace

extern "C" {

size_t ekernel_paged_attention_kv8_workspace_bytes(const ekernel_paged_attn_desc_t *desc, size_t window,
                                                   size_t sinks) {
    (void)window, (void)sinks;
    return kv8_check_desc(desc, "ekernel_paged_attention_kv8_workspace_bytes") == ECPU_OK ? 256 : 0;
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
    AttnParams p;
    p.q = (const __nv_bfloat16 *)q;
    p.gate = desc->output_gate ? (const __nv_bfloat16 *)gate : nullptr;
    p.kc = k_cache, p.vc = v_cache, p.ks = k_scale, p.vs = v_scale;
    p.block_table = block_table, p.cu_q = cu_q, p.ctx = context_lens;
    p.out = (__nv_bfloat16 *)out;
    p.nh = (int)desc->n_heads, p.nkv = (int)desc->n_kv_heads, p.num_seqs = (int)desc->num_seqs;
    p.max_blocks = (int)desc->max_blocks_per_seq, p.num_blocks = (int)desc->num_blocks;
    p.window = (long long)window, p.sinks = (long long)sinks;
    p.scale = 0.08838834764831845f;
    const size_t items = desc->total_q * desc->n_heads;
    launch_pdl(kv8_attn_simple, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, p, (int)desc->total_q);
    return check_launch(what);
}

}  // extern "C"
