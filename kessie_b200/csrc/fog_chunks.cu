// fog_chunks.cu -- attention of ragged chunks of new tokens over a paged KV
// cache (one launch for a whole mixed batch of decodes and prompt chunks).
//
// Query row t of sequence b (rows query_start_loc[b] .. [b + 1) of q) sits at
// position seq_lens[b] - n_b + t and sees the keys j < seq_lens[b] with
// j <= position (causal) and position - j < W (window):
//   s_j = scale q.k_j + bias_j,   O = sum_j softmax(s)_j w_j v_j
// with the V fog w_j = (j / max(cs - 1, 1))^alpha for j < cs
// (kessie_hip_kernels.py:403-413,577-593) or the additive fog bias
// (kessie_attention.py:114-139).  A row that sees no key is 0.
//
// First form: one warp per (query row, head), one key at a time.
#include "common.cuh"
#include "fog_bias.cuh"
#include "ptx.cuh"

#include <limits.h>
#include <math.h>

namespace kessie {
namespace {

struct ChunkParams {
    const void* q; int64_t q_st, q_sh;
    void* o; int64_t o_st, o_sh;
    const void* k; const void* v;
    int64_t page_stride, token_stride, head_stride;
    int num_pages, page_size;
    const int32_t* table; int64_t table_stride;
    const int32_t* start; const int32_t* seq;
    const int32_t* clear_start; float fog_alpha;
    int window, causal;
    float scale;
    int B, T, Hq, Hkv, G, max_seq;
    FogBias bias;
    int* status;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) fog_chunks_simple_kernel(const ChunkParams p) {
    const int b = blockIdx.y, lane = threadIdx.x & 31;
    const int h = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (h >= p.Hq) return;
    const int s0 = p.start[b], s1 = p.start[b + 1];
    const int r0 = min(max(s0, 0), p.T), r1 = max(r0, min(s1, p.T));
    const int len = p.seq[b];
    const int kv = min(max(len, 0), p.max_seq);
    if (r0 != s0 || r1 != s1 || kv != len) record_status(p.status, KESSIE_DEV_BAD_ARG);
    const int cs = p.clear_start && p.fog_alpha > 0.f ? p.clear_start[b] : INT_MIN;
    const int fb = p.bias.on ? fog_bias_boundary(p.bias, kv) : 0;
    constexpr int N = D / 32;
    for (int t = r0; t < r1; ++t) {
        const int pos = len - (r1 - r0) + (t - r0);
        const int hi = (p.causal || p.window > 0) ? min(kv, pos + 1) : kv;
        const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        const T* q = static_cast<const T*>(p.q) + t * p.q_st + h * p.q_sh + lane * N;
        float qr[N], acc[N], m = -INFINITY, l = 0.f;
        for (int i = 0; i < N; ++i) { qr[i] = to_f32(q[i]) * p.scale; acc[i] = 0.f; }
        for (int j = lo; j < hi; ++j) {
            const int id = p.table[b * p.table_stride + j / p.page_size];
            const bool ok = id >= 0 && id < p.num_pages;
            if (!ok) record_status(p.status, KESSIE_DEV_BAD_PAGE_ID);
            const int64_t off = (int64_t)(ok ? id : 0) * p.page_stride + (j % p.page_size) * p.token_stride +
                                (h / p.G) * p.head_stride + lane * N;
            float s = 0.f;
            for (int i = 0; i < N; ++i) s += ok ? qr[i] * to_f32(static_cast<const T*>(p.k)[off + i]) : 0.f;
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            if (p.bias.on) s += fog_bias_at(p.bias, fb, j);
            const float m_new = fmaxf(m, s), f = expf(m - m_new), e = expf(s - m_new);
            const float w = j < cs ? powf((float)j / (float)max(cs - 1, 1), p.fog_alpha) : 1.f;
            l = l * f + e;
            m = m_new;
            for (int i = 0; i < N; ++i)
                acc[i] = acc[i] * f + (ok ? e * w * to_f32(static_cast<const T*>(p.v)[off + i]) : 0.f);
        }
        T* o = static_cast<T*>(p.o) + t * p.o_st + h * p.o_sh + lane * N;
        for (int i = 0; i < N; ++i) o[i] = from_f32<T>(l > 0.f ? acc[i] / l : 0.f);
    }
}

}  // namespace
}  // namespace kessie

using namespace kessie;

extern "C" size_t kessie_paged_fog_chunks_workspace_size(int num_q_heads, int num_kv_heads, int head_dim) {
    return num_q_heads > 0 && num_kv_heads > 0 && head_dim > 0 ? 256 : 0;
}

extern "C" int kessie_paged_fog_chunks_v2(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                                          const void* v_cache, int64_t page_stride, int64_t token_stride,
                                          int64_t head_stride, int num_pages, int page_size,
                                          const int32_t* block_table, int64_t block_table_stride,
                                          const int32_t* query_start_loc, const int32_t* seq_lens,
                                          const int32_t* clear_start, float fog_alpha, int window_size, int is_causal,
                                          float sm_scale, int batch, int num_tokens, int num_q_heads, int num_kv_heads,
                                          int head_dim, int max_seq_len, int dtype, const kessie_fog_bias* bias,
                                          void* out, int64_t o_stride_t, int64_t o_stride_h, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_range("kessie_paged_fog_chunks_v2");
    if (dtype != KESSIE_DTYPE_BF16 && dtype != KESSIE_DTYPE_F16)
        return set_error(KESSIE_ERR_UNSUPPORTED, "paged_fog_chunks_v2: dtype %d (f16/bf16 only)", dtype);
    if (head_dim != 64 && head_dim != 128)
        return set_error(KESSIE_ERR_UNSUPPORTED, "paged_fog_chunks_v2: head_dim %d (64 or 128)", head_dim);
    if (page_size <= 0 || page_size % 16)
        return set_error(KESSIE_ERR_UNSUPPORTED, "paged_fog_chunks_v2: page_size %d (a multiple of 16)", page_size);
    if (batch < 0 || num_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        num_pages <= 0 || max_seq_len < 0)
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: bad shape B=%d T=%d Hq=%d Hkv=%d pages=%d", batch,
                         num_tokens, num_q_heads, num_kv_heads, num_pages);
    if (num_q_heads / num_kv_heads > 128)
        return set_error(KESSIE_ERR_UNSUPPORTED, "paged_fog_chunks_v2: %d query heads per KV head (at most 128)",
                         num_q_heads / num_kv_heads);
    if (!(sm_scale > 0.f) || isinf(sm_scale))
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: sm_scale %g (positive and finite)", (double)sm_scale);
    if (batch == 0 || num_tokens == 0) { clear_error(); return KESSIE_OK; }
    if (!q || !k_cache || !v_cache || !block_table || !query_start_loc || !seq_lens || !out)
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: null pointer");
    if (((token_stride | head_stride | page_stride | q_stride_t | q_stride_h | o_stride_t | o_stride_h) & 7) ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_cache) |
          reinterpret_cast<uintptr_t>(v_cache)) & 15))
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: q, out and cache rows must be 16-byte aligned");
    const size_t need = kessie_paged_fog_chunks_workspace_size(num_q_heads, num_kv_heads, head_dim);
    if (!workspace || workspace_bytes < need)
        return set_error(KESSIE_ERR_WORKSPACE, "paged_fog_chunks_v2: workspace %zu < %zu", workspace_bytes, need);
    ChunkParams p{};
    p.q = q; p.q_st = q_stride_t; p.q_sh = q_stride_h;
    p.o = out; p.o_st = o_stride_t; p.o_sh = o_stride_h;
    p.k = k_cache; p.v = v_cache;
    p.page_stride = page_stride; p.token_stride = token_stride; p.head_stride = head_stride;
    p.num_pages = num_pages; p.page_size = page_size;
    p.table = block_table; p.table_stride = block_table_stride;
    p.start = query_start_loc; p.seq = seq_lens;
    p.clear_start = clear_start; p.fog_alpha = fog_alpha;
    p.window = window_size > 0 ? window_size : 0; p.causal = is_causal ? 1 : 0;
    p.scale = sm_scale;
    p.B = batch; p.T = num_tokens; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads;
    p.max_seq = max_seq_len;
    const int brc = fog_bias_from_c(bias, &p.bias);
    if (brc) return brc;
    p.status = device_status_ptr();
    const dim3 grid((num_q_heads + 3) / 4, batch);
    auto kern = dtype == KESSIE_DTYPE_BF16
                    ? (head_dim == 128 ? fog_chunks_simple_kernel<__nv_bfloat16, 128> : fog_chunks_simple_kernel<__nv_bfloat16, 64>)
                    : (head_dim == 128 ? fog_chunks_simple_kernel<__half, 128> : fog_chunks_simple_kernel<__half, 64>);
    kern<<<grid, 128, 0, as_stream(stream)>>>(p);
    return check_launch("paged_fog_chunks");
}
