// step_tables.cu -- page tables and slot maps of one scheduler step, built on
// the device from the requests' lengths.
//
// For request r with c_r cached and n_r new tokens and pages of ps tokens:
//   query_start_loc = exclusive prefix sum of n,  seq_lens = c + n
//   owned_r = ceil(c_r / ps) pages are in block_table[r] already; the pages
//   [owned_r, need_r), need_r = ceil((c_r + n_r) / ps), are taken from the end
//   of the free list in request order: the batch's j-th new page is
//   free_pages[F - 1 - j] (the order KeSSiePagedKVCache.allocate_pages pops
//   them, kessie_hip_kernels.py:520-524) and is written into the table
//   new token t of r: position c_r + (t - start_r), slot = page * ps + pos % ps
//
// One launch.  Every CTA scans all the lengths itself (8 bytes a request, from
// L2) into two prefix arrays in shared memory, so no CTA waits on another;
// then the tokens and the new pages are spread over the grid and each finds its
// request by bisection.  A token on a new page reads its page id from the free
// list, not from the table another CTA may be writing.
//
// Bound by latency: 8 requests take 5 us of GPU time a call in a row of calls,
// 2,048 requests with 167,899 tokens no more than the ~18 us of the host's call.
#include "common.cuh"

#include <limits.h>
#include <stdint.h>

namespace kessie {
namespace {

constexpr int kStThreads = 1024;
constexpr int kStMaxRequests = 8192;      // two int32 prefix arrays in 64 KB of shared memory

struct StepTablesParams {
    const int32_t* ctx;
    const int32_t* qlen;
    int R;
    int32_t* table;
    int64_t table_stride;
    int max_pages, page_size, num_pages;
    const int32_t* free_pages;
    int num_free;
    const int32_t* free_count;
    int num_tokens;
    int32_t* start;
    int32_t* seq;
    int32_t* positions;
    int64_t* slots;
    int32_t* used;
    int* status;
};

struct Lens { int ctx, n, owned, fresh; bool bad; };

// Request r's lengths in page terms.  Negative lengths count as zero, a
// sequence past INT_MAX or past the table's width is cut (bad = true).
__device__ __forceinline__ Lens step_lens(const StepTablesParams& p, int r) {
    Lens l;
    const int c = p.ctx[r], n = p.qlen[r];
    l.ctx = max(c, 0);
    const int64_t end = (int64_t)l.ctx + max(n, 0);
    l.n = (int)min(end, (int64_t)INT_MAX) - l.ctx;
    l.owned = (int)(((int64_t)l.ctx + p.page_size - 1) / p.page_size);
    const int64_t need = ((int64_t)l.ctx + l.n + p.page_size - 1) / p.page_size;
    l.fresh = max((int)min(need, (int64_t)p.max_pages) - l.owned, 0);
    l.bad = c < 0 || n < 0 || end > INT_MAX || need > p.max_pages;
    return l;
}

// Last index r in [0, n) with a[r] <= x (a[0] = 0 <= x).
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kStThreads) step_tables_kernel(const StepTablesParams p) {
    extern __shared__ int sm[];
    int* tok = sm;                       // [R + 1] exclusive prefix of new tokens
    int* pgs = sm + p.R + 1;             // [R + 1] exclusive prefix of new pages
    __shared__ int64_t wsum[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t base_t = 0, base_p = 0;
    bool bad = false;
    for (int r0 = 0; r0 < p.R; r0 += kStThreads) {
        const int r = r0 + tid;
        Lens l{};
        if (r < p.R) l = step_lens(p, r);
        bad |= l.bad;
        int64_t xt = l.n, xp = l.fresh;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t yt = __shfl_up_sync(0xffffffffu, xt, d), yp = __shfl_up_sync(0xffffffffu, xp, d);
            if (lane >= d) { xt += yt; xp += yp; }
        }
        if (lane == 31) { wsum[0][warp] = xt; wsum[1][warp] = xp; }
        __syncthreads();
        int64_t bt = base_t, bp = base_p, all_t = 0, all_p = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) { bt += wsum[0][w]; bp += wsum[1][w]; }
            all_t += wsum[0][w];
            all_p += wsum[1][w];
        }
        if (r < p.R) {
            tok[r] = (int)min(bt + xt - l.n, (int64_t)INT_MAX);
            pgs[r] = (int)min(bp + xp - l.fresh, (int64_t)INT_MAX);
            if (blockIdx.x == 0) {
                p.start[r] = tok[r];
                p.seq[r] = l.ctx + l.n;
            }
        }
        base_t += all_t;
        base_p += all_p;
        __syncthreads();
    }
    const int total = (int)min(base_t, (int64_t)INT_MAX);
    const int fresh = (int)min(base_p, (int64_t)INT_MAX);
    const int F = p.free_count ? max(0, min(*p.free_count, p.num_free)) : p.num_free;
    if (tid == 0) {
        tok[p.R] = total;
        pgs[p.R] = fresh;
        if (blockIdx.x == 0) {
            p.start[p.R] = total;
            *p.used = min(fresh, F);
            if (base_t > p.num_tokens || base_p > F) record_status(p.status, KESSIE_DEV_BAD_ARG);
        }
    }
    if (bad && blockIdx.x == 0) record_status(p.status, KESSIE_DEV_BAD_ARG);
    __syncthreads();

    auto fresh_page = [&](int j) -> int { return j < F ? p.free_pages[F - 1 - j] : -1; };
    bool bad_page = false;
    const int step = gridDim.x * kStThreads;
    for (int64_t t = (int64_t)blockIdx.x * kStThreads + tid; t < p.num_tokens; t += step) {
        int pos = 0;
        int64_t slot = -1;
        if (t < total) {
            // requests without new tokens share a prefix value with the next
            // one: the last of them is the request that holds token t
            const int r = last_not_above(tok, p.R, (int)t);
            const int c = max(p.ctx[r], 0);
            pos = c + ((int)t - tok[r]);
            const int pg = pos / p.page_size, owned = (int)(((int64_t)c + p.page_size - 1) / p.page_size);
            if (pg < p.max_pages) {
                const int j = pgs[r] + (pg - owned);
                const int id = pg < owned ? p.table[r * p.table_stride + pg] : fresh_page(j);
                if (id >= 0 && id < p.num_pages) slot = (int64_t)id * p.page_size + pos % p.page_size;
                else if (pg < owned || j < F) bad_page = true;
            }
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
    for (int64_t j = (int64_t)blockIdx.x * kStThreads + tid; j < fresh; j += step) {
        const int r = last_not_above(pgs, p.R, (int)j);
        const int owned = (int)(((int64_t)max(p.ctx[r], 0) + p.page_size - 1) / p.page_size);
        p.table[r * p.table_stride + owned + ((int)j - pgs[r])] = fresh_page((int)j);
    }
    if (bad_page) record_status(p.status, KESSIE_DEV_BAD_PAGE_ID);
}

}  // namespace
}  // namespace kessie

using namespace kessie;

extern "C" int kessie_step_tables_v2(const int32_t* context_lens, const int32_t* query_lens, int num_requests,
                                     int32_t* block_table, int64_t block_table_stride, int max_pages, int page_size,
                                     int num_pages, const int32_t* free_pages, int num_free_pages,
                                     const int32_t* free_count, int num_tokens, int32_t* query_start_loc,
                                     int32_t* seq_lens, int32_t* positions, int64_t* slot_mapping,
                                     int32_t* pages_used, void* stream) {
    NvtxRange nvtx_range("kessie_step_tables_v2");
    if (num_requests < 0 || max_pages < 0 || page_size <= 0 || num_pages < 0 || num_free_pages < 0 || num_tokens < 0)
        return set_error(KESSIE_ERR_ARG, "step_tables_v2: bad sizes (requests %d, max_pages %d, page_size %d, "
                         "num_pages %d, free %d, tokens %d)", num_requests, max_pages, page_size, num_pages,
                         num_free_pages, num_tokens);
    if (num_requests > kStMaxRequests)
        return set_error(KESSIE_ERR_UNSUPPORTED, "step_tables_v2: %d requests (at most %d)", num_requests, kStMaxRequests);
    if (block_table_stride < max_pages && num_requests > 1)
        return set_error(KESSIE_ERR_ARG, "step_tables_v2: table stride below its width");
    if (!query_start_loc || !pages_used || (num_requests && (!context_lens || !query_lens || !seq_lens)) ||
        (num_requests && max_pages && !block_table) || (num_free_pages && !free_pages) ||
        (num_tokens && (!positions || !slot_mapping)))
        return set_error(KESSIE_ERR_ARG, "step_tables_v2: null pointer");
    // every CTA reads the inputs while others write
    struct Span { const void* at; size_t bytes; };
    const size_t R = (size_t)num_requests, T = (size_t)num_tokens;
    const Span in[] = {{context_lens, R * 4}, {query_lens, R * 4}, {free_pages, (size_t)num_free_pages * 4},
                       {free_count, free_count ? 4u : 0u}};
    const Span res[] = {{query_start_loc, (R + 1) * 4}, {seq_lens, R * 4}, {positions, T * 4}, {slot_mapping, T * 8},
                        {pages_used, 4},
                        {block_table, R && max_pages ? ((R - 1) * block_table_stride + max_pages) * 4 : 0}};
    for (const Span& a : in)
        for (const Span& b : res) {
            const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
            if (a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes)
                return set_error(KESSIE_ERR_ARG, "step_tables_v2: an output shares memory with an input");
        }
    StepTablesParams p{};
    p.ctx = context_lens; p.qlen = query_lens; p.R = num_requests;
    p.table = block_table; p.table_stride = block_table_stride;
    p.max_pages = max_pages; p.page_size = page_size; p.num_pages = num_pages;
    p.free_pages = free_pages; p.num_free = num_free_pages; p.free_count = free_count;
    p.num_tokens = num_tokens;
    p.start = query_start_loc; p.seq = seq_lens; p.positions = positions; p.slots = slot_mapping; p.used = pages_used;
    p.status = device_status_ptr();
    const size_t smem = 2 * sizeof(int) * (size_t)(num_requests + 1);
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return check_launch("step_tables: set smem attribute");
    const int64_t ctas = ((int64_t)num_tokens + kStThreads - 1) / kStThreads;
    const int grid = (int)(ctas < 1 ? 1 : ctas < sm_count() ? ctas : sm_count());
    step_tables_kernel<<<grid, kStThreads, smem, as_stream(stream)>>>(p);
    return check_launch("step_tables");
}
