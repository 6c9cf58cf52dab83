// rope_axes.cu -- rotary embedding with one position per axis (time, height,
// width, ...) for each token: new tokens on their way into the paged cache,
// and recalled keys moved to new positions.
//
// Frequency d (0 <= d < half) belongs to axis a(d); token t turns the pair
// (x_d, x_{d + half}) of every q and k head by
//   angle_d(t) = (target[a(d), t] - orig[a(d), t]) * f_d,  orig = 0 when absent,
// with f_d = theta^(-d / half) held in fp32 as the one-axis remap holds it
// (kessie_hip_kernels.py:596-606); dimensions past 2 * half pass through.
//
// Angles.  Positions reach 10^6 and f_0 = 1, so an fp32 product would be off
// by up to 0.06 rad.  The host stores F_d = frac(f_d / 2 pi) as a 64-bit
// fixed-point fraction of a turn; the integer product delta * F_d mod 2^64 is
// the angle's fraction of a turn, off by less than |delta| * 2^-64 turns, with
// no range reduction; sincospif takes it from there (fp32, ~1e-7 rad).
//
// HBM-bound: every row is read and written once (16 bytes a lane and access).
// A warp takes one token: its lanes compute the token's cos / sin once into
// shared memory, each keeps those of its own vector in registers, and then
// runs through the q, k and v rows, 32 / (half / VEC) rows at a time.
#include "common.cuh"

#include <math.h>
#include <string.h>

namespace kessie {
namespace {

constexpr int kRaWarps = 8;
constexpr int kRaMaxHalf = 256;
constexpr int kRaMaxAxes = 8;

struct RopeAxesTable {
    uint64_t turn[kRaMaxHalf];      // f_d / (2 pi) mod 1, in units of 2^-64
    uint8_t axis[kRaMaxHalf];
};

struct RopeAxesParams {
    const void* q; int64_t q_st, q_sh;
    void* oq; int64_t oq_st, oq_sh;
    const void* k; int64_t k_st, k_sh;
    const void* v; int64_t v_st, v_sh;
    int T, Hq, Hkv, D, half, axes;
    const int32_t* target; int64_t target_sa;
    const int32_t* orig; int64_t orig_sa;
    const int64_t* slots;
    void* kv; int64_t page_stride, token_stride, kv_stride, head_stride;
    int64_t num_slots;
    int page_size;
    int iters;                      // row groups per work item
    int chunks;                     // work items per token
    int* status;
};

template <typename T, int VEC> struct RaVec;
template <typename T> struct RaVec<T, 1> {
    T x[1];
    __device__ void load(const T* p) { x[0] = *p; }
    __device__ void store(T* p) const { *p = x[0]; }
};
template <typename T, int VEC> struct alignas(16) RaVec {
    T x[VEC];
    __device__ void load(const T* p) {
        uint4 u;
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
        *reinterpret_cast<uint4*>(x) = u;
    }
    __device__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x); }
};

template <typename T, int VEC>
__device__ __forceinline__ void ra_rotate(RaVec<T, VEC>& lo, RaVec<T, VEC>& hi, const float2* cs) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const float a = to_f32(lo.x[i]), b = to_f32(hi.x[i]);
        lo.x[i] = from_f32<T>(a * cs[i].x - b * cs[i].y);       // one rounding to the stored type
        hi.x[i] = from_f32<T>(a * cs[i].y + b * cs[i].x);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kRaWarps * 32) rope_axes_kernel(const __grid_constant__ RopeAxesParams p,
                                                                  const __grid_constant__ RopeAxesTable tab) {
    extern __shared__ __align__(16) uint8_t ra_smem[];
    uint64_t* turn = reinterpret_cast<uint64_t*>(ra_smem);
    float2* cs_all = reinterpret_cast<float2*>(turn + p.half);
    uint8_t* axis = reinterpret_cast<uint8_t*>(cs_all + kRaWarps * p.half);
    for (int d = threadIdx.x; d < p.half; d += blockDim.x) {
        turn[d] = tab.turn[d];
        axis[d] = tab.axis[d];
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float2* cs = cs_all + warp * p.half;
    const int npair = p.half / VEC;                               // vectors per half row (<= 32 when VEC > 1)
    const int rpi = VEC > 1 ? 32 / npair : 1;                     // rows per warp step
    const int sub = VEC > 1 ? lane / npair : 0;
    const int rows = p.Hq + 2 * p.Hkv;
    const int64_t items = (int64_t)p.T * p.chunks;
    bool bad = false;
    for (int64_t it = (int64_t)blockIdx.x * kRaWarps + warp; it < items; it += (int64_t)gridDim.x * kRaWarps) {
        const int t = (int)(it / p.chunks), chunk = (int)(it - (int64_t)t * p.chunks);
        __syncwarp();
        for (int d = lane; d < p.half; d += 32) {
            const int a = axis[d];
            int64_t delta = p.target[a * p.target_sa + t];
            if (p.orig) delta -= p.orig[a * p.orig_sa + t];
            const int32_t half_turns = (int32_t)(((uint64_t)delta * turn[d] + (1ull << 31)) >> 32);
            float s, c;
            sincospif((float)half_turns * 0x1p-31f, &s, &c);
            cs[d] = make_float2(c, s);
        }
        __syncwarp();
        float2 mine[VEC > 1 ? VEC : 1];
        if (VEC > 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) mine[i] = cs[min((lane - sub * npair) * VEC + i, p.half - 1)];
        }
        int64_t cache_row = -1;
        if (p.Hkv) {
            const int64_t slot = p.slots[t];
            if (slot >= p.num_slots) bad = true;
            else if (slot >= 0) cache_row = (slot / p.page_size) * p.page_stride + (slot % p.page_size) * p.token_stride;
        }
        const int r_end = min(rows, (chunk + 1) * p.iters * rpi);
        for (int r = chunk * p.iters * rpi + sub; r < r_end; r += rpi) {
            if (sub >= rpi) break;                               // lanes past the last whole row
            const T* src;
            T* dst;
            if (r < p.Hq) {
                src = static_cast<const T*>(p.q) + t * p.q_st + r * p.q_sh;
                dst = static_cast<T*>(p.oq) + t * p.oq_st + r * p.oq_sh;
            } else {
                const int h = r - p.Hq, is_v = h >= p.Hkv, hh = h - is_v * p.Hkv;
                if (cache_row < 0) continue;
                src = is_v ? static_cast<const T*>(p.v) + t * p.v_st + hh * p.v_sh
                           : static_cast<const T*>(p.k) + t * p.k_st + hh * p.k_sh;
                dst = static_cast<T*>(p.kv) + cache_row + is_v * p.kv_stride + hh * p.head_stride;
            }
            const bool turned = r < p.Hq + p.Hkv;
            const int first = VEC > 1 ? lane - sub * npair : lane, stride = VEC > 1 ? npair : 32;
            for (int e = first; e < npair; e += stride) {
                RaVec<T, VEC> lo, hi;
                lo.load(src + e * VEC);
                hi.load(src + p.half + e * VEC);
                if (turned) ra_rotate<T, VEC>(lo, hi, VEC > 1 ? mine : cs + e);
                lo.store(dst + e * VEC);
                hi.store(dst + p.half + e * VEC);
            }
            for (int e = 2 * npair + first; e < p.D / VEC; e += stride) {
                RaVec<T, VEC> x;
                x.load(src + e * VEC);
                x.store(dst + e * VEC);
            }
        }
    }
    if (bad) record_status(p.status, KESSIE_DEV_BAD_PAGE_ID);
}

// The frequency table: f_d in double, rounded to fp32, then its fraction of a
// turn in long double (64-bit mantissa).
int fill_table(RopeAxesTable* tab, const int* sections, int axes, int interleaved, float theta, int* half_out) {
    int half = 0;
    for (int a = 0; a < axes; ++a) {
        if (sections[a] < 0 || sections[a] > kRaMaxHalf) return set_error(KESSIE_ERR_ARG, "rope_axes: section %d", sections[a]);
        half += sections[a];
    }
    if (half <= 0 || half > kRaMaxHalf)
        return set_error(KESSIE_ERR_UNSUPPORTED, "rope_axes: %d frequencies (1 to %d)", half, kRaMaxHalf);
    int count[kRaMaxAxes] = {0};
    for (int d = 0, a = 0, left = sections[0]; d < half; ++d) {
        if (interleaved) {
            a = d % axes;
            if (d >= axes * sections[a]) a = 0;
        } else {
            while (left == 0) left = sections[++a];
            --left;
        }
        tab->axis[d] = (uint8_t)a;
        ++count[a];
        const float f = (float)pow((double)theta, -(double)d / half);
        const long double turns = (long double)f / 6.283185307179586476925286766559L;
        long double frac = turns - floorl(turns);
        tab->turn[d] = (uint64_t)(frac * 0x1p64L);
    }
    for (int a = 0; a < axes; ++a)
        if (count[a] != sections[a])
            return set_error(KESSIE_ERR_ARG, "rope_axes: sections do not interleave (axis %d gets %d of %d frequencies)",
                             a, count[a], sections[a]);
    *half_out = half;
    return KESSIE_OK;
}

template <typename T, int VEC>
int launch_typed(RopeAxesParams& p, const RopeAxesTable& tab, cudaStream_t st) {
    const int npair = p.half / VEC;
    const int rpi = VEC > 1 ? 32 / npair : 1;
    const int groups = (p.Hq + 2 * p.Hkv + rpi - 1) / rpi;
    // One warp walks all rows of a token once there are tokens for 16 warps an
    // SM; below that the rows are spread over more warps (each redoes the
    // token's angles), so that a decode step's few tokens still fill the GPU.
    const int64_t want = 16LL * sm_count();
    int64_t iters = (int64_t)p.T * groups / want;
    p.iters = (int)(iters < 1 ? 1 : iters < groups ? iters : groups);
    p.chunks = (groups + p.iters - 1) / p.iters;
    const size_t smem = p.half * (sizeof(uint64_t) + kRaWarps * sizeof(float2) + 1);
    const int64_t ctas = ((int64_t)p.T * p.chunks + kRaWarps - 1) / kRaWarps;
    const int64_t cap = 8LL * sm_count();
    rope_axes_kernel<T, VEC><<<(int)(ctas < cap ? ctas : cap), kRaWarps * 32, smem, st>>>(p, tab);
    return check_launch("rope_axes");
}

template <typename T>
int launch_rope_axes(RopeAxesParams& p, const RopeAxesTable& tab, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t es = sizeof(T);
    uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.oq) |
                     reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | reinterpret_cast<uintptr_t>(p.kv);
    int64_t steps = p.q_st | p.q_sh | p.oq_st | p.oq_sh | p.k_st | p.k_sh | p.v_st | p.v_sh | p.page_stride |
                    p.token_stride | p.kv_stride | p.head_stride | p.half | p.D;
    const bool vec = !(bits & 15) && !((steps * es) & 15) && p.half / VEC <= 32;
    return vec ? launch_typed<T, VEC>(p, tab, st) : launch_typed<T, 1>(p, tab, st);
}

int run_rope_axes(RopeAxesParams& p, int dtype, const int* sections, int interleaved, float theta, cudaStream_t st) {
    if (p.axes < 1 || p.axes > kRaMaxAxes || !sections)
        return set_error(KESSIE_ERR_ARG, "rope_axes: %d axes (1 to %d)", p.axes, kRaMaxAxes);
    if (!(theta > 0.f) || isinf(theta)) return set_error(KESSIE_ERR_ARG, "rope_axes: theta %g", (double)theta);
    // The table of the thread's last call is kept: a model uses one, and 64
    // powers and remainders cost more host time than the launch.
    struct Last { int axes = 0, sections[kRaMaxAxes], interleaved, half; float theta; RopeAxesTable tab; };
    static thread_local Last last;
    if (last.axes != p.axes || last.interleaved != interleaved || last.theta != theta ||
        memcmp(last.sections, sections, p.axes * sizeof(int)) != 0) {
        last.axes = 0;
        const int rc = fill_table(&last.tab, sections, p.axes, interleaved, theta, &last.half);
        if (rc) return rc;
        last.axes = p.axes; last.interleaved = interleaved; last.theta = theta;
        memcpy(last.sections, sections, p.axes * sizeof(int));
    }
    const RopeAxesTable& tab = last.tab;
    p.half = last.half;
    if (2 * p.half > p.D) return set_error(KESSIE_ERR_ARG, "rope_axes: %d rotated dimensions of %d", 2 * p.half, p.D);
    p.status = device_status_ptr();
    if (p.T == 0) { clear_error(); return KESSIE_OK; }
    switch (dtype) {
        case KESSIE_DTYPE_F16: return launch_rope_axes<__half>(p, tab, st);
        case KESSIE_DTYPE_BF16: return launch_rope_axes<__nv_bfloat16>(p, tab, st);
        default: return launch_rope_axes<float>(p, tab, st);
    }
}

}  // namespace
}  // namespace kessie

using namespace kessie;

extern "C" int kessie_rope_axes_remap_v2(const void* k, int64_t k_token_stride, int64_t k_head_stride, void* out,
                                         int64_t out_token_stride, int64_t out_head_stride, int dtype, int num_tokens,
                                         int num_heads, int head_dim, const int32_t* orig_positions,
                                         int64_t orig_axis_stride, const int32_t* target_positions,
                                         int64_t target_axis_stride, const int* sections, int num_axes,
                                         int interleaved, float rope_theta, void* stream) {
    NvtxRange nvtx_range("kessie_rope_axes_remap_v2");
    if (!dtype_ok(dtype)) return set_error(KESSIE_ERR_UNSUPPORTED, "rope_axes_remap_v2: dtype %d", dtype);
    if (num_tokens < 0 || num_heads <= 0 || head_dim <= 0)
        return set_error(KESSIE_ERR_ARG, "rope_axes_remap_v2: bad shape T=%d H=%d D=%d", num_tokens, num_heads, head_dim);
    if (num_tokens && (!k || !out || !target_positions))
        return set_error(KESSIE_ERR_ARG, "rope_axes_remap_v2: null pointer");
    RopeAxesParams p{};
    p.q = k; p.q_st = k_token_stride; p.q_sh = k_head_stride;
    p.oq = out; p.oq_st = out_token_stride; p.oq_sh = out_head_stride;
    p.T = num_tokens; p.Hq = num_heads; p.Hkv = 0; p.D = head_dim; p.axes = num_axes;
    p.target = target_positions; p.target_sa = target_axis_stride;
    p.orig = orig_positions; p.orig_sa = orig_axis_stride;
    p.page_size = 1;
    return run_rope_axes(p, dtype, sections, interleaved, rope_theta, as_stream(stream));
}

extern "C" int kessie_rope_axes_insert_v2(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* out_q,
                                          int64_t out_token_stride, int64_t out_head_stride, const void* k,
                                          int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                          int64_t v_token_stride, int64_t v_head_stride, int dtype, int num_tokens,
                                          int num_q_heads, int num_kv_heads, int head_dim, const int32_t* positions,
                                          int64_t positions_axis_stride, const int* sections, int num_axes,
                                          int interleaved, float rope_theta, void* kv_cache, int64_t page_stride,
                                          int64_t token_stride, int64_t kv_stride, int64_t head_stride, int num_pages,
                                          int page_size, const int64_t* slot_mapping, void* stream) {
    NvtxRange nvtx_range("kessie_rope_axes_insert_v2");
    if (!dtype_ok(dtype)) return set_error(KESSIE_ERR_UNSUPPORTED, "rope_axes_insert_v2: dtype %d", dtype);
    if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads <= 0 || head_dim <= 0 || num_pages <= 0 || page_size <= 0)
        return set_error(KESSIE_ERR_ARG, "rope_axes_insert_v2: bad shape T=%d Hq=%d Hkv=%d D=%d pages=%d x %d",
                         num_tokens, num_q_heads, num_kv_heads, head_dim, num_pages, page_size);
    if (num_tokens && ((num_q_heads && (!q || !out_q)) || !k || !v || !positions || !slot_mapping || !kv_cache))
        return set_error(KESSIE_ERR_ARG, "rope_axes_insert_v2: null pointer");
    RopeAxesParams p{};
    p.q = q; p.q_st = q_token_stride; p.q_sh = q_head_stride;
    p.oq = out_q; p.oq_st = out_token_stride; p.oq_sh = out_head_stride;
    p.k = k; p.k_st = k_token_stride; p.k_sh = k_head_stride;
    p.v = v; p.v_st = v_token_stride; p.v_sh = v_head_stride;
    p.T = num_tokens; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.D = head_dim; p.axes = num_axes;
    p.target = positions; p.target_sa = positions_axis_stride;
    p.slots = slot_mapping; p.kv = kv_cache;
    p.page_stride = page_stride; p.token_stride = token_stride; p.kv_stride = kv_stride; p.head_stride = head_stride;
    p.num_slots = (int64_t)num_pages * page_size; p.page_size = page_size;
    return run_rope_axes(p, dtype, sections, interleaved, rope_theta, as_stream(stream));
}
