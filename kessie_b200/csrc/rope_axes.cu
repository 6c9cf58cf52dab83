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
// fixed-point fraction of a turn; position * F_d mod 2^64 is the angle's
// fraction of a turn, off by less than |position| * 2^-64 turns, with no range
// reduction, and its top 32 bits are kept.  As a float a fraction is off by at
// most 2^-25 half turns (9.4e-8 rad).  For fp32 rows sincospif takes it from there
// (2 ulp); for 16-bit rows the hardware sine and cosine on [-pi, pi] do: 4.2e-7 at
// most, and 3.0e-7 for the argument (that rounding, the one of the product with
// pi and of pi itself): below 7.2e-7, against 2^-11 of the stored rounding.
//
// HBM-bound: every row is read and written once (16 bytes a thread and access).
// A thread owns one vector pair (VEC neighbouring frequencies) of one token and
// runs through the token's q, k and v heads, kRaBatch of them in flight: the
// token's angles are computed once over its threads, stay in registers, and
// nothing is shared.  Forms that shared angles through shared memory (a warp or
// a CTA per block of tokens) issued 500 to 570 instructions a token for the remap
// of 65,536 keys of 8 fp16 heads and took 55 to 76 us; this one takes 46.6 us,
// 246 instructions a token (5.8 TB/s; a plain copy of the same bytes: 44 us).
// 8,197 new tokens of 32 + 8 + 8 bf16 heads into their slots: 38.7 us, 5.2 TB/s.
#include "common.cuh"
#include "ptx.cuh"

#include <limits.h>
#include <math.h>
#include <string.h>

namespace kessie {
namespace {

constexpr int kRaThreads = 64;
constexpr int kRaBatch = 4;                // heads in flight per thread
constexpr int kRaWarps = 8;                // warps an SM wanted before threads take whole tokens
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
    int rows, parts;                // rows (of Hq + 2 Hkv) that a thread takes, threads per vector pair and token
    int* status;
};

template <typename T> struct alignas(16) RaVec {
    static constexpr int N = 16 / sizeof(T);
    T x[N];
    __device__ void load(const T* p) {
        uint4 u;
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
        *reinterpret_cast<uint4*>(x) = u;
    }
    __device__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x); }
};

template <typename T>
__device__ __forceinline__ void ra_rotate(T& lo, T& hi, float2 cs) {
    const float a = to_f32(lo), b = to_f32(hi);
    lo = from_f32<T>(a * cs.x - b * cs.y);                     // one rounding to the stored type
    hi = from_f32<T>(a * cs.y + b * cs.x);
}

// Two neighbouring elements as a packed fp32 pair, and back (one rounding).
__device__ __forceinline__ uint64_t ra_load2(const __half* x) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(x));
    return ptx::f2_pack(f.x, f.y);
}
__device__ __forceinline__ uint64_t ra_load2(const __nv_bfloat16* x) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x));
    return ptx::f2_pack(f.x, f.y);
}
__device__ __forceinline__ uint64_t ra_load2(const float* x) { return ptx::f2_pack(x[0], x[1]); }
__device__ __forceinline__ void ra_store2(__half* x, uint64_t v) {
    float a, b;
    ptx::f2_unpack(v, a, b);
    *reinterpret_cast<__half2*>(x) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void ra_store2(__nv_bfloat16* x, uint64_t v) {
    float a, b;
    ptx::f2_unpack(v, a, b);
    *reinterpret_cast<__nv_bfloat162*>(x) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void ra_store2(float* x, uint64_t v) { ptx::f2_unpack(v, x[0], x[1]); }

// Rotate elements x[0], x[1] of both halves; cs = (cos, cos, sin, sin).
template <typename T>
__device__ __forceinline__ void ra_rotate2(T* lo, T* hi, float4 cs) {
    const uint64_t a = ra_load2(lo), b = ra_load2(hi);
    const uint64_t c = ptx::f2_pack(cs.x, cs.y), s = ptx::f2_pack(cs.z, cs.w), ns = ptx::f2_pack(-cs.z, -cs.w);
    ra_store2(lo, ptx::ffma2(a, c, ptx::fmul2(b, ns)));
    ra_store2(hi, ptx::ffma2(a, s, ptx::fmul2(b, c)));
}

// cos and sin of a signed fraction of a turn in units of 2^-32.
template <bool EXACT>
__device__ __forceinline__ float2 ra_cos_sin(int32_t turn) {
    float s, c;
    if (EXACT) sincospif((float)turn * 0x1p-31f, &s, &c);
    else __sincosf((float)turn * (3.14159265358979f * 0x1p-31f), &s, &c);
    return make_float2(c, s);
}

// Top 32 bits of position * turn mod 2^64.
__device__ __forceinline__ uint32_t ra_turns(uint64_t turn, int position) {
    const uint32_t lo = (uint32_t)turn, hi = (uint32_t)(turn >> 32), u = (uint32_t)position;
    return __umulhi(lo, u) + hi * u - (position < 0 ? lo : 0u);
}
// cos and sin of the move from orig to target (each product's truncation: 2^-32 turns).
template <typename T>
__device__ __forceinline__ float2 ra_angle(uint64_t turn, int target, int orig) {
    return ra_cos_sin<sizeof(T) == 4>((int32_t)(ra_turns(turn, target) - ra_turns(turn, orig)));
}
// Element offset of slot's row in the cache, or -1 (not written; bad: past the cache).
__device__ __forceinline__ int64_t ra_cache_row(const RopeAxesParams& p, int64_t slot, bool& bad) {
    if (slot < 0) return -1;
    if (slot >= p.num_slots) { bad = true; return -1; }
    const int64_t page = slot <= 0x7fffffff ? (int64_t)((uint32_t)slot / (uint32_t)p.page_size) : slot / p.page_size;
    return page * p.page_stride + (slot - page * p.page_size) * p.token_stride;
}

// Vector pairs of kRaBatch heads (of the n from src on).
template <typename T> struct RaHeads {
    RaVec<T> lo[kRaBatch], hi[kRaBatch];
    __device__ __forceinline__ void load(const T* src, int64_t sh, int n, int half) {
#pragma unroll
        for (int u = 0; u < kRaBatch; ++u)
            if (u < n) {
                lo[u].load(src + u * sh);
                hi[u].load(src + u * sh + half);
            }
    }
};
// n heads from src to dst, rotated (or copied) by this thread's angles; the
// first kRaBatch are in x already.
template <bool TURN, typename T>
__device__ __forceinline__ void ra_heads(RaHeads<T>& x, const T* src, int64_t sh, T* dst, int64_t dh, int n, int half,
                                         const float4 (&cs)[RaVec<T>::N / 2]) {
    while (true) {
#pragma unroll
        for (int u = 0; u < kRaBatch; ++u)
            if (u < n) {
                if (TURN)
#pragma unroll
                    for (int e = 0; e < RaVec<T>::N / 2; ++e) ra_rotate2(&x.lo[u].x[2 * e], &x.hi[u].x[2 * e], cs[e]);
                x.lo[u].store(dst + u * dh);
                x.hi[u].store(dst + u * dh + half);
            }
        n -= kRaBatch;
        if (n <= 0) break;
        src += kRaBatch * sh;
        dst += kRaBatch * dh;
        x.load(src, sh, n, half);
    }
}

template <typename T>
__global__ void __launch_bounds__(kRaThreads) rope_axes_kernel(const __grid_constant__ RopeAxesParams p,
                                                               const __grid_constant__ RopeAxesTable tab) {
    constexpr int VEC = RaVec<T>::N;
    __shared__ uint64_t turn[kRaMaxHalf];
    __shared__ uint8_t axis[kRaMaxHalf];
    const int npair = p.half / VEC;                               // threads per token
    const int per_cta = kRaThreads / npair;
    const int sub = threadIdx.x / npair, vec = threadIdx.x - sub * npair, off = vec * VEC;
    const int64_t item = (int64_t)blockIdx.x * per_cta + sub;     // (token, part of its rows)
    const int64_t t = p.parts == 1 ? item : item / p.parts;
    const int part = (int)(item - t * p.parts);
    const bool on = sub < per_cta && t < p.T;
    // rows [r0, r1) of q heads, k heads, v heads: heads [q0, q1), [k0, k1), [v0, v1)
    const int r0 = part * p.rows, r1 = on ? min(r0 + p.rows, p.Hq + 2 * p.Hkv) : r0;
    const int q0 = r0, q1 = min(r1, p.Hq), k0 = max(r0 - p.Hq, 0), k1 = min(r1 - p.Hq, p.Hkv);
    const int v0 = max(r0 - p.Hq - p.Hkv, 0), v1 = r1 - p.Hq - p.Hkv;
    const T* q = static_cast<const T*>(p.q) + t * p.q_st + q0 * p.q_sh + off;
    const T* k = static_cast<const T*>(p.k) + t * p.k_st + k0 * p.k_sh + off;
    const T* v = static_cast<const T*>(p.v) + t * p.v_st + v0 * p.v_sh + off;
    // the first rows are on their way while the angles are computed
    RaHeads<T> x;
    if (q0 < q1) x.load(q, p.q_sh, q1 - q0, p.half);
    else if (k0 < k1) x.load(k, p.k_sh, k1 - k0, p.half);
    for (int d = threadIdx.x; d < p.half; d += kRaThreads) {
        turn[d] = tab.turn[d];
        axis[d] = tab.axis[d];
    }
    __syncthreads();
    if (r0 >= r1) return;
    float4 cs[VEC / 2];                                           // (cos, cos, sin, sin) of two dimensions
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
        float2 a2[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = off + 2 * e + i, a = axis[d];
            a2[i] = ra_angle<T>(turn[d], __ldg(p.target + a * p.target_sa + t), p.orig ? __ldg(p.orig + a * p.orig_sa + t) : 0);
        }
        cs[e] = make_float4(a2[0].x, a2[1].x, a2[0].y, a2[1].y);
    }
    bool bad = false;
    const int64_t row = r1 > p.Hq ? ra_cache_row(p, p.slots[t], bad) : -1;
    T* kv = static_cast<T*>(p.kv) + row + off;
    if (q0 < q1) {
        ra_heads<true>(x, q, p.q_sh, static_cast<T*>(p.oq) + t * p.oq_st + q0 * p.oq_sh + off, p.oq_sh, q1 - q0, p.half, cs);
        if (k0 < k1 && row >= 0) x.load(k, p.k_sh, k1 - k0, p.half);
    }
    if (k0 < k1 && row >= 0) ra_heads<true>(x, k, p.k_sh, kv + k0 * p.head_stride, p.head_stride, k1 - k0, p.half, cs);
    if (v0 < v1 && row >= 0) {
        x.load(v, p.v_sh, v1 - v0, p.half);
        ra_heads<false>(x, v, p.v_sh, kv + p.kv_stride + v0 * p.head_stride, p.head_stride, v1 - v0, p.half, cs);
    }
    if (2 * p.half < p.D) {                                       // dimensions past the rotated ones
        for (int r = r0; r < r1; ++r) {
            const int sec = r < p.Hq ? 0 : r < p.Hq + p.Hkv ? 1 : 2, h = r - (sec == 0 ? 0 : p.Hq + (sec - 1) * p.Hkv);
            if (sec != 0 && row < 0) break;
            const T* src = sec == 0 ? static_cast<const T*>(p.q) + t * p.q_st + h * p.q_sh
                         : sec == 1 ? static_cast<const T*>(p.k) + t * p.k_st + h * p.k_sh
                                    : static_cast<const T*>(p.v) + t * p.v_st + h * p.v_sh;
            T* dst = sec == 0 ? static_cast<T*>(p.oq) + t * p.oq_st + h * p.oq_sh
                              : static_cast<T*>(p.kv) + row + (sec == 2 ? p.kv_stride : 0) + h * p.head_stride;
            for (int d = 2 * p.half + off; d < p.D; d += p.half) {
                RaVec<T> y;
                y.load(src + d);
                y.store(dst + d);
            }
        }
    }
    if (bad) record_status(p.status, KESSIE_DEV_BAD_PAGE_ID);
}

// Rows that are not 16-byte aligned, or half not a multiple of a vector: a
// warp per token, one element a lane.
template <typename T>
__global__ void __launch_bounds__(kRaThreads) rope_axes_scalar_kernel(const __grid_constant__ RopeAxesParams p,
                                                                         const __grid_constant__ RopeAxesTable tab) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool bad = false;
    for (int64_t t = (int64_t)blockIdx.x * (kRaThreads / 32) + warp; t < p.T; t += (int64_t)gridDim.x * (kRaThreads / 32)) {
        const int64_t row = p.Hkv ? ra_cache_row(p, p.slots[t], bad) : -1;
        for (int d = lane; d < p.D - p.half; d += 32) {              // [0, half): a pair; above: a dimension as it is
            const int e = d < p.half ? d : d + p.half;
            const float2 c = d < p.half ? ra_angle<T>(tab.turn[d], p.target[tab.axis[d] * p.target_sa + t],
                                                        p.orig ? p.orig[tab.axis[d] * p.orig_sa + t] : 0) : make_float2(1.f, 0.f);
            for (int h = 0; h < p.Hq + 2 * p.Hkv; ++h) {
                const int sec = h < p.Hq ? 0 : h < p.Hq + p.Hkv ? 1 : 2, r = h - (sec == 0 ? 0 : p.Hq + (sec - 1) * p.Hkv);
                if (sec != 0 && row < 0) break;
                const T* src = sec == 0 ? static_cast<const T*>(p.q) + t * p.q_st + r * p.q_sh
                             : sec == 1 ? static_cast<const T*>(p.k) + t * p.k_st + r * p.k_sh
                                        : static_cast<const T*>(p.v) + t * p.v_st + r * p.v_sh;
                T* dst = sec == 0 ? static_cast<T*>(p.oq) + t * p.oq_st + r * p.oq_sh
                                  : static_cast<T*>(p.kv) + row + (sec == 2 ? p.kv_stride : 0) + r * p.head_stride;
                T lo = src[e];
                if (d < p.half) {
                    T hi = src[e + p.half];
                    if (sec != 2) ra_rotate(lo, hi, c);
                    dst[e + p.half] = hi;
                }
                dst[e] = lo;
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
        if (isinf(f))                    // theta below about 1e-39: no fraction of a turn
            return set_error(KESSIE_ERR_ARG, "rope_axes: theta %g: frequency %d is past fp32", (double)theta, d);
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

template <typename T>
int launch_rope_axes(RopeAxesParams& p, const RopeAxesTable& tab, cudaStream_t st) {
    constexpr int VEC = RaVec<T>::N;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.oq) |
                           reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                           reinterpret_cast<uintptr_t>(p.kv);
    const int64_t steps = p.q_st | p.q_sh | p.oq_st | p.oq_sh | p.k_st | p.k_sh | p.v_st | p.v_sh | p.page_stride |
                          p.token_stride | p.kv_stride | p.head_stride | p.half | p.D;
    const int64_t sms = sm_count();
    if ((bits & 15) || (steps % VEC) || p.half / VEC > 32) {
        const int64_t ctas = ((int64_t)p.T + kRaThreads / 32 - 1) / (kRaThreads / 32);
        rope_axes_scalar_kernel<T><<<(int)(ctas < 16 * sms ? ctas : 16 * sms), kRaThreads, 0, st>>>(p, tab);
        return check_launch("rope_axes");
    }
    // One thread takes all rows of its vector pair, unless that leaves less
    // than kRaWarps warps an SM: then the rows are shared out (each thread
    // redoes the angles), down to kRaBatch of them.
    const int per_cta = kRaThreads / (p.half / VEC), all_rows = p.Hq + 2 * p.Hkv;
    const int64_t warps = ((int64_t)p.T + per_cta - 1) / per_cta * (kRaThreads / 32), want = kRaWarps * sms;
    int64_t parts = warps < want ? (want + warps - 1) / warps : 1;
    if (parts > (all_rows + kRaBatch - 1) / kRaBatch) parts = (all_rows + kRaBatch - 1) / kRaBatch;
    p.rows = (int)((all_rows + parts - 1) / parts);
    p.parts = (all_rows + p.rows - 1) / p.rows;
    const int64_t ctas = ((int64_t)p.T * p.parts + per_cta - 1) / per_cta;
    if (ctas > INT_MAX) return set_error(KESSIE_ERR_UNSUPPORTED, "rope_axes: %d tokens", p.T);
    rope_axes_kernel<T><<<(int)ctas, kRaThreads, 0, st>>>(p, tab);
    return check_launch("rope_axes");
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
    if ((p.T > 1 && p.Hq && p.oq_st == 0) || (p.Hq > 1 && p.oq_sh == 0))
        return set_error(KESSIE_ERR_ARG, "rope_axes: rows of the output share memory");
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
