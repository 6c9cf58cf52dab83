// fog_chunks.cu -- attention of ragged chunks of new tokens over a paged KV
// cache: a whole mixed batch of decodes and prompt chunks, planned on the
// device, on the 5th-generation tensor cores.
//
// Query row t of sequence b (rows query_start_loc[b] .. [b + 1) of q) sits at
// position seq_lens[b] - n_b + t and sees the keys j < seq_lens[b] with
// j <= position (causal) and position - j < W (window):
//   s_j = scale q.k_j + bias_j,   O = sum_j softmax(s)_j w_j v_j
// with the V fog w_j = (j / max(cs - 1, 1))^alpha for j < cs
// (kessie_hip_kernels.py:403-413,577-593) or the additive fog bias
// (kessie_attention.py:114-139).  A row that sees no key is 0.
//
// Tiles.  Rows are (token, head-in-group) pairs of one KV head, so the G query
// heads that share a KV head share every K/V tile.  TH = 128 / G tokens make
// one 128-row half; a tile is two halves A, B (a "pair" tile: both read each
// 128-key tile) or, when its tokens fit one half (decodes, short chunks), a
// "single" tile: the same rows twice, A over the even and B over the odd key
// tiles, merged at the end.  Either way two independent score / softmax /
// product chains alternate on the tensor core.
//
// Plan.  The key tiles of all (sequence, KV head, tile) triples are laid end
// to end, each weighted with what it costs (kCostPair / kCostSingle per key
// tile, kCostTile per tile), and the persistent grid's CTA c streams the
// equal range [c L, (c + 1) L): no wave quantisation, whatever the mix of
// lengths.  Cutting puts the CTAs at different keys of a head at any time, so
// each would fetch its K/V for itself: when several tiles share a long context
// (kWholeCost), the CTAs first take whole tiles in waves -- neighbours run
// through the same keys together, from L2 -- and cut only what is left.
// Every CTA derives the plan itself from the length arrays.  A tile cut by a
// range boundary leaves fp32 partials (O, m, l) of each piece in the workspace,
// at most two a CTA, and fog_chunks_merge_kernel joins them in order, so
// results do not depend on timing.
//
// CTA = 12 warps: 0-3 / 4-7 softmax of A / B (one row per thread: TMEM lane =
// row), 8 Q and K producer, 9 / 11 MMA issuers of A / B (one thread each; 9
// owns the TMEM), 10 V producer and fog weights.  TMEM columns: S_A [0,128) S_B
// [128,256) O_A [256,..) O_B [384,..); P (16-bit pairs) overwrites the first 64
// columns of its S.  Per key tile a chain's issuer waits for P (three quarters, then
// the rest, so that the product starts under the last exponentials: 12.1 -> 11.6
// Mcycles at 4,096 tokens over 131k keys), issues O += P V and S = Q K^T of its
// next key tile into the region that P leaves, so one chain's MMAs run under the
// other's softmax.  One issuer for both chains was
// slower (4,600 against 3,600 cycles a pair of key tiles): its barrier waits
// left the tensor pipe idle.  Producers run ahead over tile ends.
//
// K/V come straight from the pages: one TMA box per page (up to 128 tokens)
// lands as [token / 8][D / 64][8][64] with 128-byte swizzle, whose 8-row groups
// have one stride, so a K or V tile of any page size is one matrix operand.
//
// Bound by: the serial chain scores -> exponentials -> P -> product of chunks
// (2,048 tokens of 32 / 8 heads of 128 over 32,768 keys, bf16: tensor pipe 60 %,
// MUFU 61 % busy under ncu, 0.99 ms; 4,096 over 131,072: 6.8-7.1 ms = 1,220-1,270
// TFLOP/s in the first launches, 7.65 ms = 1,130 in a row of them, 9.0 ms with the
// V fog, where the power cap holds the clock near 1.75 GHz), HBM for decodes (28
// of 1k-16k keys, 0.69 GB of K/V: 141 us = 4.9 TB/s; 28 of 1.04 GB: 6.0 TB/s under
// ncu, every key read once), launches and the plan for the smallest (17 us).
//
// Every mbarrier wait is bounded; on a timeout all warps still reach the final
// barrier and the TMEM is freed.
#include "common.cuh"
#include "fog_bias.cuh"
#include "ptx.cuh"
#include "tma_host.cuh"

#include <limits.h>
#include <math.h>

#include <atomic>

namespace kessie {
namespace {

constexpr int kThreads = 384;
constexpr int kSoftmaxWarps = 8;
constexpr int kMaxBatch = 8192;              // sequences whose prefix sums the plan keeps in shared memory
constexpr int kWStages = 4;                  // key tiles of fog weights in flight
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;    // log2 units the running max may lag behind
// P is rounded to the 16-bit type of V for the product (relative 2^-11 in fp16, 2^-8 in bf16; the row sum takes it
// unrounded).  In fp16 a small P is also subnormal, off by 2^-25, and over 131,072 keys these add up to 2^-8 of the
// largest value (one key against 131,071 of e^-16.25 each lost a quarter of what those bring).  So fp16 holds P times
// 2^7, which with the lag above stays within 2^15; the factor is in l and O alike and leaves with 1 / l.
constexpr float kHalfHeadroom = 7.0f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kProducerRegs = 88;
static_assert(256 * kSoftmaxRegs + 128 * kProducerRegs <= kThreads * kLaunchRegs, "register split exceeds the pool");

// Plan weights of a 128-key tile (pair / single) and of starting and ending a tile
// (with 4 for the latter, 208 short sequences took 209 us, with 7 188 us, with 14
// 193 us; an 8,192-token prompt 530, 498, 506 us).
constexpr int kCostPair = 3, kCostSingle = 2, kCostTile = 7;

// Whole tiles in waves first when the mean tile costs at least this (8k keys; at 2,048 tokens over 65k keys the pure
// cut read 6.2 GB for 0.27 GB of K/V), at most kMaxWhole a CTA.
constexpr int kWholeCost = 64 * kCostPair, kMaxWhole = 128;

enum FogMode { kNoFog = 0, kValueFog = 1, kScoreFog = 2 };

struct ChunkParams {
    void* o; int64_t o_st, o_sh;
    int num_pages, page_size;
    const int32_t* table; int64_t table_stride;
    const int32_t* start; const int32_t* seq;
    const int32_t* clear_start; float fog_alpha;
    int window, causal;
    float scale_log2;
    int B, T, Hkv, G, TH, max_seq;
    FogBias bias;
    int* status;
    // K/V boxes: tokens per box, page coordinate = page * page_mul + head * head_in_page, third coordinate =
    // head * head_in_row; split: one box per 64 dims into separate half tiles
    int box, page_mul, head_in_page, head_in_row, split;
    int oob_page;                            // page coordinate that reads zeros
    char* ws;
};

template <int D> struct Cfg {
    static constexpr int DH = D / 64;
    static constexpr int kTile = 128 * D * 2;          // one K, V or Q half tile
    static constexpr int kNK = D == 128 ? 2 : 4;
    static constexpr int kNV = D == 128 ? 2 : 4;
    static constexpr int kQ = 0;                       // two half slots
    static constexpr int kK = 2 * kTile;
    static constexpr int kV = kK + kNK * kTile;
    static constexpr int kW = kV + kNV * kTile;        // fog weights
    static constexpr int kMl = kW + kWStages * 128 * 4;    // (m, l) of a single tile's B chain
    static constexpr int kBar = kMl + 128 * 8;
    static constexpr int kNumBar = 4 + 2 * kNK + 2 * kNV + 2 * kWStages + 2 + 2 + 2 + 2 + 2;
    static constexpr int kPlan = kBar + kNumBar * 8;   // plan result and TMEM slot
    static constexpr int kWalk = kPlan + 96;           // a Walker per warp
    static constexpr int kWhole = kWalk + (kThreads / 32) * 128;   // whole tiles of this CTA
    static constexpr int kBytes = kWhole + kMaxWhole * 12;
    static constexpr int kAlloc = kBytes + 1024;
    static_assert(kNV * kTile >= kMaxBatch * 8 && kNK * kTile >= kMaxBatch * 4, "the plan's prefix sums use the rings");
    // partial slot in the workspace: O float4 [D / 4][256 rows], (m, l) float2 [256]
    static constexpr size_t kSlotBytes = (size_t)256 * D * 4 + 256 * 8;
};

// What the merge needs to know of a CTA's range: no pieces, a first piece that starts its tile, or one that does not.
enum PieceState { kNoPiece = 0, kStartsTile = 1, kMidTile = 2 };
struct PieceDesc { int state, ends, b, hk, tok0, ntok, row0, pad; };

struct Seq { int n, q0, kv, row0; };

// This CTA's range [u0, u1) of the plan and the tile (sequence b, KV head hk, tile i, at pos) that u0 lies in.
struct Plan { int64_t u0, u1, pos; int b, hk, i, any; Seq s; int whole; };
struct WholeTile { int b, hk, i; };

__device__ __forceinline__ Seq load_seq(const ChunkParams& p, int b, bool* bad = nullptr) {
    const int s0 = __ldg(p.start + b), s1 = __ldg(p.start + b + 1), len = __ldg(p.seq + b);
    Seq s;
    s.row0 = min(max(s0, 0), p.T);
    const int e = max(s.row0, min(s1, p.T));
    s.n = e - s.row0;
    s.kv = min(max(len, 0), p.max_seq);
    s.q0 = len - s.n;
    if (bad && (s.row0 != s0 || e != s1 || s.kv != len)) *bad = true;
    return s;
}

// Key range of tile i of a sequence: keys [j_lo, j_hi), key tiles [t_lo, t_hi) (at least one).
struct TileKeys { int ntok, j_lo, j_hi, t_lo, t_hi; bool single; };

__device__ __forceinline__ TileKeys tile_keys(const ChunkParams& p, const Seq& s, int i) {
    TileKeys k;
    const int tok0 = i * 2 * p.TH;
    k.ntok = min(s.n - tok0, 2 * p.TH);
    k.single = k.ntok <= p.TH;
    const int p_lo = s.q0 + tok0, p_hi = p_lo + k.ntok - 1;
    k.j_hi = (p.causal || p.window > 0) ? max(0, min(s.kv, p_hi + 1)) : s.kv;
    k.j_lo = p.window > 0 ? min(max(p_lo - p.window + 1, 0), k.j_hi) : 0;
    k.t_lo = k.j_lo >> 7;
    k.t_hi = max(k.t_lo + 1, (k.j_hi + 127) >> 7);
    return k;
}
__device__ __forceinline__ int tile_cost(const TileKeys& k) {
    return (k.t_hi - k.t_lo) * (k.single ? kCostSingle : kCostPair) + kCostTile;
}
// Key tile of a tile's range at plan position x (relative to the tile's start).
__device__ __forceinline__ int key_tile_at(const TileKeys& k, int64_t x) {
    const int y = (int)max((int64_t)0, min(x - kCostTile, (int64_t)INT_MAX - 8));
    return min(k.single ? (y + kCostSingle - 1) / kCostSingle : (y + kCostPair - 1) / kCostPair, k.t_hi - k.t_lo);
}



// One piece of work: key tiles [k0, k1) of tile i of (b, hk).
struct Item {
    int b, hk, tok0, ntok, row0, q0, kv, j_lo, j_hi;
    int key0;                 // first key of the piece's first key tile
    int n;                    // key tiles
    bool single, first, last; // one half; starts / ends with its tile
};

// Walks the pieces of this CTA's range.  Every warp walks them for itself, in
// shared memory: lane 0 steps, all lanes read the piece.
struct Walker {
    int64_t u0, u1, pos;
    const WholeTile* tiles;
    int b, hk, i, whole;
    Seq s;
    bool more, has;
    Item it;
    __device__ void begin(const Plan& pl, const WholeTile* list, int lane) {
        if (lane == 0) {
            tiles = list; whole = pl.whole;
            u0 = pl.u0; u1 = pl.u1; pos = pl.pos; b = pl.b; hk = pl.hk; i = pl.i; s = pl.s; more = pl.any != 0;
        }
        __syncwarp();
    }
    __device__ bool next(const ChunkParams& p, int lane) {
        __syncwarp();
        if (lane == 0) has = step(p);
        __syncwarp();
        return has;
    }
    __device__ void piece(const ChunkParams& p, const Seq& q, const TileKeys& k, int b_, int hk_, int i_, int a, int e) {
        it.b = b_; it.hk = hk_; it.tok0 = i_ * 2 * p.TH; it.ntok = k.ntok; it.row0 = q.row0 + it.tok0;
        it.q0 = q.q0 + it.tok0; it.kv = q.kv; it.j_lo = k.j_lo; it.j_hi = k.j_hi;
        it.key0 = (k.t_lo + a) << 7; it.n = e - a; it.single = k.single;
        it.first = a == 0; it.last = e == k.t_hi - k.t_lo;
    }
    __device__ bool step(const ChunkParams& p) {
        if (whole > 0) {
            const WholeTile w = *tiles;
            ++tiles;
            --whole;
            const Seq q = load_seq(p, w.b);
            const TileKeys k = tile_keys(p, q, w.i);
            piece(p, q, k, w.b, w.hk, w.i, 0, k.t_hi - k.t_lo);
            return true;
        }
        while (more) {
            const TileKeys k = tile_keys(p, s, i);
            const int cost = tile_cost(k);
            piece(p, s, k, b, hk, i, key_tile_at(k, u0 - pos), key_tile_at(k, u1 - pos));
            // on to the next tile
            pos += cost;
            if (pos >= u1) more = false;
            else if ((i + 1) * 2 * p.TH < s.n) ++i;
            else {
                i = 0;
                if (++hk == p.Hkv) {
                    hk = 0;
                    do {
                        if (++b >= p.B) { more = false; break; }
                        s = load_seq(p, b);
                    } while (s.n == 0);
                }
            }
            if (it.n > 0) return true;
        }
        return false;
    }
};

// Inclusive sum over the block's threads of x; *total gets the whole sum.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* wsum, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) x += wsum[w];
        all += wsum[w];
    }
    __syncthreads();
    *total = all;
    return x;
}
// First index whose inclusive prefix (times mul) is above x.
template <typename T>
__device__ __forceinline__ int first_above(const T* pre, int n, int64_t mul, int64_t x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)pre[mid] * mul > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}
// The flat-th tile of the batch in (sequence, KV head, tile) order; cnt: prefix sums of the sequences' tiles.
__device__ __forceinline__ WholeTile tile_of(const ChunkParams& p, const int* cnt, int64_t flat) {
    WholeTile w;
    w.b = first_above(cnt, p.B, p.Hkv, flat);
    const int before = w.b ? cnt[w.b - 1] : 0, nt = cnt[w.b] - before;
    const int rem = (int)(flat - (int64_t)before * p.Hkv);
    w.hk = rem / nt;
    w.i = rem - w.hk * nt;
    return w;
}

// This CTA's share of the plan (all threads; pre and cnt: shared scratch for B prefix sums of cost and tiles).
__device__ __forceinline__ void make_plan(const ChunkParams& p, int64_t* pre, int* cnt, int64_t* wsum, Plan* out,
                                          WholeTile* list) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t ctas = gridDim.x;
    int64_t W = 0, tiles = 0;
    bool bad = false, unordered = false;
    const int TT = 2 * p.TH;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
        const int b = b0 + tid;
        Seq s{0, 0, 0, 0};
        if (b < p.B) {
            s = load_seq(p, b, &bad);
            unordered |= __ldg(p.start + b + 1) < __ldg(p.start + b);
        }
        const int nt = (s.n + TT - 1) / TT;
        int64_t c = 0;
        if (nt <= 2)
            for (int i = 0; i < nt; ++i) c += tile_cost(tile_keys(p, s, i));
        // long sequences: the warp's lanes share the tiles
        for (unsigned m = __ballot_sync(0xffffffffu, nt > 2); m; m &= m - 1) {
            const int src = __ffs(m) - 1;
            Seq t;
            t.n = __shfl_sync(0xffffffffu, s.n, src);
            t.q0 = __shfl_sync(0xffffffffu, s.q0, src);
            t.kv = __shfl_sync(0xffffffffu, s.kv, src);
            t.row0 = 0;
            const int tn = (t.n + TT - 1) / TT;
            int64_t x = 0;
            for (int i = lane; i < tn; i += 32) x += tile_cost(tile_keys(p, t, i));
#pragma unroll
            for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            if (lane == src) c = x;
        }
        // one scan for both sums: tiles (below 2^24: rows of q) above the cost (below 2^40)
        int64_t all;
        const int64_t both = block_scan(((int64_t)nt << 40) | c, wsum, &all);
        const int64_t mask = (1ll << 40) - 1;
        if (b < p.B) {
            pre[b] = W + (both & mask);
            cnt[b] = (int)(tiles + (both >> 40));
        }
        W += all & mask;
        tiles += all >> 40;
    }
    if (bad && blockIdx.x == 0) record_status(p.status, KESSIE_DEV_BAD_ARG);
    W *= p.Hkv;                                    // pre stays per head
    // starts that fall would let sequences share rows, without a bound on the tiles: nothing is computed
    if (__syncthreads_or(unordered)) W = tiles = 0;
    // whole tiles first, where several share a long context
    const int64_t n_tiles = tiles * p.Hkv;
    int whole = 0;
    if (W >= n_tiles * kWholeCost && n_tiles >= 2 * (int64_t)p.B * p.Hkv) whole = (int)min(n_tiles / ctas, (int64_t)kMaxWhole);
    int64_t u_first = 0, u0, u1;
    if (whole) {
        // the cut part gives each CTA what its whole tiles leave of an equal share
        int64_t share = 0, total;
        if (tid < ctas) {
            share = (W + ctas - 1) / ctas;
            for (int k = 0; k < whole; ++k) {
                const WholeTile w = tile_of(p, cnt, tid + k * ctas);
                share -= tile_cost(tile_keys(p, load_seq(p, w.b), w.i));
            }
            share = max(share, (int64_t)0);
        }
        if (tid < whole) list[tid] = tile_of(p, cnt, blockIdx.x + tid * ctas);
        const int64_t upto = block_scan(share, wsum, &total);
        if (tid == blockIdx.x) { wsum[16] = upto - share; wsum[17] = upto; }
        __syncthreads();
        u_first = W;
        if (whole * ctas < n_tiles) {
            const WholeTile w = tile_of(p, cnt, whole * ctas);
            const Seq s = load_seq(p, w.b);
            const int64_t base = w.b ? pre[w.b - 1] : 0;
            u_first = base * p.Hkv + w.hk * (pre[w.b] - base);
            int64_t x = 0;
            for (int i = lane; i < w.i; i += 32) x += tile_cost(tile_keys(p, s, i));
#pragma unroll
            for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            u_first += x;
        }
        const double f = total > 0 ? (double)(W - u_first) / (double)total : 0.0;
        u0 = u_first + (int64_t)((double)wsum[16] * f);
        u1 = blockIdx.x == ctas - 1 ? W : u_first + (int64_t)((double)wsum[17] * f);
    } else {
        // at least one key tile a range
        const int64_t L = max((W + ctas - 1) / ctas, (int64_t)(2 * kCostPair));
        u0 = min(blockIdx.x * L, W);
        u1 = min(u0 + L, W);
    }
    if (warp == 0) {
        Plan pl{u0, u1, 0, 0, 0, 0, u0 < u1 ? 1 : 0, Seq{0, 0, 0, 0}, whole};
        if (pl.any) {
            pl.b = first_above(pre, p.B, p.Hkv, u0);
            const int64_t before = pl.b ? pre[pl.b - 1] : 0, per_head = pre[pl.b] - before;
            const int64_t base = before * p.Hkv;
            pl.hk = (u0 - base) >> 32 || per_head >> 32 ? (int)((u0 - base) / per_head)
                                                        : (int)((uint32_t)(u0 - base) / (uint32_t)per_head);
            int64_t at = base + pl.hk * per_head;
            const Seq s = load_seq(p, pl.b);
            pl.s = s;
            for (int i0 = 0;; i0 += 32) {
                const int i = i0 + lane;
                int64_t c = i * TT < s.n ? tile_cost(tile_keys(p, s, i)) : 0;
                const int64_t own = c;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int64_t y = __shfl_up_sync(0xffffffffu, c, d);
                    if (lane >= d) c += y;
                }
                const unsigned m = __ballot_sync(0xffffffffu, at + c > u0);
                if (m) {
                    const int src = __ffs(m) - 1;
                    pl.i = i0 + src;
                    pl.pos = at + __shfl_sync(0xffffffffu, c - own, src);
                    break;
                }
                at += __shfl_sync(0xffffffffu, c, 31);
                if ((i0 + 32) * TT >= s.n) { pl.any = 0; break; }      // not reached: the head holds u0
            }
        }
        if (lane == 0) *out = pl;
    }
}

__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, int n) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0], %1;\n\t}"
                 :: "r"(ptx::smem_u32(bar)), "r"(n) : "memory");
}
// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_lane() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// tcgen05.mma with the operand descriptors as two words each: stepping through
// an operand only adds to the low word (the address field), so a step costs
// the issuing thread one 32-bit add instead of rebuilding a 64-bit descriptor.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
__device__ __forceinline__ uint32_t desc_hi(uint32_t sbo) { return (sbo >> 4) | 1u << 14 | 2u << 29; }
template <bool ACCUM>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t alo, uint32_t ahi, uint32_t blo, uint32_t bhi, uint32_t idesc) {
    asm volatile("{\n\t.reg .b64 a, b;\n\t.reg .pred p;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
                 "setp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}"
                 :: "r"(d), "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "n"(ACCUM ? 1 : 0) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t bhi, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n\t.reg .b64 b;\n\t.reg .pred p;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
                 :: "r"(d), "r"(a), "r"(blo), "r"(bhi), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity));
}

// Key tiles of a piece, from its first on, that need per-key weights.
template <int FOG>
__device__ __forceinline__ int fog_tiles(const ChunkParams& p, const Item& it, int edge) {
    if (FOG == kNoFog) return 0;
    if (FOG == kScoreFog && p.bias.recall) return it.n;
    return edge <= it.key0 ? 0 : min(it.n, ((edge - it.key0 - 1) >> 7) + 1);     // holds for an edge of INT_MAX
}
// First key past the fog of a sequence.
template <int FOG>
__device__ __forceinline__ int fog_edge(const ChunkParams& p, int b, int kv) {
    if (FOG == kValueFog) return __ldg(p.clear_start + b);
    if (FOG == kScoreFog) return fog_bias_boundary(p.bias, kv);
    return 0;
}

// Score-fog bias of the four keys from `key` (a multiple of 4), times log2 e:
// fog_bias_at without branches, so that the four run side by side.  The
// product with the double reciprocal rounds to the same fp32 as the division:
// a quotient of two 24-bit numbers is never within 2^-50 (relative) of a
// midpoint of fp32.
__device__ __forceinline__ float4 score_fog4(const FogBias& f, int fb, double inv_fb, int key, int kv) {
    uint32_t bits = 0;
    if (f.recall && key < f.recall_nbits) bits = __ldg(f.recall + (key >> 5)) >> (key & 31);
    const float boost = fog_bias_round(f.boost, f.round_mode) * kLog2e;
    float4 out;
    float* w = &out.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int j = key + e, m = f.round_mode;
        const float pos = fog_bias_round((float)j, m);
        const float t = fog_bias_round((float)((double)pos * inv_fb), m);
        float d = fog_bias_round(1.0f - t, m);
        d = fog_bias_round(d * d, m);
        d = j < fb ? fog_bias_round(d * f.neg_alpha, m) * kLog2e : 0.f;
        if (j < f.recall_nbits && ((bits >> e) & 1u)) d = boost;
        w[e] = j < kv ? d : 0.f;
    }
    return out;
}

// Four weights from shared memory, in program order: left to itself the
// compiler gathers all 32 loads of a tile in front, and spills.
__device__ __forceinline__ void lds_quad(ulonglong2& w, uint32_t saddr) {
    asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(w.x), "=l"(w.y) : "r"(saddr));
}

// p = 2^(s * scale + nb) of one row's 128 scores (nb: minus the reference, plus
// fp16's headroom), packed to 16-bit pairs over the first 64 columns of the
// row's S; FOG == kValueFog with `wts`: p * w is packed.  Returns the row sum of
// the unweighted, unrounded p.
template <bool BF16, bool WEIGHTED>
__device__ __forceinline__ float softmax_p(const uint32_t (&sv)[4][32], uint32_t sreg, float scale, float nb,
                                           const float* wts, uint64_t* half_bar) {
    const uint64_t sc2 = ptx::f2_pack(scale, scale), nb2 = ptx::f2_pack(nb, nb);
    uint64_t sum[2] = {0ull, 0ull};
    // quads of weights on their way: 1 ahead 1,073 us, 4 1,037, 6 1,014, 8 1,065, 12 1,037 (2,048 tokens over 32,768
    // keys); the score fog's reads show no difference between 1 and 8
    constexpr int kAhead = 6;
    const uint32_t wa = WEIGHTED ? ptx::smem_u32(wts) : 0u;
    ulonglong2 w[kAhead];
    if (WEIGHTED)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) lds_quad(w[k], wa + k * 16);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint64_t s2 = ptx::f2_pack(__uint_as_float(sv[c][2 * i]), __uint_as_float(sv[c][2 * i + 1]));
            float e0, e1;
            ptx::f2_unpack(ptx::ffma2(s2, sc2, nb2), e0, e1);
            float p0 = ptx::ex2(e0), p1 = ptx::ex2(e1);
            const uint64_t p2 = ptx::f2_pack(p0, p1);
            sum[i & 1] = ptx::fadd2(sum[i & 1], p2);
            if (WEIGHTED) {
                const int quad = c * 8 + (i >> 1);
                ptx::f2_unpack(ptx::fmul2(p2, i & 1 ? w[quad % kAhead].y : w[quad % kAhead].x), p0, p1);
                if ((i & 1) && quad + kAhead < 32) lds_quad(w[quad % kAhead], wa + (quad + kAhead) * 16);
            }
            pk[i] = ptx::pack2<BF16>(p0, p1);
        }
        ptx::tmem_st16(sreg + c * 16, pk);
        if (c == 2) {
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            __syncwarp();
            if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(half_bar);
        }
    }
    ptx::tmem_st_wait();
    float a0, a1, b0, b1;
    ptx::f2_unpack(sum[0], a0, a1);
    ptx::f2_unpack(sum[1], b0, b1);
    return (a0 + a1) + (b0 + b1);
}

template <int D, bool BF16, int FOG>
__global__ void __launch_bounds__(kThreads, 1) fog_chunks_kernel(const __grid_constant__ CUtensorMap tmQ,
                                                                 const __grid_constant__ CUtensorMap tmK,
                                                                 const __grid_constant__ CUtensorMap tmV,
                                                                 const __grid_constant__ ChunkParams p) {
    using C = Cfg<D>;
    constexpr int DH = C::DH;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBar);
    uint64_t* q_full = bars;                       // [2] half slots
    uint64_t* q_empty = q_full + 2;
    uint64_t* k_full = q_empty + 2;
    uint64_t* k_empty = k_full + C::kNK;
    uint64_t* v_full = k_empty + C::kNK;
    uint64_t* v_empty = v_full + C::kNV;
    uint64_t* w_full = v_empty + C::kNV;
    uint64_t* w_empty = w_full + kWStages;
    uint64_t* s_full = w_empty + kWStages;         // [2] chains A, B
    uint64_t* p_full = s_full + 2;
    uint64_t* o_full = p_full + 2;
    uint64_t* o_free = o_full + 2;                 // every softmax warp is done with the piece's O
    uint64_t* ml_full = o_free + 1;                // B's (m, l) of a single tile
    uint64_t* ph_full = ml_full + 1;               // [2] first three quarters of P
    Plan* plan = reinterpret_cast<Plan*>(smem + C::kPlan);
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::kPlan + 80);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&q_full[i], 1); ptx::mbar_init(&q_empty[i], 2);
            ptx::mbar_init(&s_full[i], 1); ptx::mbar_init(&p_full[i], 4); ptx::mbar_init(&ph_full[i], 4); ptx::mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < C::kNK; ++i) { ptx::mbar_init(&k_full[i], 1); ptx::mbar_init(&k_empty[i], 2); }
        for (int i = 0; i < C::kNV; ++i) { ptx::mbar_init(&v_full[i], 1); ptx::mbar_init(&v_empty[i], 2); }
        for (int i = 0; i < kWStages; ++i) { ptx::mbar_init(&w_full[i], 1); ptx::mbar_init(&w_empty[i], kSoftmaxWarps); }
        ptx::mbar_init(o_free, kSoftmaxWarps);
        ptx::mbar_init(ml_full, 4);
        ptx::fence_mbar_init();
    }
    if (warp == 9) {
        ptx::tmem_alloc(slot, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::launch_dependents();                      // the merge waits for this grid's end by itself
    make_plan(p, reinterpret_cast<int64_t*>(smem + C::kV), reinterpret_cast<int*>(smem + C::kK),
              reinterpret_cast<int64_t*>(smem + C::kMl), plan, reinterpret_cast<WholeTile*>(smem + C::kWhole));
    ptx::fence_proxy_async_smem();                 // the plan's scratch becomes the K and V rings
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *slot;
    static_assert(sizeof(Walker) <= 128 && sizeof(Plan) <= 80, "plan and walker slots");
    Walker& walk = *reinterpret_cast<Walker*>(smem + C::kWalk + warp * 128);
    walk.begin(*plan, reinterpret_cast<const WholeTile*>(smem + C::kWhole), lane);
    const Item& it = walk.it;

    if (warp >= kSoftmaxWarps) {
    // ==================================================================== producer warpgroup
    ptx::setmaxnreg_dec<kProducerRegs>();
    if (warp == 8 || warp == 10) {
        // ================================================================ producers: Q and K / V
        const bool is_k = warp == 8;
        const int NS = is_k ? C::kNK : C::kNV;
        uint64_t* full = is_k ? k_full : v_full;
        uint64_t* empty = is_k ? k_empty : v_empty;
        const CUtensorMap* map = is_k ? &tmK : &tmV;
        uint8_t* ring = smem + (is_k ? C::kK : C::kV);
        const int nbox = 128 / p.box;
        const int my_box = lane % nbox, my_half = p.split ? lane / nbox : 0;
        const bool loads = lane < nbox * (p.split ? DH : 1);
        uint32_t count = 0, qcount = 0, wcount = 0;
        bool ok = true;
        if (lane == 0) ptx::prefetch_tensormap(map);
        while (ok && walk.next(p, lane)) {
            if (is_k) {
                // the piece's Q half tiles into the next half slots
                for (int x = 0; x < (it.single ? 1 : 2) && ok; ++x, ++qcount) {
                    const int sl = qcount & 1;
                    if (lane == 0) {
                        ok = qcount < 2 || ptx::mbar_wait(&q_empty[sl], ((qcount >> 1) & 1u) ^ 1u);
                        if (ok) {
                            ptx::mbar_arrive_expect_tx(&q_full[sl], (uint32_t)(p.TH * p.G * D * 2));
                            for (int dh = 0; dh < DH; ++dh)
                                ptx::tma_load_5d(smem + C::kQ + sl * C::kTile + dh * 16384, &tmQ, &q_full[sl], 0, 0,
                                                 it.row0 + x * p.TH, dh, it.hk);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                }
            }
            // this lane's page of the piece's key tiles, read one tile ahead;
            // pages without a key that the tile sees are neither looked up nor read
            const int32_t* row = p.table + (int64_t)it.b * p.table_stride;
            auto page_of = [&](int t) -> int {
                const int key = it.key0 + t * 128 + my_box * p.box;
                if (!loads || t >= it.n || key >= it.j_hi || key + p.box <= it.j_lo) return -1;
                return __ldg(row + key / p.page_size);
            };
            int nxt = page_of(0);
            // fog weights of key tile t, two tiles ahead of its V: that V's stage was free, so this slot is
            const int edge = is_k ? 0 : fog_edge<FOG>(p, it.b, it.kv);
            const int nw = is_k ? 0 : fog_tiles<FOG>(p, it, edge);
            const float inv_den = 1.f / (float)(max(edge, 2) - 1);
            const double inv_fb = FOG == kScoreFog ? 1.0 / (double)(float)max(edge, 1) : 0.0;
            auto weights = [&](int t) {
                if (FOG == kNoFog || t >= nw) return;
                const uint32_t c = wcount++;
                const int st = c % kWStages;
                if (c >= (uint32_t)kWStages && !wait_all(&w_empty[st], ((c / kWStages) & 1u) ^ 1u)) { ok = false; return; }
                float4 w4;
                const int key = it.key0 + t * 128 + lane * 4;
                if (FOG == kValueFog) {         // (key / (cs - 1))^alpha as 2^(alpha log2 ..), kessie_hip_kernels.py:411-412
                    float* w = &w4.x;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = key + e >= edge ? 1.f : ptx::ex2(p.fog_alpha * ptx::lg2((float)(key + e) * inv_den));
                } else {
                    w4 = score_fog4(p.bias, edge, inv_fb, key, it.kv);
                }
                reinterpret_cast<float4*>(smem + C::kW)[st * 32 + lane] = w4;
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&w_full[st]);
            };
            weights(0);
            weights(1);
            for (int t = 0; t < it.n && ok; ++t, ++count) {
                int page = nxt;
                nxt = page_of(t + 1);
                const int key = it.key0 + t * 128 + my_box * p.box;
                if (loads && key < it.j_hi && key + p.box > it.j_lo && (page < 0 || page >= p.num_pages)) {
                    record_status(p.status, KESSIE_DEV_BAD_PAGE_ID);
                    page = -1;
                }
                const int st = count % NS;
                if (lane == 0) {
                    ok = count < (uint32_t)NS || ptx::mbar_wait(&empty[st], ((count / NS) & 1u) ^ 1u);
                    if (ok) ptx::mbar_arrive_expect_tx(&full[st], (uint32_t)C::kTile);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (ok && loads) {
                    const int tok = key % p.page_size;
                    const int c4 = page < 0 ? p.oob_page : page * p.page_mul + it.hk * p.head_in_page;
                    uint8_t* dst = ring + st * C::kTile;
                    if (p.split) ptx::tma_load_5d(dst + my_half * 16384 + my_box * p.box * 128, map, &full[st], 0, tok, my_half, it.hk, c4);
                    else ptx::tma_load_5d(dst + my_box * p.box * D * 2, map, &full[st], 0, 0, it.hk * p.head_in_row, tok >> 3, c4);
                }
                __syncwarp();
                weights(t + 2);
            }
        }
        // every issued load has landed before the CTA can exit
        if (lane == 0) {
            if (!ok) record_status(p.status, KESSIE_DEV_WAIT_TIMEOUT);
            for (uint32_t c = count > (uint32_t)NS ? count - NS : 0; c < count; ++c)
                if (!ptx::mbar_wait(&full[c % NS], (c / NS) & 1u)) break;
            for (uint32_t c = qcount > 2 ? qcount - 2 : 0; c < qcount; ++c)
                if (!ptx::mbar_wait(&q_full[c & 1], (c >> 1) & 1u)) break;
        }
    } else if (elect_lane()) {
        // ================================================================ MMA issuers: warp 9 chain A, warp 11 chain B
        // A K or V stage is released by two arrivals: one of each chain (pair tiles), or two of the only one that
        // used it (single tiles).  The piece's Q slots get one arrival of each chain, so that neither chain can pass
        // a phase that the other still waits for.
        const int x = warp == 9 ? 0 : 1;
        const uint32_t idS = ptx::umma_idesc_f16(BF16, false, 128);
        const uint32_t idPV = ptx::umma_idesc_f16(BF16, true, D);
        // 8-row groups of a K/V tile: 1024 * DH apart with the halves interleaved, or 1024 in split half tiles
        const uint32_t grp = p.split ? 1024u : 1024u * DH, half_off = p.split ? 16384u : 1024u;
        const uint32_t q_base = ptx::smem_u32(smem + C::kQ), k_base = ptx::smem_u32(smem + C::kK), v_base = ptx::smem_u32(smem + C::kV);
        const uint32_t q_hi = desc_hi(1024), kv_hi = desc_hi(grp);
        const uint32_t tS = tmem + x * 128, tO = tmem + 256 + x * 128;
        uint32_t tiles = 0, qc = 0, last_q = 0, pc = 0, items = 0;               // running stage / phase counters
        bool ok = true;
        Walker w = walk;                                             // this thread's own copy
        while (ok && w.step(p)) {
            const bool single = w.it.single;
            const int n = w.it.n, nev = single ? (n + 1 - x) >> 1 : n;
            const uint32_t slot_c = single ? qc : qc + x, q_slot = slot_c & 1u;
            const uint32_t qlo = desc_lo(q_base + q_slot * C::kTile, 16);
            auto issue_s = [&](int ev) {
                const uint32_t t = tiles + (single ? 2 * ev + x : ev), st = t % C::kNK;
                ok = ok && ptx::mbar_wait(&k_full[st], (t / C::kNK) & 1u);
                if (!ok) return;
                ptx::tc_fence_after();
                const uint32_t klo = desc_lo(k_base + st * C::kTile, 16);
                mma_ss<false>(tS, qlo, q_hi, klo, kv_hi, idS);
#pragma unroll
                for (int kk = 1; kk < D / 16; ++kk)
                    mma_ss<true>(tS, qlo + (kk >> 2) * 1024 + (kk & 3) * 2, q_hi,
                                 klo + (kk >> 2) * (half_off >> 4) + (kk & 3) * 2, kv_hi, idS);
                ptx::umma_commit(&s_full[x]);
                ptx::umma_commit(&k_empty[st]);
                if (single) ptx::umma_commit(&k_empty[st]);
                if (ev == nev - 1) {                                 // the last scores: one arrival for each Q slot
                    ptx::umma_commit(&q_empty[qc & 1u]);
                    if (!single) ptx::umma_commit(&q_empty[(qc + 1) & 1u]);
                }
            };
            // Parity waits tell a phase only from its neighbours, and in a single tile a chain passes over the
            // stages of the other: before this piece's first K, all scores of the last piece are done (its Q slots
            // are free), before its first V, all products (o_free).
            for (uint32_t c = qc - last_q; c != qc && ok; ++c) ok = ptx::mbar_wait(&q_empty[c & 1u], (c >> 1) & 1u);
            last_q = single ? 1 : 2;
            ok = ok && ptx::mbar_wait(&q_full[q_slot], (slot_c >> 1) & 1u);
            if (ok && nev > 0) issue_s(0);
            for (int ev = 0; ev < nev && ok; ++ev) {
                const uint32_t t = tiles + (single ? 2 * ev + x : ev), st = t % C::kNV;
                const uint32_t vlo = desc_lo(v_base + st * C::kTile, half_off);
                // the first product overwrites O: the last piece's has been read
                if (ev == 0 && items > 0) ok = ptx::mbar_wait(o_free, (items - 1) & 1u);
                ok = ok && ptx::mbar_wait(&v_full[st], (t / C::kNV) & 1u);
                ok = ok && ptx::mbar_wait(&ph_full[x], pc & 1u);
                if (!ok) break;
                ptx::tc_fence_after();
                mma_ts(tO, tS, vlo, kv_hi, idPV, ev > 0 ? 1u : 0u);
#pragma unroll
                for (int kk = 1; kk < 6; ++kk) mma_ts(tO, tS + kk * 8, vlo + kk * (grp >> 3), kv_hi, idPV, 1u);
                ok = ptx::mbar_wait(&p_full[x], pc & 1u);
                ++pc;
                if (!ok) break;
                ptx::tc_fence_after();
#pragma unroll
                for (int kk = 6; kk < 8; ++kk) mma_ts(tO, tS + kk * 8, vlo + kk * (grp >> 3), kv_hi, idPV, 1u);
                ptx::umma_commit(&v_empty[st]);
                if (single) ptx::umma_commit(&v_empty[st]);
                // last: who sees it has seen every arrival of this thread's MMAs, so none is under way when the CTA ends
                if (ev == nev - 1) ptx::umma_commit(&o_full[x]);
                if (ev + 1 < nev) issue_s(ev + 1);
            }
            if (nev == 0 && ok) {                                    // a single tile's only key tile is chain A's
                if (items > 0) ok = ptx::mbar_wait(o_free, (items - 1) & 1u);
                ptx::mbar_arrive(&q_empty[q_slot]);
                ptx::mbar_arrive(&o_full[x]);
            }
            tiles += n;
            qc += single ? 1 : 2;
            ++items;
        }
        if (!ok) record_status(p.status, KESSIE_DEV_WAIT_TIMEOUT);
    }
    } else {
        // ================================================================ softmax warpgroups
        ptx::setmaxnreg_inc<kSoftmaxRegs>();
        const int x = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t sreg = tmem + lane_off + (uint32_t)(x * 128);
        const uint32_t oreg = tmem + lane_off + 256;
        const float* wring = reinterpret_cast<const float*>(smem + C::kW);
        float2* mlbuf = reinterpret_cast<float2*>(smem + C::kMl);
        uint32_t sc = 0, wc = 0, tiles = 0, items = 0, singles = 0;
        bool ok = true;
        PieceDesc desc{0, 0, 0, 0, 0, 0, 0, 0};
        const int r_tok = r / p.G, gh = r - r_tok * p.G;             // row: token of the half, head of the group
        const int rows_half = p.TH * p.G;
        const int w_tok0 = (q4 * 32) / p.G, w_tok1 = min(q4 * 32 + 31, rows_half - 1) / p.G;
        while (ok && walk.next(p, lane)) {
            if (!it.first) desc = PieceDesc{kMidTile, it.last ? 1 : 0, it.b, it.hk, it.tok0, it.ntok, it.row0, 0};
            else if (!it.last && desc.state == kNoPiece) desc.state = kStartsTile;
            const int nev = it.single ? (it.n + 1 - x) >> 1 : it.n;
            const int edge = fog_edge<FOG>(p, it.b, it.kv);
            const int nw = fog_tiles<FOG>(p, it, edge);
            // this thread's row: token and head of the group
            const int base_tok = it.single ? 0 : x * p.TH;
            const int tok = base_tok + r_tok;
            const bool valid = r < rows_half && tok < it.ntok;
            const bool any = __any_sync(0xffffffffu, valid);
            const int pos = it.q0 + tok;
            const bool limited = p.causal || p.window > 0;
            int hi_r = limited ? min(it.kv, pos + 1) : it.kv;
            int lo_r = p.window > 0 ? pos - p.window + 1 : 0;
            if (!valid) hi_r = lo_r = 0;
            // positions of the warp's rows, for the tiles that need no mask
            const int w_lo = it.q0 + base_tok + w_tok0, w_hi = it.q0 + min(it.ntok - 1, base_tok + w_tok1);
            // key tiles [t_in0, t_in1) need no mask for this warp's rows; from t_cut on (and before the window in the
            // first) a key tile holds keys that no row of the tile sees
            const bool single = it.single;
            const int key_base = it.key0, kv = it.kv;
            const int t_in1 = (min(kv, limited ? w_lo + 1 : kv) - key_base) >> 7;
            const int t_in0 = p.window > 0 ? (w_hi - p.window + 1 - key_base + 127) >> 7 : 0;
            const int t_cut = (kv - key_base) >> 7;
            const bool cut_first = key_base < it.j_lo;
            float m_used = -INFINITY, l = 0.f;
            for (int ev = 0; ev < nev; ++ev, ++sc) {
                const int t = single ? 2 * ev + x : ev;
                const bool weighted = FOG != kNoFog && t < nw;
                const uint32_t wi = (wc + t) % kWStages;
                if (weighted && !wait_all(&w_full[wi], ((wc + t) / kWStages) & 1u)) { ok = false; break; }
                if (!wait_all(&s_full[x], sc & 1u)) { ok = false; break; }
                if (t >= t_cut || (cut_first && t == 0)) {
                    // V rows of keys that no row of the tile sees (slots behind the last key, keys before the
                    // window) may hold anything: zero them, so that 0 * NaN cannot reach O.  In a pair tile both
                    // chains do (the same zeros).  o_free: see the issuers' first V.
                    const uint32_t vt = tiles + t, st = vt % C::kNV;
                    if (ev == 0 && items > 0 && !wait_all(o_free, (items - 1) & 1u)) { ok = false; break; }
                    if (!wait_all(&v_full[st], (vt / C::kNV) & 1u)) { ok = false; break; }
                    const int key0 = key_base + t * 128;
                    const int lo = min(128, max(0, it.j_lo - key0)), hi = min(128, max(lo, kv - key0));
                    uint8_t* vb = smem + C::kV + st * C::kTile;
                    const int n_zero = (lo + 128 - hi) * DH * 8;                  // rows [0, lo) and [hi, 128)
                    for (int z = r; z < n_zero; z += 128) {
                        const int zr = z / (DH * 8), vr = zr < lo ? zr : zr - lo + hi, dh = (z >> 3) % DH, ch = z & 7;
                        const uint32_t off = p.split ? dh * 16384 + vr * 128 : (vr >> 3) * 1024 * DH + dh * 1024 + (vr & 7) * 128;
                        *reinterpret_cast<uint4*>(vb + off + ch * 16) = make_uint4(0, 0, 0, 0);
                    }
                    ptx::fence_proxy_async_smem();
                }
                if (any) {
                    ptx::tc_fence_after();
                    const float* wts = wring + wi * 128;
                    uint32_t sv[4][32];
#pragma unroll
                    for (int c = 0; c < 4; ++c) ptx::tmem_ld32(sreg + c * 32, sv[c]);
                    ptx::tmem_ld_wait();
                    float scale = p.scale_log2;
                    if (FOG == kScoreFog && weighted) {
                        // to log2 units with the bias; the exponent below then has scale 1
                        const uint64_t sc2 = ptx::f2_pack(scale, scale);
                        scale = 1.f;
                        const uint32_t wa = ptx::smem_u32(wts);
                        ulonglong2 ahead[2];
                        lds_quad(ahead[0], wa);
                        lds_quad(ahead[1], wa + 16);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const int quad = c * 8 + (i >> 2);
                                const ulonglong2 b2 = ahead[quad & 1];
                                if (quad + 2 < 32) lds_quad(ahead[quad & 1], wa + (quad + 2) * 16);
                                float s0, s1, s2, s3;
                                ptx::f2_unpack(ptx::ffma2(ptx::f2_pack(__uint_as_float(sv[c][i]), __uint_as_float(sv[c][i + 1])), sc2, b2.x), s0, s1);
                                ptx::f2_unpack(ptx::ffma2(ptx::f2_pack(__uint_as_float(sv[c][i + 2]), __uint_as_float(sv[c][i + 3])), sc2, b2.y), s2, s3);
                                sv[c][i] = __float_as_uint(s0);
                                sv[c][i + 1] = __float_as_uint(s1);
                                sv[c][i + 2] = __float_as_uint(s2);
                                sv[c][i + 3] = __float_as_uint(s3);
                            }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (t >= t_in0 && t < t_in1) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; i += 2)
                                mx4[(i >> 1) & 3] = ptx::max3(mx4[(i >> 1) & 3], __uint_as_float(sv[c][i]), __uint_as_float(sv[c][i + 1]));
                    } else {
                        // bit i of seen: key c * 32 + i of the tile is in [lo_r, hi_r)
                        const int lo = lo_r - key_base - t * 128, hi = hi_r - key_base - t * 128;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int a = min(max(lo - c * 32, 0), 32), b = min(max(hi - c * 32, 0), 32);
                            const uint32_t seen = (uint32_t)((1ull << b) - 1) & ~(uint32_t)((1ull << a) - 1);
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float s = seen & (1u << i) ? __uint_as_float(sv[c][i]) : -INFINITY;
                                sv[c][i] = __float_as_uint(s);
                                mx4[i & 3] = fmaxf(mx4[i & 3], s);
                            }
                        }
                    }
                    const float m_tile = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale;
                    // the reference moves when the maximum outgrows it by 2^8 (from -inf: at once)
                    const bool need = m_tile > m_used + kRescaleThreshold;
                    const float old = m_used;
                    if (need) {
                        const float factor = ptx::ex2(m_used - m_tile);       // 0 from -inf
                        l *= factor;
                        m_used = m_tile;
                    }
                    const float nb = m_used == -INFINITY ? 0.f : BF16 ? -m_used : kHalfHeadroom - m_used;
                    const bool moved = __any_sync(0xffffffffu, need && old != -INFINITY);
                    // O moves with the reference (rare): its last product is complete, the next waits for P
                    if (moved) {
                        const float f = need && old != -INFINITY ? ptx::ex2(old - m_used) : 1.f;
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t ov[16];
                            tmem_ld16(oreg + x * 128 + c * 16, ov);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                            ptx::tmem_st16(oreg + x * 128 + c * 16, ov);
                        }
                        ptx::tmem_st_wait();
                    }
                    if (FOG == kValueFog && weighted) l += softmax_p<BF16, true>(sv, sreg, scale, nb, wts, &ph_full[x]);
                    else l += softmax_p<BF16, false>(sv, sreg, scale, nb, wts, &ph_full[x]);
                    ptx::tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) {
                    if (!any) ptx::mbar_arrive(&ph_full[x]);
                    ptx::mbar_arrive(&p_full[x]);
                    if (weighted) mbar_arrive_n(&w_empty[wi], single ? 2 : 1);
                }
            }
            if (!ok) break;
            wc += nw;
            tiles += it.n;
            // ---- end of the piece: O, m, l of this warp's rows
            if (!wait_all(&o_full[x], items & 1u)) { ok = false; break; }
            const bool mine = !it.single || x == 0;        // A writes a single tile for both chains
            float f0 = 1.f, f1 = 0.f;
            bool two = false;
            if (it.single) {
                if (x == 1) {
                    mlbuf[r] = make_float2(m_used, l);
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ml_full);
                } else {
                    if (!wait_all(&o_full[1], items & 1u) || !wait_all(ml_full, singles & 1u)) { ok = false; break; }
                    const float2 o = mlbuf[r];
                    const float m = fmaxf(m_used, o.x);
                    f0 = m_used == -INFINITY ? 0.f : ptx::ex2(m_used - m);
                    f1 = o.x == -INFINITY ? 0.f : ptx::ex2(o.x - m);
                    l = l * f0 + o.y * f1;
                    m_used = m;
                    two = it.n > 1;
                }
                ++singles;
            }
            if (mine && any) {
                ptx::tc_fence_after();
                const bool whole = it.first && it.last;
                const float inv = l > 0.f ? 1.f / l : 0.f;
                uint16_t* orow = static_cast<uint16_t*>(p.o) + (int64_t)(it.row0 + tok) * p.o_st + (int64_t)(it.hk * p.G + gh) * p.o_sh;
                char* part = p.ws + (size_t)gridDim.x * sizeof(PieceDesc) + (size_t)(2 * blockIdx.x + (it.first ? 1 : 0)) * C::kSlotBytes;
                const int prow = it.single ? r : x * 128 + r;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t ov[32];
                    ptx::tmem_ld32(oreg + x * 128 + c * 32, ov);
                    ptx::tmem_ld_wait();
                    if (it.single) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f0);
                        if (two) {
                            uint32_t o2[32];
                            ptx::tmem_ld32(oreg + 128 + c * 32, o2);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), f1, __uint_as_float(ov[i])));
                        }
                    }
                    if (valid && whole) {
                        uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            uint32_t pk[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                pk[i] = ptx::pack2<BF16>(__uint_as_float(ov[8 * v + 2 * i]) * inv, __uint_as_float(ov[8 * v + 2 * i + 1]) * inv);
                            dst[v] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                        }
                    } else if (valid) {
                        uint4* dst = reinterpret_cast<uint4*>(part) + (size_t)(c * 8) * 256 + prow;
#pragma unroll
                        for (int v = 0; v < 8; ++v) dst[v * 256] = make_uint4(ov[4 * v], ov[4 * v + 1], ov[4 * v + 2], ov[4 * v + 3]);
                    }
                    __syncwarp();                  // tcgen05.ld is warp-collective
                }
                if (valid && !whole) reinterpret_cast<float2*>(part + (size_t)256 * D * 4)[prow] = make_float2(m_used, l);
                ptx::tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(o_free);
            ++items;
        }
        if (!ok) record_status(p.status, KESSIE_DEV_WAIT_TIMEOUT);
        if (threadIdx.x == 0) reinterpret_cast<PieceDesc*>(p.ws)[blockIdx.x] = desc;
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the pieces of cut tiles: blocks (c, *) take the tile whose second piece
// opens CTA c's range, 32 rows a block, 8 columns a warp.  The tile's first
// piece is in the second slot of the CTA before, the others in the first slots of
// c, c + 1, ... to the one that ends the tile; they are joined in that order, the
// loads of kMergeBatch pieces in flight (one at a time took 32.6 us for the 19
// pieces a tile of 17 queries over 262k keys).
constexpr int kMergeBatch = 4;                       // pieces in flight

template <int D, bool BF16>
__global__ void __launch_bounds__(256) fog_chunks_merge_kernel(const ChunkParams p, int ctas) {
    ptx::grid_dependency_wait();
    const PieceDesc* desc = reinterpret_cast<const PieceDesc*>(p.ws);
    const int c = blockIdx.x + 1;
    const PieceDesc d = desc[c];
    if (d.state != kMidTile) return;
    int before = c - 1;                                          // the CTA with the piece before this one
    while (before > 0 && desc[before].state == kNoPiece) --before;
    if (desc[before].state == kMidTile && !desc[before].ends) return;      // an earlier boundary cut this tile
    __shared__ int piece[kThreads + 1];                          // the tile's pieces in order: slots
    __shared__ int count;
    if (threadIdx.x < 32) {
        // a warp looks at 32 CTAs at a time, up to the piece that ends the tile
        const int lane = threadIdx.x;
        int n = 2;
        if (lane == 0) { piece[0] = 2 * before + 1; piece[1] = 2 * c; }
        for (int k0 = c + 1, over = d.ends; !over && k0 < ctas; k0 += 32) {
            const bool in = k0 + lane < ctas;
            const bool mid = in && desc[k0 + lane].state == kMidTile;
            const unsigned mids = __ballot_sync(0xffffffffu, mid), ends = __ballot_sync(0xffffffffu, mid && desc[k0 + lane].ends);
            const unsigned upto = ends ? (ends & -ends) * 2 - 1 : 0xffffffffu;          // lanes to the end of the tile
            const unsigned mine = mids & upto;
            if ((mine >> lane) & 1u) piece[n + __popc(mine & ((1u << lane) - 1))] = 2 * (k0 + lane);
            n += __popc(mine);
            over = ends != 0;
        }
        if (lane == 0) count = n;
    }
    __syncthreads();
    const int n = count;
    const char* slots = p.ws + (size_t)ctas * sizeof(PieceDesc);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.y * 32 + lane, half = row >> 7, r = row & 127, tok = half * p.TH + r / p.G;
    const int c8 = blockIdx.z * 8 + warp;
    if (r >= p.TH * p.G || tok >= d.ntok || (half && d.ntok <= p.TH)) return;
    // running maximum over batches of pieces
    float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < n; i0 += kMergeBatch) {
        float2 ml[kMergeBatch];
        float4 x[kMergeBatch][2];
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
            const char* s = slots + (size_t)piece[min(i0 + u, n - 1)] * Cfg<D>::kSlotBytes;
            ml[u] = reinterpret_cast<const float2*>(s + (size_t)256 * D * 4)[row];
            x[u][0] = reinterpret_cast<const float4*>(s)[(2 * c8) * 256 + row];
            x[u][1] = reinterpret_cast<const float4*>(s)[(2 * c8 + 1) * 256 + row];
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
            if (i0 + u >= n) ml[u].x = -INFINITY;
            top = fmaxf(top, ml[u].x);
        }
        const float old = m == -INFINITY ? 0.f : ptx::ex2(m - top);
        l *= old;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= old;
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
            const float f = ml[u].x == -INFINITY ? 0.f : ptx::ex2(ml[u].x - top);
            l += ml[u].y * f;
            const float* v = &x[u][0].x;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += f == 0.f ? 0.f : v[i] * f;
        }
        m = top;
    }
    // only a row without keys has l = 0.  A row whose scores are NaN (its query is not finite) has a NaN l beside a
    // maximum of -inf (maxima pass NaN over), which the factors above would drop: it stays NaN, as in an uncut tile
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t pk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) pk[i] = ptx::pack2<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
    uint16_t* o = static_cast<uint16_t*>(p.o) + (int64_t)(d.row0 + tok) * p.o_st + (int64_t)(d.hk * p.G + r % p.G) * p.o_sh;
    *reinterpret_cast<uint4*>(o + c8 * 8) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
}

// Tensor map of K (or V); fills the box geometry of `p`.  The 8-row groups of
// a box need (8 tokens, D/64, token / 8) as separate dimensions, which leaves
// two for head and page: the head joins the 64-wide columns when heads are
// adjacent (head stride D), or the page when the page stride is a multiple of
// the head stride.  Other layouts load the 64-wide halves separately.
CUresult encode_kv(CUtensorMap* map, const void* base, bool bf16, int D, int64_t page_stride, int64_t token_stride,
                   int64_t head_stride, ChunkParams& p) {
    const cuuint64_t DH = D / 64;
    int box = 128;
    while (p.page_size % box) box >>= 1;
    p.box = box;
    p.split = 0;
    const cuuint64_t tok = (cuuint64_t)token_stride * 2, page = (cuuint64_t)page_stride * 2, head = (cuuint64_t)head_stride * 2;
    if (head_stride == D || p.Hkv == 1) {
        p.page_mul = 1; p.head_in_page = 0; p.head_in_row = (int)DH; p.oob_page = p.num_pages;
        const cuuint64_t dims[5] = {64, 8, DH * p.Hkv, (cuuint64_t)p.page_size / 8, (cuuint64_t)p.num_pages};
        const cuuint64_t str[4] = {tok, 128, 8 * tok, page};
        const cuuint32_t bx[5] = {64, 8, (cuuint32_t)DH, (cuuint32_t)box / 8, 1};
        return encode_tiled_5d_sw128(map, base, bf16, dims, str, bx);
    }
    const int64_t ratio = head_stride > 0 && page_stride % head_stride == 0 ? page_stride / head_stride : 0;
    const int64_t merged = ratio > 0 ? (p.num_pages - 1) * ratio + p.Hkv : 0;
    if (ratio >= p.Hkv && merged < INT_MAX) {
        p.page_mul = (int)ratio; p.head_in_page = 1; p.head_in_row = 0; p.oob_page = (int)merged;
        const cuuint64_t dims[5] = {64, 8, DH, (cuuint64_t)p.page_size / 8, (cuuint64_t)merged};
        const cuuint64_t str[4] = {tok, 128, 8 * tok, head};
        const cuuint32_t bx[5] = {64, 8, (cuuint32_t)DH, (cuuint32_t)box / 8, 1};
        return encode_tiled_5d_sw128(map, base, bf16, dims, str, bx);
    }
    p.page_mul = 1; p.head_in_page = 0; p.head_in_row = 0; p.oob_page = p.num_pages; p.split = 1;
    const cuuint64_t dims[5] = {64, (cuuint64_t)p.page_size, DH, (cuuint64_t)p.Hkv, (cuuint64_t)p.num_pages};
    const cuuint64_t str[4] = {tok, 128, head, page};
    const cuuint32_t bx[5] = {64, (cuuint32_t)box, 1, 1, 1};
    return encode_tiled_5d_sw128(map, base, bf16, dims, str, bx);
}

size_t chunks_workspace_bytes(int head_dim) {
    return (size_t)sm_count() * (sizeof(PieceDesc) + 2 * ((size_t)256 * head_dim * 4 + 256 * 8));
}

template <int D, bool BF16, int FOG>
int launch_chunks(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ChunkParams& p, int grid, cudaStream_t st) {
    auto kern = fog_chunks_kernel<D, BF16, FOG>;
    static std::atomic<uint64_t> ready{0};                    // devices on which the kernel is set up
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("paged_fog_chunks: device");
    if (dev >= 64 || !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        // setmaxnreg.inc draws on the registers of the launch: valid only if the kernel was built with kLaunchRegs
        cudaFuncAttributes fa;
        if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) return check_launch("paged_fog_chunks: attributes");
        if (fa.numRegs < kLaunchRegs)
            return set_error(KESSIE_ERR_UNSUPPORTED, "paged_fog_chunks: built with %d registers", fa.numRegs);
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kAlloc) != cudaSuccess)
            return check_launch("paged_fog_chunks: set smem attribute");
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    // held over both launches: a call of another host thread on this stream must not come between them (the
    // workspace), nor a programmatic one
    LaunchOrderGuard order;
    kern<<<grid, kThreads, Cfg<D>::kAlloc, st>>>(q, k, v, p);
    const int rc = check_launch("paged_fog_chunks");
    if (rc || grid < 2) return rc;
    // The merge is a programmatic dependent of the kernel above (its launch
    // overlaps that one's run; it reads nothing before its wait).  It signals
    // nothing early itself, and is on record for a programmatic launch behind it.
    const ByteRange wrote[2] = {byte_span(p.o, 2 * ((int64_t)(p.T - 1) * p.o_st + (int64_t)(p.Hkv * p.G - 1) * p.o_sh + D)),
                                byte_span(p.ws, (int64_t)chunks_workspace_bytes(D))};
    claim_early_reads(st, nullptr, 0, wrote, 2);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid - 1, 8, D / 64);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, fog_chunks_merge_kernel<D, BF16>, p, grid);
    return check_launch("paged_fog_chunks merge");
}

template <int D, bool BF16>
int launch_fog(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ChunkParams& p, int grid, cudaStream_t st) {
    if (p.bias.on) return launch_chunks<D, BF16, kScoreFog>(q, k, v, p, grid, st);
    if (p.clear_start) return launch_chunks<D, BF16, kValueFog>(q, k, v, p, grid, st);
    return launch_chunks<D, BF16, kNoFog>(q, k, v, p, grid, st);
}

}  // namespace
}  // namespace kessie

using namespace kessie;

extern "C" size_t kessie_paged_fog_chunks_workspace_size(int num_q_heads, int num_kv_heads, int head_dim) {
    if (num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    return chunks_workspace_bytes(head_dim);
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
    if ((num_tokens > 1 && o_stride_t == 0) || (num_q_heads > 1 && o_stride_h == 0))
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: rows of out share memory");
    const size_t need = kessie_paged_fog_chunks_workspace_size(num_q_heads, num_kv_heads, head_dim);
    if (!workspace || workspace_bytes < need)
        return set_error(KESSIE_ERR_WORKSPACE, "paged_fog_chunks_v2: workspace %zu < %zu", workspace_bytes, need);
    if (batch > kMaxBatch)
        return set_error(KESSIE_ERR_UNSUPPORTED, "paged_fog_chunks_v2: %d sequences (at most %d)", batch, kMaxBatch);
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return set_error(KESSIE_ERR_WORKSPACE, "paged_fog_chunks_v2: workspace must be 16-byte aligned");
    ChunkParams p{};
    p.o = out; p.o_st = o_stride_t; p.o_sh = o_stride_h;
    p.num_pages = num_pages; p.page_size = page_size;
    p.table = block_table; p.table_stride = block_table_stride;
    p.start = query_start_loc; p.seq = seq_lens;
    p.clear_start = fog_alpha > 0.f ? clear_start : nullptr; p.fog_alpha = fog_alpha;
    // a window as wide as the longest sequence masks no more than causality does
    const bool wide = window_size > 0 && window_size >= max_seq_len;
    p.window = window_size > 0 && !wide ? window_size : 0; p.causal = is_causal || wide ? 1 : 0;
    p.scale_log2 = sm_scale * kLog2e;
    p.B = batch; p.T = num_tokens; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads; p.TH = 128 / p.G;
    p.max_seq = max_seq_len < INT_MAX - 255 ? max_seq_len : INT_MAX - 255;     // key tiles end below 2^31
    const int brc = fog_bias_from_c(bias, &p.bias);
    if (brc) return brc;
    if (p.bias.on && p.clear_start)
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: fog on the values or on the scores, not both");
    p.status = device_status_ptr();
    p.ws = static_cast<char*>(workspace);
    const bool bf16 = dtype == KESSIE_DTYPE_BF16;
    CUtensorMap mq, mk, mv;
    // q rows as {64 dims, head in group, token, 64-dim half, KV head}
    const cuuint64_t dims[5] = {64, (cuuint64_t)p.G, (cuuint64_t)p.T, (cuuint64_t)head_dim / 64, (cuuint64_t)p.Hkv};
    const cuuint64_t str[4] = {(cuuint64_t)q_stride_h * 2, (cuuint64_t)q_stride_t * 2, 128, (cuuint64_t)p.G * q_stride_h * 2};
    const cuuint32_t bx[5] = {64, (cuuint32_t)p.G, (cuuint32_t)p.TH, 1, 1};
    const CUresult rq = encode_tiled_5d_sw128(&mq, q, bf16, dims, str, bx);
    const CUresult rk = encode_kv(&mk, k_cache, bf16, head_dim, page_stride, token_stride, head_stride, p);
    const CUresult rv = encode_kv(&mv, v_cache, bf16, head_dim, page_stride, token_stride, head_stride, p);
    if (rq != CUDA_SUCCESS || rk != CUDA_SUCCESS || rv != CUDA_SUCCESS)
        return set_error(KESSIE_ERR_ARG, "paged_fog_chunks_v2: TMA descriptor rejected (q %d, k %d, v %d)", (int)rq, (int)rk, (int)rv);
    const int grid = sm_count() < kThreads ? sm_count() : kThreads;
    cudaStream_t st = as_stream(stream);
    if (head_dim == 128) return bf16 ? launch_fog<128, true>(mq, mk, mv, p, grid, st) : launch_fog<128, false>(mq, mk, mv, p, grid, st);
    return bf16 ? launch_fog<64, true>(mq, mk, mv, p, grid, st) : launch_fog<64, false>(mq, mk, mv, p, grid, st);
}
