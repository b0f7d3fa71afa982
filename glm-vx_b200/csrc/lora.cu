// Low-rank adapters of many requests beside a shared projection:
//   y[t] += s_a * B_a (A_a x[t]),   a = adapter_ids[t]  (-1: none, row t stays)
// with A_a [rank_a][cols] and B_a [rows][rank_a] taken from stacks padded to
// max_rank.  Two kernels: lora_shrink (h = A x, f32, into the workspace, the
// columns split over CTAs) and lora_expand (the parts of h joined, y += s B h),
// the second launched while the first runs; for few tiles of small adapters one
// kernel of clusters does both.
//
// Both are products of a weight tile with a few tokens, bound by reading the
// weights (few tokens an adapter) or x and y (many): tensor-core tiles whose
// M is the weights' rows and whose N is the tokens, so that one token wastes
// only multiplications, and every operand goes from memory straight into the
// fragment that needs it: the order of K is free, so a lane takes eight
// neighbouring columns where the fragment layout names t and t + 4 of each eight.
// F16 and BF16 weights are TF32 numbers as they are; x, h and F32 weights go
// in as two, hi + lo, which leaves up to 2^-23 of them over.  With F32 weights the
// product of the two lo, up to 2^-22, is not made: a product loses 2^-23 of
// itself at most, of F32 weights 2^-21.  Sums are f32; the tensor cores cut what
// an addition leaves over, so their chains end after 64 columns (of A) or ranks
// (of B) and go on as rounded sums.  Error of the whole change against 64 bits,
// in norms, at 6144 columns of rank 16: 3.4e-7 (F32 weights 4.9e-7), of rank 256
// 5.8e-7 (7.9e-7); a plain f32 product's 1.5e-7 to 4.3e-7 and 3.1e-7 to 6.1e-7.
//
// Tokens of one adapter are gathered into tiles.  A token's sums are made in
// the same order whatever tile and place it lands in.
//
// Measured in CUDA graphs, beside the time that a copy of the bytes read and
// written takes (6.57 TB/s): 1 token, 576 x 6144, rank 8, BF16 5.1 us (0.02);
// 64 tokens of 64 adapters, 16384 x 2048, rank 16, BF16 20.9 us (7.1); 48 tokens
// of 5 adapters, 6144 x 16384, rank 64, F16 12.5 us (2.6); 1000 tokens of 11
// adapters, 2048 x 6144, rank 64, F16 32 us (7.0); 4096 tokens of 16 adapters,
// 12288 x 6144, rank 32, BF16 138 us (79.5).  Few tokens are bound by the chain
// of waits (ids, ranks, weights, h, weights), many by instructions and the L1's
// data path: of 4096 tokens' call expand takes 100 us with the LSU's data path
// at 81 % and the schedulers issuing in 42 % of the cycles, DRAM at 45 %.
#include <cuda_bf16.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.cuh"

namespace glmvx {

namespace {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraThreads = 256, kLoraWarps = kLoraThreads / 32;
// Tokens up to which each CTA finds the tiles itself (a word of bits).  More take a kernel that plans and tiles of 16:
// at 64 tokens of 64 adapters of 16384 x 2048, rank 16, that is 26.6 us against 20.8; at 40 19.1 against 13.9.
constexpr int kLoraScan = 64;
constexpr int kLoraMaxSplits = 32;
constexpr int kLoraRankChunk = 64;   // ranks a shrink CTA takes
constexpr int kLoraRows = 32;        // rows of B a warp takes at once
constexpr int kLoraChain = 64;       // ranks that expand's sums go through in the tensor cores

// A tile of the plan: n tokens of one adapter (the places behind them hold anything).
constexpr int kLoraTile = 16;
struct LoraTile {
    int adapter, n, rank, pad, tokens[kLoraTile];
};

struct LoraArgs {
    float *y;
    const float *x;
    const int32_t *ids;
    const void *a, *b;
    const int32_t *ranks;
    const float *scales;
    float *h;         // [splits][tokens][lora_h_pitch(max_rank)]
    LoraTile *tiles;  // the plan (NULL: CTAs scan the ids)
    int *counts, *places, *ntiles;
    int64_t y_stride, x_stride;
    int tokens, rows, cols, adapters, max_rank, splits, units, team;
    int how_a, how_b, how_x, how_y;  // LoraHow: how rows that are not all on 16-byte boundaries are read
    int *err;
};

__host__ __device__ constexpr int lora_h_pitch(int max_rank) { return (max_rank + 3) & ~3; }
__device__ __forceinline__ int lora_rank(const LoraArgs &p, int a) { return min(max(p.ranks[a], 0), p.max_rank); }

// N neighbouring values (4 or 8) as they stand in memory.  With VEC they are on their boundary and are read where
// n > 0.  Without it only n values may be read there, and those from n on are 0: 16 bytes at once where they are on
// that boundary, else (16-bit) four at once on theirs, else by the words of two that hold them, which has to leave
// one value behind them; else value by value.  1000 tokens, 2050 x 6146, rank 37: 66 us, value by value 88; 4096
// tokens, 12288 x 6144, rank 31: 194 us, value by value 244.
template <class W>
using LoraRaw = std::conditional_t<sizeof(W) == 4, uint4, uint2>;

enum LoraHow : int { kLoraSingle, kLoraWords, kLoraQuads, kLoraWhole };

template <class W>
struct LoraEight {
    LoraRaw<W> q[2];
};

template <class T>
__device__ __forceinline__ T lora_as(const void *from) {
    return __ldg(static_cast<const T *>(from));
}

// Words 0 .. N - 1 of the 2 N values of 16 bits at w.
template <int N>
__device__ __forceinline__ void lora_words(uint32_t (&to)[N], const void *w) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(w);
    const uint32_t *from = reinterpret_cast<const uint32_t *>(at & ~uintptr_t{3});
    const uint32_t shift = (at & 2) * 8;
    uint32_t u[N + 1];
#pragma unroll
    for (int k = 0; k < N; ++k) u[k] = __ldg(from + k);
    u[N] = shift ? __ldg(from + N) : 0;
#pragma unroll
    for (int k = 0; k < N; ++k) to[k] = __funnelshift_r(u[k], u[k + 1], shift);
}

template <class W, bool VEC>
__device__ __forceinline__ LoraRaw<W> lora_load4(const W *w, int n, int how) {
    LoraRaw<W> raw{};
    if constexpr (VEC) {
        if (n > 0) raw = lora_as<LoraRaw<W>>(w);
    } else if constexpr (sizeof(W) == 4) {
        if (n >= 4 && how == kLoraWhole) {
            raw = lora_as<uint4>(w);
        } else {
            if (n > 0) raw.x = lora_as<uint32_t>(w);
            if (n > 1) raw.y = lora_as<uint32_t>(w + 1);
            if (n > 2) raw.z = lora_as<uint32_t>(w + 2);
            if (n > 3) raw.w = lora_as<uint32_t>(w + 3);
        }
    } else if (n >= 4 && how >= kLoraQuads) {
        raw = lora_as<uint2>(w);
    } else if (n >= 5 && how == kLoraWords) {
        uint32_t u[2];
        lora_words(u, w);
        raw = make_uint2(u[0], u[1]);
    } else {
        if (n > 0) raw.x = lora_as<uint16_t>(w);
        if (n > 1) raw.x |= static_cast<uint32_t>(lora_as<uint16_t>(w + 1)) << 16;
        if (n > 2) raw.y = lora_as<uint16_t>(w + 2);
        if (n > 3) raw.y |= static_cast<uint32_t>(lora_as<uint16_t>(w + 3)) << 16;
    }
    return raw;
}

template <class W, bool VEC>
__device__ __forceinline__ LoraEight<W> lora_load8(const W *w, int n, int how) {
    LoraEight<W> v{};
    if constexpr (sizeof(W) == 2) {
        if (VEC ? n > 0 : n >= 8 && how == kLoraWhole) {
            const uint4 u = lora_as<uint4>(w);
            v.q[0] = make_uint2(u.x, u.y), v.q[1] = make_uint2(u.z, u.w);
            return v;
        }
        if constexpr (VEC) return v;
        if (n >= 9 && how == kLoraWords) {
            uint32_t u[4];
            lora_words(u, w);
            v.q[0] = make_uint2(u[0], u[1]), v.q[1] = make_uint2(u[2], u[3]);
            return v;
        }
    }
    v.q[0] = lora_load4<W, VEC>(w, n, how);
    v.q[1] = lora_load4<W, VEC>(w + 4, n - 4, how);
    return v;
}

// Keeps the first n of the four values (n <= 0: none).
template <class W>
__device__ __forceinline__ LoraRaw<W> lora_mask(int n) {
    if constexpr (sizeof(W) == 4) {
        return make_uint4(n > 0 ? ~0u : 0u, n > 1 ? ~0u : 0u, n > 2 ? ~0u : 0u, n > 3 ? ~0u : 0u);
    } else {
        return make_uint2(n > 1 ? ~0u : n > 0 ? 0xffffu : 0u, n > 3 ? ~0u : n > 2 ? 0xffffu : 0u);
    }
}

__device__ __forceinline__ void lora_keep(uint2 &raw, const uint2 &mask) { raw.x &= mask.x, raw.y &= mask.y; }
__device__ __forceinline__ void lora_keep(uint4 &raw, const uint4 &mask) {
    raw.x &= mask.x, raw.y &= mask.y, raw.z &= mask.z, raw.w &= mask.w;
}

template <class W>
__device__ __forceinline__ float4 lora_f32(const LoraRaw<W> &raw) {
    if constexpr (sizeof(W) == 4) {
        return make_float4(__uint_as_float(raw.x), __uint_as_float(raw.y), __uint_as_float(raw.z),
                           __uint_as_float(raw.w));
    } else if constexpr (std::is_same_v<W, __half>) {
        const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    } else {
        return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u),
                           __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u));
    }
}

__device__ __forceinline__ uint32_t lora_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}

// The same, and the largest TF32 number of the sign where that is beyond it.
__device__ __forceinline__ uint32_t lora_tf32_within(float x) {
    uint32_t r;
    asm("cvt.rna.satfinite.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}

// x = hi + lo, both TF32.  Of an infinite x (and of one that hi rounds up to infinity) lo is not a number, but with
// WIDE: infinity is then the largest number and infinity, whose products with a weight have one sign.
template <bool WIDE>
__device__ __forceinline__ void lora_split(float x, uint32_t &hi, uint32_t &lo) {
    hi = WIDE ? lora_tf32_within(x) : lora_tf32(x);
    lo = lora_tf32(x - __uint_as_float(hi));
}

template <bool WIDE>
__device__ __forceinline__ void lora_split(const float4 &x, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) lora_split<WIDE>(v[e], hi[e], lo[e]);
}

__device__ __forceinline__ void lora_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// c += W x over 16 columns, four a lane: `top` and `low` are the lane's weights of rows g and
// g + 8 of the tile (g = lane / 4), hi and lo its token's x.  SPLIT: the weights are not TF32 numbers.
template <bool SPLIT>
__device__ __forceinline__ void lora_unit(float (&c)[4], const float4 &top, const float4 &low, const uint32_t (&hi)[4],
                                          const uint32_t (&lo)[4]) {
    uint32_t th[4], lh[4];
    if constexpr (SPLIT) {
        uint32_t tl[4], ll[4];
        lora_split<false>(top, th, tl);
        lora_split<false>(low, lh, ll);
#pragma unroll
        for (int s = 0; s < 4; s += 2) lora_mma(c, tl[s], ll[s], tl[s + 1], ll[s + 1], hi[s], hi[s + 1]);
    } else {
        th[0] = __float_as_uint(top.x), th[1] = __float_as_uint(top.y);
        th[2] = __float_as_uint(top.z), th[3] = __float_as_uint(top.w);
        lh[0] = __float_as_uint(low.x), lh[1] = __float_as_uint(low.y);
        lh[2] = __float_as_uint(low.z), lh[3] = __float_as_uint(low.w);
    }
#pragma unroll
    for (int s = 0; s < 4; s += 2) lora_mma(c, th[s], lh[s], th[s + 1], lh[s + 1], lo[s], lo[s + 1]);
#pragma unroll
    for (int s = 0; s < 4; s += 2) lora_mma(c, th[s], lh[s], th[s + 1], lh[s + 1], hi[s], hi[s + 1]);
}

// The tiles of a call as a CTA knows them: the plan's, or (few tokens) a table that
// each CTA makes for itself: a token leads a tile if it is the first, or TILE-th,
// 2 TILE-th ..., of its adapter's tokens; the tile is it and the next ones.
template <int TILE>
struct LoraTiles {
    int count;
    int tokens[TILE], adapter, n, rank;  // of the tile last opened
    alignas(16) int ids[kLoraScan];
    int leads[kLoraScan / 32];
    int tile_adapter[kLoraScan], tile_n[kLoraScan], tile_rank[kLoraScan], tile_tokens[kLoraScan][TILE];
};

template <int TILE>
__device__ __forceinline__ void lora_tiles(LoraTiles<TILE> &s, const LoraArgs &p, bool report) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.tiles) {  // read past L1: written by a kernel that may have run beside this one
        if (tid == 0) s.count = __ldcg(p.ntiles);
        __syncthreads();
        return;
    }
    int a = -1, rank = 0;
    if (tid < kLoraScan) {
        a = tid < p.tokens ? p.ids[tid] : -1;
        if (a >= p.adapters) {
            if (report) report_device_error(p.err, kDevErrBadIndex);
            a = -1;
        }
        s.ids[tid] = a;
        rank = __ldg(p.ranks + max(a, 0));  // on its way while the tiles are found
    }
    __syncthreads();
    uint64_t same = 0;  // the tokens of this one's adapter
    if (tid < kLoraScan) {
        for (int j0 = 0; j0 < p.tokens; j0 += 8) {
            const int4 u = *reinterpret_cast<const int4 *>(s.ids + j0);
            const int4 v = *reinterpret_cast<const int4 *>(s.ids + j0 + 4);
            const uint32_t m = (u.x == a) | (u.y == a) << 1 | (u.z == a) << 2 | (u.w == a) << 3 | (v.x == a) << 4 |
                               (v.y == a) << 5 | (v.z == a) << 6 | (v.w == a) << 7;
            same |= static_cast<uint64_t>(m) << j0;
        }
        const bool leads = a >= 0 && __popcll(same & ((1ull << tid) - 1)) % TILE == 0;
        const uint32_t m = __ballot_sync(0xffffffffu, leads);
        if (lane == 0) s.leads[warp] = m;
        if (!leads) same = 0;
    }
    __syncthreads();
    if (tid < kLoraScan && same) {
        int k = __popc(s.leads[warp] & ((1u << lane) - 1));
        for (int w = 0; w < warp; ++w) k += __popc(s.leads[w]);
        int n = 0;
        for (uint64_t left = same >> tid << tid; left && n < TILE; left &= left - 1)
            s.tile_tokens[k][n++] = __ffsll(left) - 1;
        s.tile_adapter[k] = a;
        s.tile_n[k] = n;
        s.tile_rank[k] = min(max(rank, 0), p.max_rank);
    }
    if (tid == 0) {
        int all = 0;
        for (int w = 0; w < kLoraScan / 32; ++w) all += __popc(s.leads[w]);
        s.count = all;
    }
    __syncthreads();
}

// Opens tile k: its adapter and rank, its tokens (of those it lacks, its first).
template <int TILE>
__device__ __forceinline__ void lora_open(LoraTiles<TILE> &s, const LoraArgs &p, int k) {
    const int tid = threadIdx.x;
    int v = 0;
    if (p.tiles && tid < 32) {  // on its way while the CTA meets
        static_assert(sizeof(LoraTile) == 4 * (4 + kLoraTile) && kLoraTile <= 28);
        if (tid < 4 + kLoraTile) v = __ldcg(reinterpret_cast<const int *>(p.tiles + k) + tid);
    }
    __syncthreads();  // the tile before is done with
    if (p.tiles) {
        if (tid < 32) {
            const int n = __shfl_sync(0xffffffffu, v, 1), first = __shfl_sync(0xffffffffu, v, 4);
            if (tid >= 4 && tid < 4 + TILE) s.tokens[tid - 4] = tid - 4 < n ? v : first;
            if (tid == 0) s.adapter = v;
            if (tid == 1) s.n = v;
            if (tid == 2) s.rank = v;
        }
    } else {
        if (tid < TILE) s.tokens[tid] = s.tile_tokens[k][tid < s.tile_n[k] ? tid : 0];
        if (tid == 0) s.adapter = s.tile_adapter[k], s.n = s.tile_n[k], s.rank = s.tile_rank[k];
    }
    __syncthreads();
}

// Tiles of up to kLoraTile tokens of one adapter: one CTA counts the adapters' tokens
// (in shared memory when the adapters fit), gives each adapter its tiles, and each
// token its place in them.  The order within an adapter is that of the atomics,
// which no result depends on.
constexpr int kLoraPlanThreads = 1024, kLoraPlanOwn = 4, kLoraPlanCounts = 4096;
__global__ void __launch_bounds__(kLoraPlanThreads) lora_plan_kernel(LoraArgs p) {
    __shared__ int warp_tiles[32], near_counts[kLoraPlanCounts];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    allow_dependent_launch();
    int *counts = p.adapters <= kLoraPlanCounts ? near_counts : p.counts;
    for (int a = tid; a < p.adapters; a += kLoraPlanThreads) counts[a] = 0;
    int own[kLoraPlanOwn], place[kLoraPlanOwn];  // the thread's first tokens
#pragma unroll
    for (int k = 0; k < kLoraPlanOwn; ++k) {
        const int t = tid + k * kLoraPlanThreads;
        own[k] = t < p.tokens ? p.ids[t] : -1;
    }
    int rank = tid < p.adapters ? lora_rank(p, tid) : 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kLoraPlanOwn; ++k) {
        if (own[k] >= p.adapters) {
            report_device_error(p.err, kDevErrBadIndex);
            own[k] = -1;
        }
        place[k] = own[k] >= 0 ? atomicAdd(counts + own[k], 1) : 0;
    }
    for (int t = tid + kLoraPlanOwn * kLoraPlanThreads; t < p.tokens; t += kLoraPlanThreads) {
        const int a = p.ids[t];
        if (a >= p.adapters) report_device_error(p.err, kDevErrBadIndex);
        p.places[t] = a >= 0 && a < p.adapters ? atomicAdd(counts + a, 1) : 0;
    }
    __syncthreads();
    int base = 0;  // the tiles of the adapters before these
    for (int a0 = 0; a0 < p.adapters; a0 += kLoraPlanThreads) {
        const int a = a0 + tid, n = a < p.adapters ? counts[a] : 0, nt = (n + kLoraTile - 1) / kLoraTile;
        if (a0) rank = a < p.adapters ? lora_rank(p, a) : 0;
        int sum = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 31) warp_tiles[warp] = sum;
        __syncthreads();
        int first = base + sum - nt, all = warp_tiles[lane];
        const int before = __reduce_add_sync(0xffffffffu, lane < warp ? all : 0);
        first += before;
        base += __reduce_add_sync(0xffffffffu, all);
        if (a < p.adapters) counts[a] = first;
        for (int i = 0; i < nt; ++i)
            *reinterpret_cast<int4 *>(p.tiles + first + i) = make_int4(a, min(kLoraTile, n - i * kLoraTile), rank, 0);
        __syncthreads();
    }
    const auto put = [&](int a, int at, int t) { p.tiles[counts[a] + at / kLoraTile].tokens[at % kLoraTile] = t; };
#pragma unroll
    for (int k = 0; k < kLoraPlanOwn; ++k)
        if (own[k] >= 0) put(own[k], place[k], tid + k * kLoraPlanThreads);
    for (int t = tid + kLoraPlanOwn * kLoraPlanThreads; t < p.tokens; t += kLoraPlanThreads) {
        const int a = p.ids[t];
        if (a >= 0 && a < p.adapters) put(a, p.places[t], t);
    }
    if (tid == 0) *p.ntiles = base;
}

__device__ __forceinline__ float lora_value(float w) { return w; }
__device__ __forceinline__ float lora_value(__half w) { return __half2float(w); }
__device__ __forceinline__ float lora_value(__nv_bfloat16 w) { return __bfloat162float(w); }

// w . x over n columns in plain f32, sixteen sums side by side; ends with the first that is not a number.
template <class W>
__device__ __noinline__ float lora_plain(const W *w, const float *x, int n) {
    float v[16] = {}, sum = 0.0f;
    for (int c = 0; c < n && sum == sum; c += 16) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (c + k < n) v[k] = fmaf(lora_value(w[c + k]), x[c + k], v[k]);
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += v[k];
    }
    return sum;
}

// A . x for a tile of 8 NT tokens, 16 MT MW ranks and a range of columns, by one
// CTA.  MW warps share a block of 32 columns, 16 MT ranks each, and take every
// 8 / MW-th block, the next one on its way meanwhile; the warps' sums are joined
// in order.  Lanes without a token or a rank of their own read the first one's:
// what they make is a column or a row of the tile that nobody keeps.
template <class W, int MT, int MW, int NT, bool VEC>
struct LoraShrink {
    static constexpr int kKWarps = kLoraWarps / MW, kRanks = 16 * MT * MW, kStride = 8 * NT + 1;
    static constexpr int kBatch = 32 * kKWarps;  // columns from a warp's block to its next
    struct Shared {
        float parts[kKWarps][kRanks * kStride];
        float4 sums[MT * NT][kLoraThreads];
    };
    struct Batch {
        LoraEight<W> w[2 * MT];
        LoraEight<float> x[NT];
    };

    // Ranks r0 .. of adapter a (of its `rank`) and the columns of units first .. u1 of 16; the warps' sums stand in
    // s.parts when it returns, for sum().
    static __device__ __forceinline__ void run(const LoraArgs &p, Shared &s, const int (&tokens)[8 * NT], int a,
                                               int rank, int r0, int first, int u1) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = 4 * (lane & 3), t8 = 2 * t4;
        const int kw = warp / MW, rw = r0 + 16 * MT * (warp % MW) + g;  // the lane's first rank
        const int u0 = first + 2 * kw;
        const W *w[2 * MT];
        const float *x[NT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int r = rw + 8 * i < rank ? rw + 8 * i : 0;
            w[i] = static_cast<const W *>(p.a) + (static_cast<int64_t>(a) * p.max_rank + r) * p.cols + 16 * u0 + t8;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j] = p.x + tokens[8 * j + g] * p.x_stride + 16 * u0 + t8;
        float acc[MT][NT][4] = {};
        const auto load = [&](Batch &t, int left) {  // left: columns from the lane's first to the end of the split
#pragma unroll
            for (int j = 0; j < NT; ++j) t.x[j] = lora_load8<float, VEC>(x[j], left, p.how_x), x[j] += kBatch;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) t.w[i] = lora_load8<W, VEC>(w[i], left, p.how_a), w[i] += kBatch;
        };
        const auto multiply = [&](const Batch &t) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    uint32_t hi[4], lo[4];
                    lora_split<false>(lora_f32<float>(t.x[j].q[k]), hi, lo);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        lora_unit<sizeof(W) == 4>(acc[i][j], lora_f32<W>(t.w[2 * i].q[k]),
                                                  lora_f32<W>(t.w[2 * i + 1].q[k]), hi, lo);
                }
            }
        };
        // The tensor cores cut what an addition leaves over: sums through thousands of columns drift by that (2.7e-6 of
        // the result at 6144).  Theirs end after two blocks and go on as rounded f32 sums, in the lane's own places.
        bool begun = false;
        const auto settle = [&]() {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float4 &sum = s.sums[i * NT + j][threadIdx.x];
                    float4 v = begun ? sum : make_float4(0.f, 0.f, 0.f, 0.f);
                    v.x += acc[i][j][0], v.y += acc[i][j][1], v.z += acc[i][j][2], v.w += acc[i][j][3];
                    sum = v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.0f;
                }
            }
            begun = true;
        };
        Batch even, odd;
        int left = min(p.cols, 16 * u1) - (16 * u0 + t8);
        // left + t8 is what the warp's first lane has left: the same in all lanes
        load(even, left);
        while (left + t8 > 0) {
            if (left + t8 > kBatch) load(odd, left - kBatch);
            multiply(even);
            if (left + t8 <= kBatch) break;
            left -= 2 * kBatch;
            if (left + t8 > 0) load(even, left);
            multiply(odd);
            if (left + t8 > 0) settle();
        }
        if (begun) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float4 v = s.sums[i * NT + j][threadIdx.x];
                    acc[i][j][0] += v.x, acc[i][j][1] += v.y, acc[i][j][2] += v.z, acc[i][j][3] += v.w;
                }
            }
        }
        // acc[i][j]: ranks rw + 16 i (+ 8), tokens 8 j + t4 / 2 (+ 1)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float *at = s.parts[kw] + (rw - r0 + 16 * i) * kStride + 8 * j + t4 / 2;
                at[0] = acc[i][j][0], at[1] = acc[i][j][1];
                at[8 * kStride] = acc[i][j][2], at[8 * kStride + 1] = acc[i][j][3];
            }
        }
        __syncthreads();
    }

    // The sum of rank r0 + r and token `token` at place tok, of the columns of units first .. u1.  What is not finite
    // is made again in plain f32, since x in parts makes infinity less infinity of an infinity: 4096 tokens 138 us as
    // without it, 0.5 ms if one has an infinite x; parts that infinity has (WIDE) for every x 138.7 us, 1000 tokens
    // 32.8 instead of 32.2.
    static __device__ __forceinline__ float sum(const LoraArgs &p, const Shared &s, int a, int r0, int r, int tok,
                                                int token, int first, int u1) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kKWarps; ++k) v += s.parts[k][r * kStride + tok];
        if (fabsf(v) < INFINITY) return v;
        const W *w = static_cast<const W *>(p.a) + (static_cast<int64_t>(a) * p.max_rank + r0 + r) * p.cols;
        return lora_plain(w + 16 * first, p.x + token * p.x_stride + 16 * first, min(p.cols, 16 * u1) - 16 * first);
    }
};

// h[split][token][r] = A[r][the split's columns] . x[token][the split's columns], item
// after item (a tile, a split, a run of ranks).
template <class W, int MT, int MW, int NT, bool VEC>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_shrink_kernel(LoraArgs p) {
    using Shrink = LoraShrink<W, MT, MW, NT, VEC>;
    constexpr int kRanks = Shrink::kRanks;
    __shared__ LoraTiles<8 * NT> tiles;
    __shared__ typename Shrink::Shared shared;
    grid_dependency_wait();  // the plan comes from the kernel before
    allow_dependent_launch();
    lora_tiles(tiles, p, blockIdx.x == 0);
    const int chunks = (p.max_rank + kRanks - 1) / kRanks, per_tile = p.splits * chunks;
    for (int64_t item = blockIdx.x; item < static_cast<int64_t>(tiles.count) * per_tile; item += gridDim.x) {
        lora_open(tiles, p, static_cast<int>(item / per_tile));
        const int part = static_cast<int>(item % per_tile), split = part / chunks, r0 = part % chunks * kRanks;
        const int rank = tiles.rank;
        if (r0 >= rank) continue;
        const int first = split * p.units, u1 = min(first + p.units, (p.cols + 15) / 16);
        Shrink::run(p, shared, tiles.tokens, tiles.adapter, rank, r0, first, u1);
        for (int i = threadIdx.x; i < tiles.n * kRanks; i += kLoraThreads) {
            const int r = i % kRanks, tok = i / kRanks, token = tiles.tokens[tok];
            if (r0 + r < rank)
                p.h[(static_cast<int64_t>(split) * p.tokens + token) * lora_h_pitch(p.max_rank) + r0 + r] =
                    Shrink::sum(p, shared, tiles.adapter, r0, r, tok, token, first, u1);
        }
    }
}

// The floats from one token's h to the next's in shared memory: 16 or 4 mod 32 banks, so that the quarters of a
// warp's 16-byte reads do not meet.
template <int KU>
__host__ __device__ constexpr int lora_pitch(int rank) {
    const int chunks = (rank + 16 * KU - 1) / (16 * KU);
    return KU == 1 ? 16 * (chunks | 1) : 32 * chunks + 4;
}

// Element r of token tok's h, as hi + lo.
template <int NT>
__device__ __forceinline__ void lora_put(float *hs, int pitch, int tok, int r, float h) {
    uint32_t hi, lo;
    lora_split<true>(h, hi, lo);
    hs[tok * pitch + r] = __uint_as_float(hi);
    hs[(8 * NT + tok) * pitch + r] = __uint_as_float(lo);
}

// Elements r .. r + 3 of token tok's h.
template <int NT>
__device__ __forceinline__ void lora_put(float *hs, int pitch, int tok, int r, const float4 &h) {
    uint32_t hi[4], lo[4];
    lora_split<true>(h, hi, lo);
    *reinterpret_cast<uint4 *>(hs + tok * pitch + r) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(hs + (8 * NT + tok) * pitch + r) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// y[token][row] += s * B[row] . h[token] for a tile of 8 NT tokens, by one warp:
// `steps` times 32 RG rows, from row_first, row_next apart.  Row 4 g + i of 32
// stands at place g of half i of two m16 tiles, so that a lane ends up with
// four neighbouring rows of two tokens: one float4 of y each.  Ranks come 16 KU at a
// time.  With VEC lanes whose rows are behind the last read the last ones and write nothing.
// prepare() puts h into hs (lora_put, zero from the rank to the end of its chunk) and
// synchronises; the first weights are on their way meanwhile.
template <class W, int NT, int RG, int KU, bool VEC, bool LONG>
struct LoraExpand {
    static constexpr int kSpan = kLoraRows * RG, kChunk = 16 * KU;
    // Chunks after which a chain of the tensor cores ends and goes on as a rounded f32 sum in shared memory, as in
    // LoraShrink: in one chain the error of rank 256 against 64 bits is 1.4e-6 instead of 5.8e-7 (F32 weights 2.1e-6
    // instead of 7.9e-7), 4096 tokens of rank 128 take 309 us instead of 324, 4 of rank 256 12.6 instead of 13.0.
    // LONG is for stacks of more ranks than that: 1000 tokens of rank 64 take 32.3 us without it, 32.8 with it.
    static constexpr int kSettle = kLoraChain / kChunk;
    static constexpr int kSums = LONG ? 2 * RG * NT * kLoraThreads : 0;  // float4s of them

    template <class F>
    static __device__ __forceinline__ void run(const LoraArgs &p, const float *hs, float4 *sums,
                                               const int (&tokens)[8 * NT], int n, int a, int rank, int row_first,
                                               int row_next, int steps, const F &prepare) {
        const int t4 = 4 * (threadIdx.x & 3);
        const int chunks = (rank + kChunk - 1) / kChunk;
        const int lane_r = KU * t4;  // a lane has 4 KU neighbouring ranks of a chunk
        const int lane = threadIdx.x & 31, g = lane >> 2, pitch = lora_pitch<KU>(rank);
        const float scale = p.scales[a];
        const float *ls = hs + 8 * NT * pitch;
        const W *b = static_cast<const W *>(p.b) + static_cast<int64_t>(a) * p.rows * p.max_rank + lane_r;
        const W *b_end = static_cast<const W *>(p.b) + static_cast<int64_t>(p.adapters) * p.rows * p.max_rank;
        float *y[NT][2];  // the lane's tokens' rows
        bool mine[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int tok = 8 * j + t4 / 2 + e;
                mine[j][e] = tok < n;
                y[j][e] = p.y + tokens[tok] * p.y_stride;
            }
        }
        struct Rows {
            float v[RG][NT][2][4];
        };
        struct Weights {
            LoraRaw<W> w[KU][RG][4];
        };
        const auto load_y = [&](Rows &to, int row) {
#pragma unroll
            for (int q = 0; q < RG; ++q) {
                const int r = row + kLoraRows * q;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (VEC) {
                            *reinterpret_cast<float4 *>(to.v[q][j][e]) =
                                *reinterpret_cast<const float4 *>(y[j][e] + min(r, p.rows - 4));
                        } else if (p.how_y == kLoraWhole && r + 4 <= p.rows) {
                            *reinterpret_cast<float4 *>(to.v[q][j][e]) = *reinterpret_cast<const float4 *>(y[j][e] + r);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) to.v[q][j][e][i] = y[j][e][min(r + i, p.rows - 1)];
                        }
                    }
                }
            }
        };
        const auto load_w = [&](Weights &to, int row, int c) {
#pragma unroll
            for (int q = 0; q < RG; ++q) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = min(row + kLoraRows * q + i, VEC ? p.rows - 4 + i : p.rows - 1);
                    const W *from = b + static_cast<int64_t>(r) * p.max_rank + kChunk * c;
                    // Behind the rank others' values may be read, up to the stack's end: the last chunk's mask drops
                    // them.
                    int n = rank - kChunk * c - lane_r;
                    if (!VEC && n > 0) n = static_cast<int>(min(b_end - from, static_cast<ptrdiff_t>(16)));
                    if constexpr (KU == 2) {
                        const LoraEight<W> v = lora_load8<W, VEC>(from, n, p.how_b);
                        to.w[0][q][i] = v.q[0], to.w[1][q][i] = v.q[1];
                    } else {
                        to.w[0][q][i] = lora_load4<W, VEC>(from, n, p.how_b);
                    }
                }
            }
        };
        // A turn: a chunk of ranks of a step's rows.  The weights of two turns are on their way while a third's are
        // multiplied; the three places take turns by name, since a copy from one to the next would wait for it.
        int row = row_first + 4 * g, chunk = 0;
        int fetch_row = row, fetch_chunk = 0, fetches = steps * chunks;
        const auto fetch = [&](Weights &to) {
            if (--fetches < 0) return;
            load_w(to, fetch_row, fetch_chunk);
            // With many tokens the rows of y into L2, a line a token: 4096 tokens 142.0 -> 137.9 us, 1000 33.3 -> 32.2
            // (few tokens' short runs lose by it: 1 token 5.05 -> 5.38, 48 12.3 -> 12.6).
            if (NT > 1 && fetch_chunk == 0 && g < RG) {
                const int r = fetch_row - 4 * g + kLoraRows * g;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (mine[j][e] && r < p.rows) asm volatile("prefetch.global.L2 [%0];" ::"l"(y[j][e] + r));
                }
            }
            if (++fetch_chunk == chunks) fetch_chunk = 0, fetch_row += row_next;
        };
        Weights one, two, three;
        fetch(one);
        fetch(two);
        prepare();
        LoraRaw<W> last_mask[KU];
#pragma unroll
        for (int k = 0; k < KU; ++k) last_mask[k] = lora_mask<W>(rank - kChunk * (chunks - 1) - lane_r - 4 * k);
        Rows old;
        float acc[RG][2][NT][4];
        const auto turn = [&](Weights &wt, Weights &later) {
            fetch(later);
            if (chunk == 0) {
                load_y(old, row);
#pragma unroll
                for (int i = 0; i < RG * 2 * NT * 4; ++i) (&acc[0][0][0][0])[i] = 0.0f;
            }
            if (chunk == chunks - 1) {
#pragma unroll
                for (int k = 0; k < KU; ++k) {
#pragma unroll
                    for (int i = 0; i < 4 * RG; ++i) lora_keep(wt.w[k][i / 4][i % 4], last_mask[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < KU; ++k) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int from = (8 * j + g) * pitch + kChunk * chunk + lane_r + 4 * k;
                    const uint4 h4 = *reinterpret_cast<const uint4 *>(hs + from);
                    const uint4 l4 = *reinterpret_cast<const uint4 *>(ls + from);
                    const uint32_t hi[4] = {h4.x, h4.y, h4.z, h4.w}, lo[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                    for (int q = 0; q < RG; ++q) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            lora_unit<sizeof(W) == 4>(acc[q][i][j], lora_f32<W>(wt.w[k][q][2 * i]),
                                                      lora_f32<W>(wt.w[k][q][2 * i + 1]), hi, lo);
                    }
                }
            }
            const bool last = ++chunk == chunks;
            if (LONG && (last ? chunks > kSettle : chunk % kSettle == 0)) {
#pragma unroll
                for (int i = 0; i < 2 * RG * NT; ++i) {
                    float4 &sum = sums[i * kLoraThreads + threadIdx.x];
                    float *c = &acc[0][0][0][0] + 4 * i;
                    const float4 v = chunk > kSettle ? sum : float4{};
                    c[0] += v.x, c[1] += v.y, c[2] += v.z, c[3] += v.w;
                    if (last) continue;
                    sum = make_float4(c[0], c[1], c[2], c[3]);
                    c[0] = c[1] = c[2] = c[3] = 0.0f;
                }
            }
            if (!last) return;
            chunk = 0;
#pragma unroll
            for (int q = 0; q < RG; ++q) {
                const int r = row + kLoraRows * q;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float *o = old.v[q][j][e];
                        const float v[4] = {fmaf(scale, acc[q][0][j][e], o[0]), fmaf(scale, acc[q][0][j][2 + e], o[1]),
                                            fmaf(scale, acc[q][1][j][e], o[2]), fmaf(scale, acc[q][1][j][2 + e], o[3])};
                        if (VEC || (p.how_y == kLoraWhole && r + 4 <= p.rows)) {
                            if (mine[j][e] && r < p.rows)
                                *reinterpret_cast<float4 *>(y[j][e] + r) = make_float4(v[0], v[1], v[2], v[3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (mine[j][e] && r + i < p.rows) y[j][e][r + i] = v[i];
                        }
                    }
                }
            }
            row += row_next;
        };
        for (int left = steps * chunks; left > 0; left -= 3) {
            turn(one, three);
            if (left > 1) turn(two, one);
            if (left > 2) turn(three, two);
        }
    }
};

// The tiles' steps in one row, a run of them a CTA; h from the workspace, its parts joined in order.
template <class W, int NT, int RG, int KU, bool VEC, bool LONG>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_expand_kernel(LoraArgs p) {
    using Expand = LoraExpand<W, NT, RG, KU, VEC, LONG>;
    extern __shared__ __align__(16) float hs[];  // [2][8 NT][pitch]: hi, lo; LONG: sums
    __shared__ LoraTiles<8 * NT> tiles;
    constexpr int kNext = kLoraWarps * Expand::kSpan;
    const int tid = threadIdx.x, warp = tid >> 5;
    lora_tiles(tiles, p, false);
    bool waited = false;
    const int per_tile = (p.rows + kNext - 1) / kNext;
    const int64_t all = static_cast<int64_t>(tiles.count) * per_tile, end = all * (blockIdx.x + 1) / gridDim.x;
    int64_t at = all * blockIdx.x / gridDim.x;
    while (at < end) {
        lora_open(tiles, p, static_cast<int>(at / per_tile));
        const int first = static_cast<int>(at % per_tile);
        const int steps = static_cast<int>(min(end - at, static_cast<int64_t>(per_tile - first)));
        at += steps;
        const int rank = tiles.rank;
        if (rank == 0) continue;
        const int row_first = (first * kLoraWarps + warp) * Expand::kSpan;
        float4 *sums = reinterpret_cast<float4 *>(hs + 16 * NT * lora_pitch<KU>(p.max_rank));
        Expand::run(p, hs, sums, tiles.tokens, tiles.n, tiles.adapter, rank, row_first, kNext, steps, [&]() {
            if (!waited) grid_dependency_wait();  // h comes from the kernel before
            waited = true;
            // Each quad of ranks is summed by 2^team lanes, four parts in flight in each: the joining is bound by
            // its instructions (of 32 parts, rank 64: a quad at once 33.4 us, single values, eight parts in flight,
            // 37.8, sixteen 40.2, of a call of 1000 tokens).
            const int quads = (rank + Expand::kChunk - 1) / Expand::kChunk * (Expand::kChunk / 4);
            const int items = 8 * NT * quads;
            const int shift = p.team, team = 1 << shift, member = tid & (team - 1);
            for (int i0 = 0; i0 < items; i0 += kLoraThreads >> shift) {
                const int i = i0 + (tid >> shift), tok = i / quads, r = 4 * (i - tok * quads);
                float4 sum{};
                if (tok < tiles.n && r < rank) {
                    const int pitch = lora_h_pitch(p.max_rank);
                    const float *h = p.h + static_cast<int64_t>(tiles.tokens[tok]) * pitch + r;
                    const int64_t on = static_cast<int64_t>(p.tokens) * pitch << shift;
                    h += member * (on >> shift);
                    for (int s = member; s < p.splits; s += 4 * team, h += 4 * on) {
                        float4 part[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            part[k] = s + k * team < p.splits ? *reinterpret_cast<const float4 *>(h + k * on)
                                                              : float4{};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            sum.x += part[k].x, sum.y += part[k].y, sum.z += part[k].z, sum.w += part[k].w;
                    }
                }
                for (int o = 1; o < team; o *= 2) {
                    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o), sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
                    sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o), sum.w += __shfl_xor_sync(0xffffffffu, sum.w, o);
                }
                if (member == 0 && i < items) {
                    sum.y = r + 1 < rank ? sum.y : 0.0f, sum.z = r + 2 < rank ? sum.z : 0.0f;
                    sum.w = r + 3 < rank ? sum.w : 0.0f;
                    lora_put<NT>(hs, lora_pitch<KU>(rank), tok, r, sum);
                }
            }
            __syncthreads();
        });
    }
    // A CTA with nothing to do must not end before the kernel before: what comes next waits for this one only.
    if (!waited) grid_dependency_wait();
}

// Few tiles of small adapters in one launch: a cluster per tile.  Each CTA takes a share of the columns, the
// cluster's CTAs read one another's sums, and each takes a share of the rows.  For adapters of up to kLoraSmall bytes
// whose clusters have an SM a CTA at once; in CUDA graphs, this against the two kernels: 1 token, 576 x 6144 of rank 8
// 5.5 against 6.1 us, 512 x 512 of rank 64 5.8 against 7.3; 16 tokens of 16 adapters, 2048 x 6144 of rank 16 7.4
// against 8.3.  Beyond: one of 4096 x 4096 of rank 64 (1 MB) 8.5 against 7.3, 36 adapters of 256 x 256 8.9 against 5.6.
constexpr int kLoraCluster = 8;
constexpr int64_t kLoraSmall = 512 << 10;

__device__ __forceinline__ float cluster_load(const float *at, uint32_t rank) {  // this CTA's `at` in CTA `rank`
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(at)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}

template <class W, int MT, int MW, int RG, int KU, bool VEC, bool LONG>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_cluster_kernel(LoraArgs p) {
    using Shrink = LoraShrink<W, MT, MW, 1, VEC>;
    using Expand = LoraExpand<W, 1, RG, KU, VEC, LONG>;
    extern __shared__ __align__(16) float hs[];  // [2][8][pitch]: hi, lo; the CTA's h [8][max_rank]; LONG: sums
    __shared__ LoraTiles<8> tiles;
    __shared__ typename Shrink::Shared shared;
    const int tid = threadIdx.x, part = blockIdx.x % kLoraCluster, tile = blockIdx.x / kLoraCluster;
    lora_tiles(tiles, p, blockIdx.x == 0);
    if (tile >= tiles.count) return;  // the whole cluster
    lora_open(tiles, p, tile);
    const int rank = tiles.rank, n = tiles.n, pitch = lora_pitch<KU>(rank);
    if (rank == 0) return;  // the whole cluster
    float *mine = hs + 16 * lora_pitch<KU>(p.max_rank);
    const int units = (p.cols + 15) / 16, share = 2 * ((units + 2 * kLoraCluster - 1) / (2 * kLoraCluster));
    const int first = min(part * share, units), u1 = min(first + share, units);
    for (int r0 = 0; r0 < rank; r0 += Shrink::kRanks) {
        if (r0) __syncthreads();  // the ranks before are read
        Shrink::run(p, shared, tiles.tokens, tiles.adapter, rank, r0, first, u1);
        for (int i = tid; i < n * Shrink::kRanks; i += kLoraThreads) {
            const int tok = i / Shrink::kRanks, r = i % Shrink::kRanks;
            if (r0 + r < rank)
                mine[tok * p.max_rank + r0 + r] =
                    Shrink::sum(p, shared, tiles.adapter, r0, r, tok, tiles.tokens[tok], first, u1);
        }
    }
    cluster_arrive();
    const int row_first = (part * kLoraWarps + (tid >> 5)) * Expand::kSpan;
    const int row_next = kLoraCluster * kLoraWarps * Expand::kSpan;
    const int steps = row_first < p.rows ? (p.rows - row_first + row_next - 1) / row_next : 0;
    float4 *sums = reinterpret_cast<float4 *>(mine + 8 * p.max_rank);
    Expand::run(p, hs, sums, tiles.tokens, n, tiles.adapter, rank, row_first, row_next, steps, [&]() {
        cluster_wait();
        const int width = (rank + Expand::kChunk - 1) / Expand::kChunk * Expand::kChunk;
        for (int i = tid; i < 8 * width; i += kLoraThreads) {
            const int tok = i / width, r = i - tok * width;
            float sum = 0.0f;
            if (tok < n && r < rank) {
                float v[kLoraCluster];
#pragma unroll
                for (int c = 0; c < kLoraCluster; ++c) v[c] = cluster_load(mine + tok * p.max_rank + r, c);
#pragma unroll
                for (int c = 0; c < kLoraCluster; ++c) sum += v[c];
            }
            lora_put<1>(hs, pitch, tok, r, sum);
        }
        cluster_arrive();
        __syncthreads();
    });
    cluster_wait();  // this CTA's sums are read
}

constexpr int lora_ceil(int64_t n, int64_t of) { return static_cast<int>((n + of - 1) / of); }

// Parts that the columns are cut into, at most: enough CTAs for few tokens, and at most so many parts of h in all
// (or one a token), a bound that fewer tokens do not pass: a workspace does for fewer tokens too.
constexpr int kLoraMaxParts = 16384;
int lora_max_splits(int tokens) { return std::clamp(kLoraMaxParts / tokens, 1, kLoraMaxSplits); }
int64_t lora_max_parts(int64_t tokens) {
    return std::min<int64_t>(kLoraMaxSplits * tokens, std::max<int64_t>(kLoraMaxParts, tokens));
}

// Tiles of `size` tokens there may be: each but an adapter's last one is full.
int64_t lora_most_tiles(int64_t tokens, int64_t adapters, int size) {
    return std::min(tokens, tokens / size + adapters);
}

// The workspace: h, then (where there is a plan) the tiles, the places, the counts.
struct LoraLayout {
    int64_t tiles, places, counts, ntiles, bytes;
};
LoraLayout lora_layout(int64_t tokens, int64_t adapters, int64_t max_rank) {
    LoraLayout l{};
    tokens = std::max<int64_t>(tokens, 1);
    const auto take = [&](int64_t n) {
        const int64_t at = l.bytes;
        l.bytes += (n + 15) & ~int64_t{15};
        return at;
    };
    take(4 * lora_max_parts(tokens) * lora_h_pitch(static_cast<int>(max_rank)));
    if (tokens > kLoraScan) {
        l.tiles = take(sizeof(LoraTile) * lora_most_tiles(tokens, adapters, kLoraTile));
        l.places = take(4 * tokens);
        l.counts = take(4 * adapters);
        l.ntiles = take(4);
    }
    return l;
}

// Launches `kernel`, which waits itself for the kernel before it where it needs it.
template <class K>
int32_t lora_start(K *kernel, dim3 grid, size_t smem, const LoraArgs &p, bool early, cudaStream_t stream,
                   const char *name) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 1 : 0;
    GLMVX_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return launch_status(name);
}

template <class W, int MT, int MW, int NT>
int32_t lora_shrink(const LoraArgs &p, dim3 grid, bool vec, cudaStream_t stream) {
    const auto kernel = vec ? lora_shrink_kernel<W, MT, MW, NT, true> : lora_shrink_kernel<W, MT, MW, NT, false>;
    return lora_start(kernel, grid, 0, p, p.tiles, stream, "lora_shrink_kernel");
}

template <class W, int NT, int RG, int KU, bool LONG>
int32_t lora_expand(const LoraArgs &p, dim3 grid, bool vec, cudaStream_t stream) {
    constexpr int sums = LoraExpand<W, NT, RG, KU, true, LONG>::kSums;
    const size_t smem = sizeof(float) * 2 * 8 * NT * lora_pitch<KU>(p.max_rank) + sizeof(float4) * sums;
    const auto kernel =
        vec ? lora_expand_kernel<W, NT, RG, KU, true, LONG> : lora_expand_kernel<W, NT, RG, KU, false, LONG>;
    if (const int32_t rc = allow_dynamic_smem(kernel, smem, "lora_expand smem", sizeof(LoraTiles<8 * NT>))) return rc;
    return lora_start(kernel, grid, smem, p, true, stream, "lora_expand_kernel");
}

template <class W, int MT, int MW, int RG, int KU, bool LONG>
int32_t lora_cluster(const LoraArgs &p, int tiles, bool vec, cudaStream_t stream) {
    const auto kernel =
        vec ? lora_cluster_kernel<W, MT, MW, RG, KU, true, LONG> : lora_cluster_kernel<W, MT, MW, RG, KU, false, LONG>;
    constexpr int sums = LoraExpand<W, 1, RG, KU, true, LONG>::kSums;
    const size_t smem =
        sizeof(float) * (16 * lora_pitch<KU>(p.max_rank) + 8 * p.max_rank) + sizeof(float4) * sums;
    constexpr size_t fixed = sizeof(LoraTiles<8>) + sizeof(typename LoraShrink<W, MT, MW, 1, true>::Shared);
    if (const int32_t rc = allow_dynamic_smem(kernel, smem, "lora_cluster smem", fixed)) return rc;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kLoraCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * kLoraCluster);
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    GLMVX_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return launch_status("lora_cluster_kernel");
}

template <class W, int NT>
int32_t lora_launch(LoraArgs &p, bool vec_a, bool vec_b, cudaStream_t stream) {
    const int sms = sm_count();
    const int tiles = static_cast<int>(lora_most_tiles(p.tokens, p.adapters, 8 * NT));
    const int64_t weights = static_cast<int64_t>(p.rows + p.cols) * p.max_rank * static_cast<int64_t>(sizeof(W));
    if (NT == 1 && tiles * kLoraCluster <= sms && weights <= kLoraSmall) {
        const bool vec = vec_a && vec_b;
        constexpr int kTwo = sizeof(W) == 4 ? 1 : 2;
        if (p.max_rank <= 16) return lora_cluster<W, 1, 1, kTwo, 1, false>(p, tiles, vec, stream);
        if (p.max_rank <= 32) return lora_cluster<W, 2, 1, 1, kTwo, false>(p, tiles, vec, stream);
        if (p.max_rank <= kLoraChain) return lora_cluster<W, 2, 2, 1, kTwo, false>(p, tiles, vec, stream);
        return lora_cluster<W, 2, 2, 1, kTwo, true>(p, tiles, vec, stream);
    }
    if (p.tiles) {
        static_assert(NT == 1 || 8 * NT == kLoraTile);
        lora_plan_kernel<<<1, kLoraPlanThreads, 0, stream>>>(p);
        if (const int32_t rc = launch_status("lora_plan_kernel")) return rc;
    }
    // Columns in as many parts as give two items an SM were every tile full, none shorter than four units a warp.
    // Half as many: 1000 tokens 39.4 us against 32.1, 48 tokens of rank 64 13.1 against 12.5; twice as many: 39.8
    // and, 4096 tokens, 140.0 against 138.1.
    const int full = lora_ceil(p.tokens, 8 * NT), all_units = lora_ceil(p.cols, 16);
    p.splits = std::clamp(2 * sms / full, 1, std::min(lora_max_splits(p.tokens), lora_ceil(all_units, 4 * kLoraWarps)));
    p.units = lora_ceil(all_units, p.splits);
    p.splits = lora_ceil(all_units, p.units);
    const int quads = 8 * NT * lora_ceil(p.max_rank, 16) * 4;  // sums that expand makes of a tile's parts of h
    while (2 * quads << p.team <= kLoraThreads && 1 << p.team < p.splits) ++p.team;
    // Ranks a shrink item takes.  64 instead of 32 for rank 32: 161 us against 138 (4096 tokens); 64 instead of 16 for
    // rank 16: 149 against 116, 64 tokens 22.4 against 20.8; 32 instead of 64 for rank 64: 1000 tokens 34.2 against
    // 32.1, 64 tokens 38.3 against 37.4.
    const int ranks = p.max_rank <= 16 ? 16 : p.max_rank <= 32 ? 32 : kLoraRankChunk;
    // Two CTAs an SM share the work, whatever the number of tiles turns out to be; fewer where there is less.
    const auto ctas = [&](int64_t items) {
        return dim3(static_cast<unsigned>(std::min<int64_t>(items * tiles, 2 * sms)));
    };
    const dim3 grid = ctas(int64_t{p.splits} * lora_ceil(p.max_rank, ranks));
    int32_t rc = kOk;
    if (ranks == 16) rc = lora_shrink<W, 1, 1, NT>(p, grid, vec_a, stream);
    else if (ranks == 32) rc = lora_shrink<W, 2, 1, NT>(p, grid, vec_a, stream);
    else rc = lora_shrink<W, 2, 2, NT>(p, grid, vec_a, stream);
    if (rc) return rc;
    // Ranks a chunk: 32 (16-byte loads of 16-bit weights) where there are more than 16: 4096 tokens of rank 32 138 us,
    // of rank 64 187, by 16 at a time 146 and 206; F32 weights fill 16 bytes with 16 ranks.  Rank 16 and few tokens
    // take twice the rows a step: 64 tokens 20.8 us against 23.7.
    const dim3 out = ctas(lora_ceil(p.rows, kLoraWarps * kLoraRows));
    constexpr int kWide = sizeof(W) == 4 ? 1 : 2;
    if (p.max_rank > kLoraChain) return lora_expand<W, NT, 1, kWide, true>(p, out, vec_b, stream);
    if (sizeof(W) == 4 || p.max_rank <= 16)
        return lora_expand<W, NT, NT == 1 && sizeof(W) == 2 ? 2 : 1, 1, false>(p, out, vec_b, stream);
    return lora_expand<W, NT, 1, kWide, false>(p, out, vec_b, stream);
}

}  // namespace

}  // namespace glmvx

using namespace glmvx;

GLMVX_EXPORT int64_t glmvx_lora_workspace_bytes(int32_t tokens, int32_t adapters, int32_t max_rank) {
    if (tokens < 0 || tokens > 1 << 20 || adapters < 1 || adapters > 1 << 24 || max_rank < 1 || max_rank > kLoraMaxRank)
        return kInvalid;
    return lora_layout(tokens, adapters, max_rank).bytes;
}

GLMVX_EXPORT int32_t glmvx_lora_add(float *y, int64_t y_stride, const float *x, int64_t x_stride,
                                    const int32_t *adapter_ids, int32_t kind, const void *a, const void *b,
                                    const int32_t *ranks, const float *scales, int32_t tokens, int32_t rows,
                                    int32_t cols, int32_t adapters, int32_t max_rank, void *workspace,
                                    uint64_t workspace_bytes, void *stream) {
    if (tokens < 0 || tokens > 1 << 20 || rows < 1 || cols < 1 || adapters < 1 || rows > 1 << 22 || cols > 1 << 22 ||
        adapters > 1 << 24)
        return set_error("lora_add: invalid dimensions"), kInvalid;
    if (max_rank < 1 || max_rank > kLoraMaxRank)
        return set_error("lora_add: max_rank must be 1..%d", kLoraMaxRank), kInvalid;
    if (kind != 0 && kind != 1 && kind != 30)
        return set_error("lora_add: adapters are kind 0 (F32), 1 (F16) or 30 (BF16), not %d", kind), kUnsupported;
    if (!tokens) return kOk;
    if (tokens > 1 && (y_stride < rows || x_stride < cols))
        return set_error("lora_add: row strides are shorter than the rows"), kInvalid;
    if (!y || !x || !adapter_ids || !a || !b || !ranks || !scales || !workspace)
        return set_error("lora_add: null pointer"), kInvalid;
    const auto bits = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
    if (((bits(y) | bits(x) | bits(adapter_ids) | bits(ranks) | bits(scales)) & 3) || (bits(workspace) & 15) ||
        ((bits(a) | bits(b)) & (kind == 0 ? 3 : 1)))
        return set_error("lora_add: misaligned pointer"), kInvalid;
    const LoraLayout layout = lora_layout(tokens, adapters, max_rank);
    if (workspace_bytes < static_cast<uint64_t>(layout.bytes))
        return set_error("lora_add: workspace smaller than glmvx_lora_workspace_bytes"), kInvalid;
    LoraArgs p{};
    p.y = y, p.x = x, p.ids = adapter_ids, p.a = a, p.b = b, p.ranks = ranks, p.scales = scales;
    p.y_stride = y_stride, p.x_stride = x_stride;
    p.tokens = tokens, p.rows = rows, p.cols = cols, p.adapters = adapters, p.max_rank = max_rank;
    p.err = device_error_word();
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    p.h = reinterpret_cast<float *>(ws);
    if (tokens > kLoraScan) {
        p.tiles = reinterpret_cast<LoraTile *>(ws + layout.tiles);
        p.places = reinterpret_cast<int *>(ws + layout.places);
        p.counts = reinterpret_cast<int *>(ws + layout.counts);
        p.ntiles = reinterpret_cast<int *>(ws + layout.ntiles);
    }
    // What stands on 16-byte boundaries (8 for ranks up to 16) has kernels of its own, the rest asks how it is read:
    // 4096 tokens of rank 32 138 us, of rank 28 (quads) 158 and 31 (words) 193, all value by value 310.
    const int size = kind == 0 ? 4 : 2, per_b = kind == 0 || max_rank <= 16 ? 4 : 8;
    const auto how = [&](const void *base, int64_t pitch, int each, int group) {
        if (!(bits(base) & (group * each - 1)) && !(pitch % group)) return kLoraWhole;
        if (each == 2 && !(bits(base) & 7) && !(pitch & 3)) return kLoraQuads;
        return each == 2 && !(bits(base) & 3) ? kLoraWords : kLoraSingle;
    };
    p.how_a = how(a, cols, size, 16 / size), p.how_b = how(b, max_rank, size, per_b);
    p.how_x = how(x, tokens == 1 ? 0 : x_stride, 4, 4), p.how_y = how(y, tokens == 1 ? 0 : y_stride, 4, 4);
    const bool vec_a = p.how_a == kLoraWhole && p.how_x == kLoraWhole;
    const bool vec_b = p.how_b == kLoraWhole && p.how_y == kLoraWhole && !(rows & 3);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = tokens > kLoraScan;
    if (kind == 0) return wide ? lora_launch<float, 2>(p, vec_a, vec_b, s) : lora_launch<float, 1>(p, vec_a, vec_b, s);
    if (kind == 1)
        return wide ? lora_launch<__half, 2>(p, vec_a, vec_b, s) : lora_launch<__half, 1>(p, vec_a, vec_b, s);
    return wide ? lora_launch<__nv_bfloat16, 2>(p, vec_a, vec_b, s) : lora_launch<__nv_bfloat16, 1>(p, vec_a, vec_b, s);
}
