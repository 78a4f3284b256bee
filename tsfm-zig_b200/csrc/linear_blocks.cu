// Products over block-scaled E4M3 operands, and products grouped by expert on 16-bit or E4M3
// operands: y[r] (+)= act(x[r] W[e]^T + bias[e]) for the rows r of group e.
//
// E4M3 operands carry one FP32 scale per 128 elements of a row of x and per 128 x 128 block of W:
//   y[m, n] = sum_b xs[m, b] ws[n / 128, b] (sum_{k in block b} xq[m, k] wq[n, k]).
// The inner sums run on the tensor cores (kind::f8f6f4, FP32 accumulators) one 128-wide block of K
// at a time; the scales differ from block to block, so each block's sums leave tensor memory and
// are added, scaled, into FP32 registers. 16-bit operands have no scales: their sums stay in tensor
// memory over the whole of K. The tensor cores cut each of their additions off, so that FP32 outputs of the
// 16-bit products end nearer zero by about 1e-9 K of their size (K 256 2.0e-7, K 4096 3.9e-6; E4M3, four
// additions at a time, 8e-8 in all).
//
// One CTA per SM walks tiles of 128 rows x BN columns, BN 64 or 128, or a CTA pair tiles of 256 x 256:
//   warp 0      TMA producer (and warp 2, for alternate stages, below 256 columns): K-major tiles of x
//               and W with the 128-byte swizzle into a ring of STAGES, 128 bytes of K a stage. For
//               gated pairs ([g | u] blocks of 256 rows) W's box holds BN / 2 rows of each, so that
//               a tile holds g and u of the same columns.
//   warp 1      tensor-memory allocation, MMA issue (one lane) into accumulators in tensor memory:
//               one per tile (16 bits, two in turn) or one per block of K (E4M3).
//   warp 2      E4M3, 256 columns: issues the TMA stores of the boxes that the epilogue fills.
//   warp 3      E4M3: the scales of the tile's rows and columns into a ring of shared memory, four
//               blocks of K at a time, ahead of the tiles that need them, marked where a product of two
//               of them leaves FP32 (this costs the 256-wide tiles 1.3 to 2 %; looked for by the epilogue, 4 %).
//   warps 4..   epilogue: a thread owns a row and 128 (below 256 columns: 64) of its columns, which
//               are whole 32-byte sectors of y (columns past N, other alignments and sums into y pass
//               through 4 KB of shared memory a warp). E4M3 on 256 columns with a 16-bit y: through
//               boxes of 64 columns to TMA stores, so that the tile leaves while the next is summed.
// E4M3 on 256 columns: each warpgroup of the epilogue has accumulators of its own (two of 128
// columns), filled by MMAs of its half of the columns, so that one half's sums are
// loaded while the other half's are made.
// Rows of a group that end inside a tile: the tile's other rows hold whatever follows in x (or the
// stage's old bytes), are computed and not stored.
//
// What bounds it (B200, 148 SMs, random operands):
//   16 bits, 256 x 256  the tensor cores: their pipe is active 82 % of the time at M 16384, N 4096,
//                       K 1024 in 16 groups; M 32768 in 32 groups takes 179 to 190 us after a pause (1450
//                       to 1530 TFLOP/s), in a row of calls what the power limit leaves (the same 266,000
//                       cycles at 1.06 to 1.3 GHz, 200 to 250 us).
//   E4M3, 256 x 256     handing accumulators over: a block of K takes 880 cycles (K 4096: 297 us for
//                       M 75776, N 1024, 2140 TFLOP/s) where the tensor cores need 512. When it took
//                       850, it took 705 with nothing added to the sums, 693 with one load a pass: two
//                       accumulators a half and 1390 cycles for one's round (MMA, commit, wait, loads,
//                       hand-back). At K 768 a tile takes 7400 cycles (165 us at M 73856, N 2304, 1580
//                       TFLOP/s), about 1500 of them its finish.
//                       128 sums and 64 loaded values a thread leave no room for more warps, 512
//                       columns of tensor memory none for more accumulators.
//   few rows            the start and W's bytes; groups of few rows have a kernel of their own below.
// Tried and slower: 128 x 256 tiles on one SM (their loads alone 526 ns a block of K), there also 16
// epilogue warps of 64 columns (registers spill; 401 ns against 377 for 8 warps), one MMA over all 256
// columns in place of two halves (875 cycles a block), test_wait in place of try_wait (2 %).
//
// Groups: the offsets are device memory, so the tile list is made on the device: warp 0 scans the
// groups' row counts into shared memory before the roles start (32 groups a step). Offsets are
// clamped to [0, M] and to be nondecreasing, so no content of theirs reaches outside x and y.
// Every element is summed over K in a fixed order: no atomics, results do not depend on timing.
// The kernels are launched as dependent ones (dep_wait): in a row of calls the set-up runs under the tail
// of the call before. us per call, before / with it: one row (N 2304 K 768) 5.5 / 4.7, 77 rows (N 1000
// K 1032) 7.6 / 6.6, 5000 rows in 8 groups (N 672 K 768) 15.0 / 14.3; large products the same.
#include "kernels.h"
#include "ptx.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tsfm {

namespace {

// Blocks of K whose scales share a slot of the ring, and the slots.
constexpr int kScaleQuad = 4, kScaleSlots = 4;
constexpr int kScaleSlotBytes = kScaleQuad * (128 + 2 + 1) * 4;  // [row][block of K], [half tile][block of K], spare
// In place of W's first scale, which is then in the spare words: a scale of the slot is wide. (A NaN that no
// arithmetic gives; a caller's own is treated as a mark.)
constexpr uint32_t kWideMark = 0x7fedcba9u;

// KIND: element type of x and W (E_F16, E_BF16, E_U8 = E4M3).
template <int KIND, int BN>
struct BlkCfg {
    static_assert(BN == 64 || BN == 128 || BN == 256, "tile widths");
    static constexpr bool F8 = KIND == E_U8;
    static constexpr bool PAIR = BN == 256;
    static constexpr int EPI_WARPS = BN == 64 ? 4 : 8;
    static constexpr int THREADS = 128 + 32 * EPI_WARPS;
    static constexpr int TILE_M = PAIR ? 256 : 128;
    static constexpr int A_BOX = PAIR ? 128 : 32;  // rows of x per TMA box
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;   // rows of W in this CTA's shared memory
    static constexpr int B_BYTES = B_ROWS * 128;
    static constexpr int STAGES = BN == 64 ? 8 : PAIR && F8 ? 4 : 5;
    static constexpr int PRODUCERS = PAIR ? 1 : 2;
    // Accumulators: NH column parts of BN / NH columns, NBUF of each.
    static constexpr int NH = F8 && BN == 256 ? 2 : 1;
    static constexpr int NBUF = !F8 || BN == 256 ? 2 : 512 / BN;
    static constexpr int TMEM_COLS = NBUF * BN;
    // E4M3 on 256 columns stores 16-bit outputs by TMA from two 4 KB boxes per epilogue warp.
    static constexpr bool TMA_Y = F8 && PAIR;
    static constexpr int BOXES = TMA_Y ? 2 : 1;
    static constexpr int EPI_OFF = STAGES * (A_BYTES + B_BYTES);
    static constexpr int SCALE_OFF = EPI_OFF + EPI_WARPS * BOXES * 4096;
    static constexpr int BAR_OFF = SCALE_OFF + (F8 ? kScaleSlots * kScaleSlotBytes : 0);
    static constexpr int GROUP_OFF = BAR_OFF + 512;
    static int smem(int64_t groups) { return 1024 + GROUP_OFF + 8 * (int)(groups + 1); }
    static_assert((2 * STAGES + 2 * NH * NBUF + 2 * kScaleSlots + 2 * EPI_WARPS + 2) * 8 <= 512, "barriers");
};

struct BlkArgs {
    int64_t M, N, K;
    const int32_t *offsets;
    int groups, n_tiles, num_k;
    uint32_t n_inv;  // (2^32 - 1) / n_tiles
    const float *xs, *ws;
    int64_t ld_xs, ld_ws, ws_group;
    int ws_blocks;  // blocks of N
    const float *bias;
    void *y;
    int64_t ldy, ycols;
    int y_dtype, accumulate, act;
    int vec;       // y's base and row stride suit 4-element stores
    int vec32;     // and 32-byte ones
    int y_tma;     // tiles leave through tmY
    int split;     // CTAs of a cluster that share a tile's K (1: none)
    int *err;
};

// u / (1 + e^-u).
__device__ __forceinline__ float silu_fast(float u) { return u * rcp_approx(1.0f + ex2_approx(-1.44269504f * u)); }

// g silu(u) of two columns with one reciprocal, 1 / a = b / (a b): the special-function unit, 16 results a
// clock, bounds the finish of a gated tile. Each exponential is held to 2^60, so that the product of the
// factors stays in range and a NaN in its own column; below kGateFar that gives u 2^-60 in place of silu
// (held to -1: g times it stays finite), which gate_far makes up for.
constexpr float kGateFar = -41.588831f;  // e^-u = 2^60
__device__ __forceinline__ float2 gate_pair(float2 g, float2 u) {
    const float a = 1.0f + fminf(ex2_approx(-1.44269504f * u.x), 0x1p60f);
    const float b = 1.0f + fminf(ex2_approx(-1.44269504f * u.y), 0x1p60f);
    const float r = rcp_approx(a * b);
    return make_float2(g.x * max_nan(u.x * (b * r), -1.0f), g.y * max_nan(u.y * (a * r), -1.0f));
}

// gate_pair's result f of a column, times 2^60 e^u where u is below kGateFar: to zero, as silu goes, and to
// NaN at -infinity (-infinity / infinity).
__device__ __forceinline__ float gate_far(float f, float u) {
    if (!(u < kGateFar)) return f;
    return f * (ex2_approx(fmaf(1.44269504f, u, 60.0f)) + (u - u));
}

// A block's scale is the FP32 product s = xs ws, a normal number but for odd data. wide_scale: it is past FP32,
// or subnormal and not exact. (A row of zeros has the quantiser's least scale, a power of two; and since a
// block's sum is below 2^25, a scale below 2^-176 gives 0 in any case.)
__device__ __forceinline__ bool wide_scale(float xs, float ws) {
    const float s = xs * ws, m = fabsf(s);
    if (m > 1.0f) return m > 0x1.fffffep127f && fabsf(xs) <= 0x1.fffffep127f && fabsf(ws) <= 0x1.fffffep127f;
    if (!(m < 0x1p-126f)) return false;
    const float t = (xs * 0x1p50f) * (ws * 0x1p50f);
    return fabsf(t) >= 0x1p-76f && s * 0x1p100f != t;
}

// Such a block's sums are multiplied by a power of two (returned) before they meet s, now xs ws over that
// power: 2^127 or 2^-100. Sums are multiples of 2^-18, so the first step is exact or leaves FP32 as the result
// does; s held to FP32's largest number changes none that is not past FP32 itself.
__device__ __forceinline__ float split_scale(float xs, float ws, float &s) {
    s = xs * ws;
    if (!wide_scale(xs, ws)) return 1.0f;
    if (fabsf(s) > 1.0f) {
        s = copysignf(fminf(fabsf((xs * 0x1p-64f) * (ws * 0x1p-63f)), 0x1.fffffep127f), s);
        return 0x1p127f;
    }
    s = (xs * 0x1p50f) * (ws * 0x1p50f);
    return 0x1p-100f;
}

__device__ __forceinline__ bool ordinary_scales(float least, float most) { return least >= 0x1p-126f && most <= 0x1.fffffep127f; }

// Bias of four consecutive columns of group e (zero past N).
__device__ __forceinline__ void bias_quad(const BlkArgs &a, int e, int64_t col, float (&b)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = a.bias && col + j < a.N ? a.bias[e * a.N + col + j] : 0.0f;
}

// y of four consecutive columns of one row (the last columns of a row: fewer): adds to it or not,
// activates and stores.
__device__ __forceinline__ void store_quad(const BlkArgs &a, int64_t row, int64_t col, float (&v)[4]) {
    const int64_t at = row * a.ldy + col;
    const int n = (int)min((int64_t)4, a.ycols - col);
    if (a.accumulate) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) v[j] += static_cast<const float *>(a.y)[at + j];
    }
    if (a.act == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaxf(v[j], 0.0f);
    }
    if (a.y_dtype == TSFM_DTYPE_F32) {
        float *o = static_cast<float *>(a.y) + at;
        if (a.vec && n == 4) {
            *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) o[j] = v[j];
        }
    } else {
        const bool h = a.y_dtype == TSFM_DTYPE_F16;
        const uint32_t w[2] = {h ? pack16<true>(v[0], v[1]) : pack16<false>(v[0], v[1]),
                               h ? pack16<true>(v[2], v[3]) : pack16<false>(v[2], v[3])};
        uint16_t *o = static_cast<uint16_t *>(a.y) + at;
        if (a.vec && n == 4) {
            *reinterpret_cast<uint2 *>(o) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) o[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
        }
    }
}

// 32 consecutive values of one row, 32 bytes a store; o 32-byte aligned.
template <int DT>
__device__ __forceinline__ void store_sectors(void *o, const float (&v)[32]) {
    if constexpr (DT == TSFM_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(v) + 8 * i;
            st_global_v8(static_cast<float *>(o) + 8 * i, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = pack16<DT == TSFM_DTYPE_F16>(v[16 * i + 2 * j], v[16 * i + 2 * j + 1]);
            st_global_v8(static_cast<uint16_t *>(o) + 16 * i, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
        }
    }
}

// The groups' rows and tiles of TILE_M rows, by one warp: group e has rows [g_row[e], g_row[e + 1]) and
// row tiles [g_tile[e], g_tile[e + 1]). No offsets: one group of M rows.
// `first` and `o` are offsets[0] and a lane's first offset. All that runs before the first load of an operand runs once per launch, from
// instructions that no cache of the SM holds yet: about 30 cycles each, so loops stay rolled (unrolled,
// the two scans took 2.5 us) and divisions are by reciprocals from the host.
template <int TILE_M>
__device__ __forceinline__ void scan_groups(const BlkArgs &a, int lane, int first, int o, int *g_row, int *g_tile) {
    if (a.offsets == nullptr) {
        if (lane == 0) {
            g_row[0] = g_tile[0] = 0;
            g_row[1] = (int)a.M;
            g_tile[1] = (int)((a.M + TILE_M - 1) / TILE_M);
        }
        return;
    }
    const int M = (int)a.M;
    int end = min(max(first, 0), M);  // running maximum of the offsets
    int tiles = 0;
    if (lane == 0) {
        g_row[0] = end;
        g_tile[0] = 0;
    }
    for (int base = 0; base < a.groups; base += 32) {
        const int e = base + lane;
        o = max(min(max(o, 0), M), end);
#pragma unroll 1
        for (int d = 1; d < 32; d <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, o, d);
            if (lane >= d) o = max(o, p);
        }
        int start = __shfl_up_sync(0xffffffffu, o, 1);
        if (lane == 0) start = end;
        int t = (o - start + TILE_M - 1) / TILE_M;
#pragma unroll 1
        for (int d = 1; d < 32; d <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, t, d);
            if (lane >= d) t += p;
        }
        if (e < a.groups) {
            g_row[e + 1] = o;
            g_tile[e + 1] = tiles + t;
        }
        end = __shfl_sync(0xffffffffu, o, 31);
        tiles += __shfl_sync(0xffffffffu, t, 31);
        o = e + 32 < a.groups ? a.offsets[e + 33] : 0;
    }
}

// Tile t of n_tiles per row tile: its row tile (returned) and the rest. The product with n_inv is short
// of t / n_tiles by less than one.
__device__ __forceinline__ int split_tile(const BlkArgs &a, int t, int &nt) {
    int mt = (int)__umulhi((uint32_t)t, a.n_inv);
    nt = t - mt * a.n_tiles;
    if (nt >= a.n_tiles) {
        nt -= a.n_tiles;
        ++mt;
    }
    return mt;
}

// The group of row tile mt: the last e with g_tile[e] <= mt.
__device__ __forceinline__ int group_of(const int *g_tile, int groups, int mt) {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (g_tile[mid] <= mt)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <int KIND, int BN>
__global__ void __launch_bounds__((BlkCfg<KIND, BN>::THREADS), 1)
    linear_blocks_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmY, BlkArgs a) {
    using C = BlkCfg<KIND, BN>;
    constexpr bool F8 = C::F8, PAIR = C::PAIR;
    constexpr int STAGES = C::STAGES, NBUF = C::NBUF, NH = C::NH;
    constexpr int BK = F8 ? 128 : 64;  // elements of K per stage
    // 384 threads launch with 168 registers each; the epilogue's two warpgroups (128 sums and 64 loaded
    // values a thread) take them from the first one: 64,512 = 128 x 40 + 256 x 232.
    constexpr bool SPLIT_REGS = F8 && BN == 256;
    constexpr uint32_t IDESC = idesc_f32acc(KIND == E_BF16 ? 1u : 0u, C::TILE_M, BN / NH);
    const int cta_split = F8 && BN == 64 ? a.split : 1;  // CTAs that share a tile's K
    const int cta = PAIR ? 2 : cta_split;                // CTAs of a cluster
    const uint32_t rank = cta > 1 ? cluster_ctarank() : 0u;
    const bool leader = !PAIR || rank == 0;
    const int unit = (int)blockIdx.x / cta, units = (int)gridDim.x / cta;

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem;
    uint8_t *sB = smem + STAGES * C::A_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);
    uint64_t *empty = full + STAGES;
    uint64_t *pfull = empty + STAGES;       // accumulators, [NH][NBUF]
    uint64_t *pempty = pfull + NH * NBUF;
    uint64_t *sfull = pempty + NH * NBUF;   // scales
    uint64_t *sempty = sfull + kScaleSlots;
    uint64_t *bfull = sempty + kScaleSlots;  // staging boxes, per epilogue warp
    uint64_t *bempty = bfull + C::EPI_WARPS;
    uint64_t *drain = bempty + C::EPI_WARPS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *g_row = reinterpret_cast<int *>(smem + C::GROUP_OFF);  // group e has rows [g_row[e], g_row[e + 1])
    int *g_tile = g_row + a.groups + 1;                         // and row tiles [g_tile[e], g_tile[e + 1])

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 2) {
        for (uint64_t *b = full + lane; b <= drain; b += 32)
            mbar_init(b, b >= pempty && b < sfull    ? (PAIR ? 2 : 1) * C::EPI_WARPS / NH  // one arrival per epilogue warp
                         : b >= sempty && b < bfull  ? C::EPI_WARPS
                                                     : 1);
        if (lane == 0) *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, C::TMEM_COLS);
            tmem_relinquish();
        }
    }
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    dep_wait();
    if (warp == 0) {
        const int first = a.offsets ? *a.offsets : 0;
        const int o = a.offsets && lane < a.groups ? a.offsets[lane + 1] : 0;
        scan_groups<C::TILE_M>(a, lane, first, o, g_row, g_tile);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();
    dep_release();  // (not before this CTA holds its tensor memory)
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    struct Tile {
        int e, row0, row_end;  // group, first row of this CTA's 128 rows, end of the group
        int b0, b1;            // W rows of the tile's first and second BN / 2 columns
        int ocol;              // first output column
    };
    const int tiles = g_tile[a.groups] * a.n_tiles;  // the host has checked that this fits
    const bool glu = a.act == ACT_GLU;
    auto tile_at = [&](int t) {
        Tile r;
        int nt;
        const int mt = split_tile(a, t, nt);
        const int lo = r.e = group_of(g_tile, a.groups, mt);
        r.row0 = g_row[lo] + (mt - g_tile[lo]) * C::TILE_M + (PAIR ? (int)rank * 128 : 0);
        r.row_end = g_row[lo + 1];
        if (glu) {
            r.ocol = nt * (BN / 2);
            r.b0 = (r.ocol >> 7) * 256 + (r.ocol & 127);
            r.b1 = r.b0 + 128;
        } else {
            r.ocol = r.b0 = nt * BN;
            r.b1 = r.b0 + BN / 2;
        }
        return r;
    };
    // This CTA's blocks of K.
    const int kb0 = cta_split > 1 ? (int)((int64_t)a.num_k * rank / cta) : 0;
    const int kb1 = cta_split > 1 ? (int)((int64_t)a.num_k * (rank + 1) / cta) : a.num_k;
    const int kbn = kb1 - kb0;
    // Waits on barriers that hand over stages and accumulators. In a pair the other CTA's arrivals
    // stand for completed copies, MMAs and tensor-memory loads, none of them accesses that an
    // acquire at cluster scope would order: the plain form does, and the other costs over 1000 cycles.
    // Every role's loop is warp-uniform, with one elected lane that issues.
    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        return mbar_wait_warp(bar, parity, abort_flag, a.err, site);
    };

    if (warp < 4) {
        if constexpr (SPLIT_REGS) regs_dec<40>();
        if (warp == 0 || (C::PRODUCERS == 2 && warp == 2)) {
            // Producers: of two, stage use number i (over all tiles) belongs to warp 2 (i % 2).
            const bool el = elect_one();
            const int mine = warp >> 1;
            int s = mine % STAGES, turn = 0;  // turn: parity of i for the next block of K
            uint32_t ph = 0, issued = 0, issued_ph = 0;
            bool ok = true;
            for (int t = unit; t < tiles && ok; t += units) {
                const Tile tl = tile_at(t);
                const int na = min(128 / C::A_BOX, max(0, (tl.row_end - tl.row0 + C::A_BOX - 1) / C::A_BOX));
                const int c1 = glu ? tl.ocol & 127 : tl.b0, c3 = glu ? tl.ocol >> 7 : 0;
                for (int kb = kb0; kb < kb1; ++kb, turn ^= C::PRODUCERS - 1) {
                    if (turn != mine) continue;
                    ok = wait(&empty[s], ph ^ 1u, ERR_SITE_BLOCKS_PRODUCER);
                    if (!ok) break;
                    const int32_t kc = kb * BK;
                    if (el) {
                        if constexpr (PAIR) {
                            // Each CTA loads its 128 rows of x and half of W's rows.
                            if (leader) mbar_arrive_expect_tx(&full[s], 2 * (C::A_BYTES + C::B_BYTES));
                            const uint32_t fb = mapa_shared(&full[s], 0);
                            tma_load_2d_pair(sA + s * C::A_BYTES, &tmA, fb, kc, tl.row0);
                            tma_load_5d_pair(sB + s * C::B_BYTES, &tmB, fb, kc, glu ? c1 : c1 + (int)rank * (BN / 2),
                                             glu ? (int)rank : 0, c3, tl.e);
                        } else {
                            mbar_arrive_expect_tx(&full[s], na * C::A_BOX * 128 + C::B_BYTES);
                            for (int i = 0; i < na; ++i)
                                tma_load_2d(sA + s * C::A_BYTES + i * C::A_BOX * 128, &tmA, &full[s], kc,
                                            tl.row0 + i * C::A_BOX);
                            tma_load_5d(sB + s * C::B_BYTES, &tmB, &full[s], kc, c1, 0, c3, tl.e);
                        }
                    }
                    __syncwarp();
                    issued |= 1u << s;
                    issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
                    s += C::PRODUCERS;
                    if (s >= STAGES) {
                        s -= STAGES;
                        ph ^= 1u;
                    }
                }
            }
            if (!ok) {
                // Loads in flight land before the CTA can exit (bounded; a pair's second CTA, whose
                // loads count on the first one's barriers, waits by the clock).
                const unsigned long long t0 = globaltimer_ns();
                if (PAIR && !leader) {
                    while (globaltimer_ns() - t0 < 1000000ull) {
                    }
                } else {
                    for (int i = 0; i < STAGES; ++i) {
                        if (!((issued >> i) & 1u)) continue;
                        while (!mbar_try_wait(&full[i], (issued_ph >> i) & 1u) && globaltimer_ns() - t0 < 100000000ull) {
                        }
                    }
                }
            }
        } else if (warp == 1) {
            if (leader) {
                const bool el = elect_one();
                int s = 0, buf = 0;
                uint32_t ph = 0, bph = 0;
                bool ok = true;
                const uint64_t ad0 = sdesc_k128(sA), bd0 = sdesc_k128(sB);
                auto commit = [&](uint64_t *bar) {
                    if constexpr (PAIR) {
                        mma_commit_pair(mapa_shared(bar, 0));
                        mma_commit_pair(mapa_shared(bar, 1));
                    } else {
                        mma_commit(bar);
                    }
                };
                for (int t = unit; t < tiles && ok; t += units) {
                    for (int kb = 0; kb < kbn; ++kb) {
                        ok = wait(&full[s], ph, ERR_SITE_BLOCKS_MMA_FULL);
                        if (!ok) break;
                        const uint64_t ad = ad0 + (uint64_t)(s * (C::A_BYTES >> 4)), bd = bd0 + (uint64_t)(s * (C::B_BYTES >> 4));
                        const bool last = F8 || kb == kbn - 1;
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            const int acc = h * NBUF + buf;
                            if (F8 || kb == 0) {
                                ok = wait(&pempty[acc], bph ^ 1u, ERR_SITE_BLOCKS_MMA_EMPTY);
                                if (!ok) break;
                            }
                            tc_fence_after();
                            const uint32_t d = tmem_base + (uint32_t)(acc * (BN / NH));
                            const uint64_t bh = bd + (uint64_t)(h * (C::B_BYTES / NH >> 4));
                            if (el) {
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk) {
                                    const uint32_t accum = F8 ? kk != 0 : (kb | kk) != 0;
                                    if constexpr (F8) {
                                        if constexpr (PAIR)
                                            mma_f8kind_pair(d, ad + 2 * kk, bh + 2 * kk, IDESC, accum);
                                        else
                                            mma_f8kind(d, ad + 2 * kk, bh + 2 * kk, IDESC, accum);
                                    } else if constexpr (PAIR) {
                                        mma_f16kind_pair(d, ad + 2 * kk, bh + 2 * kk, IDESC, accum);
                                    } else {
                                        mma_f16kind(d, ad + 2 * kk, bh + 2 * kk, IDESC, accum);
                                    }
                                }
                                if (last) commit(&pfull[acc]);
                                if (h == NH - 1) commit(&empty[s]);
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                        if (last && ++buf == NBUF) {
                            buf = 0;
                            bph ^= 1u;
                        }
                        if (++s == STAGES) {
                            s = 0;
                            ph ^= 1u;
                        }
                    }
                }
                // All MMAs issued by this warp have completed once `drain` fires; the tensor memory can
                // then be released safely even on the abort path.
                if (el) {
                    if constexpr (PAIR)
                        mma_commit_pair(mapa_shared(drain, 0));
                    else
                        mma_commit(drain);
                    const unsigned long long t0 = globaltimer_ns();
                    while (!mbar_try_wait(drain, 0)) {
                        if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
                            if (a.err) atomicCAS(a.err, 0, ERR_SITE_BLOCKS_DRAIN);
                            break;
                        }
                    }
                }
                __syncwarp();
            }
        } else if (C::TMA_Y && warp == 2) {
            // Stores: the boxes of every epilogue warp, a tile at a time (a warp whose rows end inside its
            // 32 has stored them itself).
            if (a.y_tma) {
                const bool el = elect_one();
                uint32_t bph = 0;
                bool ok = true;
                for (int t = unit; t < tiles && ok; t += units, bph ^= 1u) {
                    const Tile tl = tile_at(t);
                    for (int w = 0; w < C::EPI_WARPS; ++w) {
                        ok = wait(&bfull[w], bph, ERR_SITE_BLOCKS_EPILOGUE);
                        if (!ok) break;
                        const int wrow0 = tl.row0 + (w & 3) * 32, wrows = tl.row_end - wrow0;
                        if (el && (wrows >= 32 || (wrows > 0 && a.offsets == nullptr))) {
                            const uint8_t *b = smem + C::EPI_OFF + w * C::BOXES * 4096;
                            const int col0 = tl.ocol + (w >> 2) * 64, col1 = tl.b1 + (w >> 2) * 64;
                            if (col0 < a.ycols) tma_store_2d(&tmY, b, col0, wrow0);
                            if (!glu && col1 < a.ycols) tma_store_2d(&tmY, b + 4096, col1, wrow0);
                            bulk_commit();
                        }
                    }
                    if (el) {
                        bulk_wait_read_0();
                        for (int w = 0; w < C::EPI_WARPS; ++w) mbar_arrive(&bempty[w]);
                    }
                    __syncwarp();
                }
                // Every box has been written before the CTA exits.
                if (el) bulk_wait_all();
                __syncwarp();
            }
        } else if (F8 && warp == 3) {
            // Scales: slot = xs[128][4] then ws[2][4] (the half tiles' column blocks), by asynchronous
            // copies; past this CTA's last block of K its scales again. A slot is looked through for wide scales
            // and handed over once the copies of the next one are under way.
            int slot = 0, landing = -1;
            uint32_t ph = 0;
            bool ok = true;
            auto hand_over = [&]() {
                __syncwarp();
                const uint32_t d = smem_u32(smem) + C::SCALE_OFF + landing * kScaleSlotBytes;
                float w0[4], w1[4], x[4];
                ld_shared_v4(d + 2048, w0);
                ld_shared_v4(d + 2064, w1);
                // The smallest and the largest of xs times those of ws (a NaN is passed over).
                float x_least = 0x1.fffffep127f, x_most = 0.0f, w_least = x_least, w_most = 0.0f;
                for (int r = lane; r < 128; r += 32) {
                    ld_shared_v4(d + r * 16, x);
#pragma unroll
                    for (int j = 0; j < kScaleQuad; j += 2) {
                        x_least = fminf(fminf(x_least, fabsf(x[j])), fabsf(x[j + 1]));
                        x_most = fmaxf(fmaxf(x_most, fabsf(x[j])), fabsf(x[j + 1]));
                    }
                }
#pragma unroll
                for (int j = 0; j < kScaleQuad; ++j) {
                    w_least = fminf(fminf(w_least, fabsf(w0[j])), fabsf(w1[j]));
                    w_most = fmaxf(fmaxf(w_most, fabsf(w0[j])), fabsf(w1[j]));
                }
                bool wide = false;
                if (!__all_sync(0xffffffffu, ordinary_scales(x_least * w_least, x_most * w_most))) {
#pragma unroll 1
                    for (int r = lane; r < 128; r += 32) {
                        ld_shared_v4(d + r * 16, x);
#pragma unroll
                        for (int j = 0; j < kScaleQuad; ++j) wide = wide || wide_scale(x[j], w0[j]) || wide_scale(x[j], w1[j]);
                    }
                    wide = __any_sync(0xffffffffu, wide) != 0;
                }
                if (lane == 0) {
                    if (wide || __float_as_uint(w0[0]) == kWideMark) {
                        st_shared_f32(d + 2080, w0[0]);
                        st_shared_f32(d + 2048, __uint_as_float(kWideMark));
                    }
                    mbar_arrive(&sfull[landing]);
                }
            };
            for (int t = unit; t < tiles && ok; t += units) {
                const Tile tl = tile_at(t);
                const float *xs = a.xs + (int64_t)tl.row0 * a.ld_xs;
                const int last = tl.row_end - 1 - tl.row0;  // rows past the group's end repeat its last
                const int nb = min((lane & 4 ? tl.b1 : tl.b0) >> 7, a.ws_blocks - 1);
                const float *ws = a.ws + tl.e * a.ws_group + (int64_t)nb * a.ld_ws;
                for (int kb = kb0; kb < kb1; kb += kScaleQuad) {
                    ok = wait(&sempty[slot], ph ^ 1u, ERR_SITE_BLOCKS_PRODUCER);
                    if (!ok) break;
                    uint8_t *d = smem + C::SCALE_OFF + slot * kScaleSlotBytes;
                    const int n = min(kScaleQuad, kb1 - kb);
                    for (int r = lane; r < 128; r += 32) {
                        const float *src = xs + (int64_t)min(r, last) * a.ld_xs + kb;
#pragma unroll
                        for (int j = 0; j < kScaleQuad; ++j) cp_async_4(d + r * 16 + j * 4, src + min(j, n - 1));
                    }
                    if (lane < 8) cp_async_4(d + 2048 + lane * 4, ws + kb + min(lane & 3, n - 1));
                    cp_async_commit();
                    if (landing >= 0) {
                        cp_async_wait_1();
                        hand_over();
                    }
                    landing = slot;
                    if (++slot == kScaleSlots) {
                        slot = 0;
                        ph ^= 1u;
                    }
                }
            }
            cp_async_wait_all();
            if (ok && landing >= 0) hand_over();
        }
    } else {
        if constexpr (SPLIT_REGS) regs_inc<232>();
        constexpr int PARTS = C::EPI_WARPS / 4;  // warps that share a row's columns
        constexpr int CH = BN / PARTS / 32;      // 32-column chunks per thread
        constexpr int CPH = CH / 2;              // of each half of the tile
        const int ew = warp - 4;
        const int eg = warp & 3, part = ew >> 2;  // tensor-memory lanes [32 eg, 32 eg + 32)
        const int half = NH == 2 ? part : 0;      // this warp's accumulators
        float4 *box = reinterpret_cast<float4 *>(smem + C::EPI_OFF + ew * C::BOXES * 4096);
        int buf = 0, slot = 0;
        uint32_t bph = 0, sph = 0, boxph = 0;
        bool ok = true;
        auto wait_epi = [&](uint64_t *bar, uint32_t parity) { return wait(bar, parity, ERR_SITE_BLOCKS_EPILOGUE); };
        const uint32_t handback = PAIR ? mapa_shared(&pempty[half * NBUF], 0) : 0u;  // the MMA-issuing CTA's barriers
        auto release = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR)
                    mbar_arrive_remote(handback + 8 * buf);
                else
                    mbar_arrive(&pempty[half * NBUF + buf]);
            }
            if (++buf == NBUF) {
                buf = 0;
                bph ^= 1u;
            }
        };
        // Chunk c of this thread: 32 columns of the accumulator from acol(c), y's columns from ycol(c).
        // Gated pairs: chunk c < CPH is g's, chunk c + CPH the same columns of u.
        auto acol = [&](int c) { return NH == 2 ? c * 32 : (c / CPH) * (BN / 2) + (part * CPH + c % CPH) * 32; };
        auto ycol = [&](const Tile &tl, int c) { return (c < CPH ? tl.ocol : tl.b1) + (part * CPH + c % CPH) * 32; };
        // The bias of this lane's column of a chunk; its row's threads fetch the others' by shuffles (an
        // address for each of the 128 columns leaves no registers for the sums).
        auto lane_bias = [&](const Tile &tl, int c) {
            const int64_t col = (int64_t)ycol(tl, c) + lane;
            return col < a.N ? a.bias[tl.e * a.N + col] : 0.0f;
        };
        const uint32_t scales = smem_u32(smem) + C::SCALE_OFF;
        for (int t = unit; t < tiles && ok; t += units) {
            if (a.bias && lane < CH && !glu) {  // on its way while the sums are made
                const Tile tl = tile_at(t);
                prefetch_l1(a.bias + tl.e * a.N + min((int64_t)ycol(tl, lane), a.N - 1));
            }
            float2 acc[F8 ? CH : 1][16];
            uint32_t tbase = 0;
            if constexpr (F8) {
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[c][j] = make_float2(0.0f, 0.0f);
                for (int kb = 0; kb < kbn && ok; kb += kScaleQuad) {
                    // Four blocks' scales at once (a read per block, behind the accumulator's loads in the
                    // same queue, cost 150 cycles each): the row's times each half's.
                    ok = wait_epi(&sfull[slot], sph);
                    if (!ok) break;
                    const uint32_t sc = scales + slot * kScaleSlotBytes;
                    float xv[4], w0[4], w1[4], s0[4], s1[4];
                    ld_shared_v4(sc + (eg * 32 + lane) * 16, xv);
                    ld_shared_v4(sc + 2048, w0);
                    ld_shared_v4(sc + 2064, w1);
                    const bool wide = __float_as_uint(w0[0]) == kWideMark;
#pragma unroll
                    for (int j = 0; j < kScaleQuad; ++j) s0[j] = xv[j] * w0[j], s1[j] = xv[j] * w1[j];
                    const int n = min(kScaleQuad, kbn - kb);
                    auto used = [&]() {  // the slot's scales
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sempty[slot]);
                        if (++slot == kScaleSlots) {
                            slot = 0;
                            sph ^= 1u;
                        }
                    };
                    auto ready = [&]() {
                        ok = wait_epi(&pfull[half * NBUF + buf], bph);
                        tc_fence_after();
                        tbase = tmem_base + ((uint32_t)(eg * 32) << 16) + (uint32_t)((half * NBUF + buf) * (BN / NH));
                    };
                    if (__builtin_expect(wide, 0)) {
#pragma unroll 1
                        for (int j = 0; j < n; ++j) {
                            ready();
                            if (!ok) break;
                            const float x = ld_shared_f32(sc + (eg * 32 + lane) * 16 + 4 * j);
                            float t0, t1;
                            const float f0 = split_scale(x, ld_shared_f32(sc + (j ? 2048 + 4 * j : 2080)), t0);
                            const float f1 = split_scale(x, ld_shared_f32(sc + 2064 + 4 * j), t1);
#pragma unroll
                            for (int c = 0; c < 4 * CH; ++c) {
                                const float f = c / 4 < CPH ? f0 : f1, t = c / 4 < CPH ? t0 : t1;
                                float p[8];
                                tmem_ld8f(tbase + acol(c / 4) + c % 4 * 8, p);
                                tmem_wait_ld();
                                if (c == 4 * CH - 1) release();
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    fma_f32x2(acc[c / 4][c % 4 * 4 + i], make_float2(p[2 * i] * f, p[2 * i + 1] * f),
                                              make_float2(t, t));
                            }
                        }
                        used();
                        continue;
                    }
                    used();
#pragma unroll 1
                    for (int j = 0; j < n; ++j) {
                        ready();
                        if (!ok) break;
                        // A chunk loads while the one before it is added; the accumulator is handed back before
                        // the last additions.
                        float p0[32], p1[32];
                        tmem_ld32f(tbase + acol(0), p0);
#pragma unroll
                        for (int c = 0; c < CH; c += 2) {
                            tmem_wait_ld();
                            tmem_ld32f(tbase + acol(c + 1), p1);
                            const float2 sa = c < CPH ? make_float2(s0[0], s0[0]) : make_float2(s1[0], s1[0]);
                            const float2 sb = c + 1 < CPH ? make_float2(s0[0], s0[0]) : make_float2(s1[0], s1[0]);
#pragma unroll
                            for (int i = 0; i < 16; ++i) fma_f32x2(acc[c][i], make_float2(p0[2 * i], p0[2 * i + 1]), sa);
                            tmem_wait_ld();
                            if (c + 2 < CH)
                                tmem_ld32f(tbase + acol(c + 2), p0);
                            else
                                release();
#pragma unroll
                            for (int i = 0; i < 16; ++i) fma_f32x2(acc[c + 1][i], make_float2(p1[2 * i], p1[2 * i + 1]), sb);
                        }
#pragma unroll
                        for (int q = 0; q < kScaleQuad - 1; ++q) s0[q] = s0[q + 1], s1[q] = s1[q + 1];
                    }
                }
                if (!ok) break;
            } else {
                ok = wait_epi(&pfull[buf], bph);
                if (!ok) break;
                tc_fence_after();
                tbase = tmem_base + ((uint32_t)(eg * 32) << 16) + (uint32_t)(buf * BN);
            }
            const Tile tl = tile_at(t);
            const int wrow0 = tl.row0 + eg * 32;
            const int wrows = min(32, tl.row_end - wrow0);  // this warp's valid rows (may be <= 0)
            auto chunk = [&](int c, float (&v)[32]) {
                if constexpr (F8) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[2 * j] = acc[c][j].x, v[2 * j + 1] = acc[c][j].y;
                } else {
                    tmem_ld32f(tbase + acol(c), v);
                    tmem_wait_ld();
                }
            };
            // v to shared memory: float4 q of this thread's row at to[q ^ (lane % 8)].
            auto dump = [&](const float (&v)[32], float4 *to) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    to[q ^ (lane & 7)] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            };
            if (wrows > 0 && cta_split > 1) {
                // A share of K: the sums go to shared memory (the stages', which are all used up), row r at
                // float4 r * BN / 4, its chunks in order.
                float4 *to = reinterpret_cast<float4 *>(smem) + (eg * 32 + lane) * (BN / 4);
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    float v[32];
                    chunk(c, v);
                    dump(v, to + acol(c) / 4);
                }
            }
            const bool tma = C::TMA_Y && a.y_tma;
            const bool boxed = tma && (wrows == 32 || (wrows > 0 && a.offsets == nullptr));
            if (tma) {
                ok = wait_epi(&bempty[ew], boxph ^ 1u);
                if (!ok) break;
                boxph ^= 1u;
            }
            if constexpr (C::TMA_Y) {
                if (boxed) {
                    // 64-column boxes (rows past M and columns past N are clipped): the tile leaves while the
                    // next one is summed. One branch per step of all chunks: with branches per chunk and word
                    // this part took 2100 cycles a tile.
                    if (glu) {
                        float least = 0.0f;
#pragma unroll
                        for (int c = 0; c < CPH; ++c)
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float2 u = acc[c + CPH][j];
                                acc[c][j] = gate_pair(acc[c][j], u);
                                least = fminf(fminf(least, u.x), u.y);
                            }
                        if (least < kGateFar) {
#pragma unroll
                            for (int c = 0; c < CPH; ++c)
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    acc[c][j].x = gate_far(acc[c][j].x, acc[c + CPH][j].x);
                                    acc[c][j].y = gate_far(acc[c][j].y, acc[c + CPH][j].y);
                                }
                        }
                    } else if (a.bias) {
#pragma unroll
                        for (int c = 0; c < CH; ++c) {
                            const float b = lane_bias(tl, c);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                acc[c][j].x += __shfl_sync(0xffffffffu, b, 2 * j);
                                acc[c][j].y += __shfl_sync(0xffffffffu, b, 2 * j + 1);
                            }
                        }
                    }
                    if (a.act == 1) {
#pragma unroll
                        for (int c = 0; c < CH; ++c)
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                acc[c][j].x = fmaxf(acc[c][j].x, 0.0f);
                                acc[c][j].y = fmaxf(acc[c][j].y, 0.0f);
                            }
                    }
                    uint4 *b = reinterpret_cast<uint4 *>(box) + lane * 8;
                    auto pack = [&](auto half) {
                        constexpr bool F16 = decltype(half)::value;
#pragma unroll
                        for (int c = 0; c < CH; ++c) {
                            if (glu && c >= CPH) break;
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                b[(c / 2) * 256 + ((4 * (c & 1) + q) ^ (lane & 7))] =
                                    make_uint4(pack16<F16>(acc[c][4 * q].x, acc[c][4 * q].y),
                                               pack16<F16>(acc[c][4 * q + 1].x, acc[c][4 * q + 1].y),
                                               pack16<F16>(acc[c][4 * q + 2].x, acc[c][4 * q + 2].y),
                                               pack16<F16>(acc[c][4 * q + 3].x, acc[c][4 * q + 3].y));
                        }
                    };
                    if (a.y_dtype == TSFM_DTYPE_F16)
                        pack(std::true_type{});
                    else
                        pack(std::false_type{});
                }
            }
            if (wrows > 0 && cta_split == 1 && !boxed) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    if (glu && c >= CPH) break;
                    const int col0 = ycol(tl, c);
                    float v[32];
                    chunk(c, v);
                    if (glu) {
                        float u[32];
                        chunk((c + CPH) % CH, u);
                        float least = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 f = gate_pair(make_float2(v[j], v[j + 1]), make_float2(u[j], u[j + 1]));
                            v[j] = f.x, v[j + 1] = f.y;
                            least = fminf(fminf(least, u[j]), u[j + 1]);
                        }
                        if (least < kGateFar) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = gate_far(v[j], u[j]);
                        }
                    } else if (a.bias) {
                        const float b = lane_bias(tl, c);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xffffffffu, b, j);
                    }
                    if (a.vec32 && col0 + 32 <= a.ycols && !a.accumulate) {
                        // A thread's 32 columns are whole 32-byte sectors of its row.
                        if (a.act == 1) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = fmaxf(v[j], 0.0f);
                        }
                        char *o = static_cast<char *>(a.y) + ((wrow0 + lane) * a.ldy + col0) * (a.y_dtype == TSFM_DTYPE_F32 ? 4 : 2);
                        if (lane < wrows) {
                            if (a.y_dtype == TSFM_DTYPE_F32)
                                store_sectors<TSFM_DTYPE_F32>(o, v);
                            else if (a.y_dtype == TSFM_DTYPE_F16)
                                store_sectors<TSFM_DTYPE_F16>(o, v);
                            else
                                store_sectors<TSFM_DTYPE_BF16>(o, v);
                        }
                    } else {
                        // Through shared memory to row-contiguous stores of whatever alignment.
                        __syncwarp();
                        dump(v, box + lane * 8);
                        __syncwarp();
                        const int q = lane & 7;
                        if (col0 + 4 * q < a.ycols) {
#pragma unroll 1
                            for (int r = lane >> 3; r < wrows; r += 4) {
                                const float4 f = box[r * 8 + (q ^ (r & 7))];
                                float w[4] = {f.x, f.y, f.z, f.w};
                                store_quad(a, wrow0 + r, col0 + 4 * q, w);
                            }
                        }
                    }
                }
            }
            if (tma) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bfull[ew]);
            }
            if constexpr (!F8) release();
        }
    }

    __syncthreads();
    if (cta_split > 1) {
        // The cluster's CTAs add their shares of the tile in order of K, each for its part of the
        // outputs, from one another's shared memory.
        cluster_sync_all();
        if (unit < tiles) {
            const Tile tl = tile_at(unit);
            const int rows = min(128, tl.row_end - tl.row0);
            const int quads = (glu ? BN / 2 : BN) / 4;
            for (int i = (int)rank * C::THREADS + threadIdx.x; i < rows * quads; i += cta * C::THREADS) {
                const int r = i / quads, q = i - r * quads;
                const int64_t col = (int64_t)tl.ocol + 4 * q;
                if (col >= a.ycols) continue;
                auto sum = [&](int quad, float (&v)[4]) {
                    const float4 *src = reinterpret_cast<const float4 *>(smem) + r * (BN / 4) + (quad ^ (r & 7));
                    v[0] = v[1] = v[2] = v[3] = 0.0f;
                    for (int p = 0; p < cta; ++p) {
                        const float4 f = ld_shared_cluster_f4(mapa_shared(src, p));
                        v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
                    }
                };
                float v[4];
                sum(q, v);
                if (glu) {
                    float u[4];
                    sum(BN / 8 + q, u);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] *= silu_fast(u[j]);
                } else {
                    float b[4];
                    bias_quad(a, tl.e, col, b);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] += b[j];
                }
                store_quad(a, (int64_t)tl.row0 + r, col, v);
            }
        }
        cluster_sync_all();
    }
    if constexpr (PAIR) cluster_sync_all();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if constexpr (PAIR)
            tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
        else
            tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    if constexpr (PAIR) cluster_sync_all();
}

// Few rows per group (serving: some tokens over many experts, each W read for a row or two): the
// operands change places. W's rows are the MMA's 128 rows and 32 rows of x its columns, so that a block
// of K costs the epilogue 8 or 32 sums a thread instead of 64, and a thread owns one output column.
// CTAs take tiles of 128 rows of W (four units of 32, one per epilogue warp; gated pairs: 16 rows of g
// and the 16 of u) by 32 rows of x in turn. Tiles of fewer units, to share the last round evenly, were
// slower: what an SM receives is its share of the bytes under way, and 200 KB a CTA keep HBM busy through
// a round that not all SMs have. Loads start before the block has met.
// Bound by W's bytes and the start. 32 rows over 24 of 32 groups, N 2048, K 1024: E4M3 12.8 us for 51 MB
// (4.0 TB/s; the first load is issued after 2.2 us, the last has landed after 11 to 12.3), BF16 21.2 us
// for 101 MB (4.8 TB/s); 128-wide tiles take 18.9 and 23.1.
//   warp 0  offsets, TMA producer        warp 1  tensor memory, MMA issue
//   warp 3  E4M3: scales                 warps 4..7  epilogue, one unit each
template <int KIND>
struct FewCfg {
    static constexpr bool F8 = KIND == E_U8;
    static constexpr int ROWS = 32, THREADS = 256, STAGES = 10;
    static constexpr int W_BYTES = 128 * 128, X_BYTES = ROWS * 128, UNIT_BYTES = 32 * 128;
    static constexpr int NBUF = 2;  // accumulators: one per tile, or (E4M3) one per quad of blocks of K, four parts
    static constexpr int ACC_COLS = F8 ? kScaleQuad * ROWS : ROWS;
    static constexpr int TMEM_COLS = NBUF * ACC_COLS;
    static constexpr int SLOTS = 8, SLOT_BYTES = kScaleQuad * (ROWS + 8) * 4;  // xs[block][row], then ws[unit][2][block]
    static constexpr int SCALE_OFF = STAGES * (W_BYTES + X_BYTES);
    static constexpr int BAR_OFF = SCALE_OFF + (F8 ? SLOTS * SLOT_BYTES : 0);
    static constexpr int GROUP_OFF = BAR_OFF + 512;
    static int smem(int64_t groups) { return 1024 + GROUP_OFF + 8 * (int)(groups + 1); }
    static_assert((2 * STAGES + 2 * NBUF + 2 * SLOTS + 2) * 8 <= 512, "barriers");
};

template <int KIND>
__global__ void __launch_bounds__((FewCfg<KIND>::THREADS), 1)
    linear_few_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                           const __grid_constant__ CUtensorMap tmW4, BlkArgs a) {
    using C = FewCfg<KIND>;
    constexpr bool F8 = C::F8;
    constexpr int STAGES = C::STAGES, NBUF = C::NBUF, SLOTS = C::SLOTS;
    constexpr int BK = F8 ? 128 : 64;
    constexpr uint32_t IDESC = idesc_f32acc(KIND == E_BF16 ? 1u : 0u, 128, C::ROWS);

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sW = smem;
    uint8_t *sX = smem + STAGES * C::W_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);
    uint64_t *empty = full + STAGES;
    uint64_t *pfull = empty + STAGES;
    uint64_t *pempty = pfull + NBUF;
    uint64_t *sfull = pempty + NBUF;
    uint64_t *sempty = sfull + SLOTS;
    uint64_t *drain = sempty + SLOTS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *g_row = reinterpret_cast<int *>(smem + C::GROUP_OFF);
    int *g_tile = g_row + a.groups + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool glu = a.act == ACT_GLU;

    struct Tile {
        int e, row0, rows;  // group, first row of x, rows (at most 32)
        int n0, cnt;        // first unit of W, units (at most 4)
    };
    auto tile_at = [&](int t) {
        Tile r;
        int nt;
        const int mt = split_tile(a, t, nt);
        r.n0 = nt * 4;
        r.cnt = min(4, (int)((a.N + 31) >> 5) - r.n0);
        r.e = group_of(g_tile, a.groups, mt);
        r.row0 = g_row[r.e] + (mt - g_tile[r.e]) * C::ROWS;
        r.rows = min(C::ROWS, g_row[r.e + 1] - r.row0);
        return r;
    };
    auto tiles = [&]() { return g_tile[a.groups] * a.n_tiles; };  // the host has checked that this fits
    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        return mbar_wait_warp(bar, parity, abort_flag, a.err, site);
    };

    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmX);
            tma_prefetch_desc(glu ? &tmW : &tmW4);
            *abort_flag = 0;
        }
        for (uint64_t *b = full + lane; b <= drain; b += 32)
            mbar_init(b, (b >= pempty && b < sfull) || (b >= sempty && b < drain) ? 4 : b >= sfull && b < sempty ? 32 : 1);
        fence_barrier_init();
        dep_wait();
        const int first = a.offsets ? *a.offsets : 0;
        const int o = a.offsets && lane < a.groups ? a.offsets[lane + 1] : 0;
        scan_groups<C::ROWS>(a, lane, first, o, g_row, g_tile);
        __syncwarp();
        // The first use of each stage waits for nothing and comes before the block has met.
        const bool el = elect_one();
        int s = 0, i = 0;
        uint32_t ph = 0, issued = 0, issued_ph = 0;
        bool ok = true, met = false;
        for (int t = (int)blockIdx.x; t < tiles() && ok; t += (int)gridDim.x) {
            const Tile tl = tile_at(t);
            for (int kb = 0; kb < a.num_k; ++kb) {
                if (i == STAGES && !met) {
                    __syncthreads();
                    met = true;
                }
                if (met) {
                    ok = wait(&empty[s], ph ^ 1u, ERR_SITE_BLOCKS_PRODUCER);
                    if (!ok) break;
                }
                const int32_t kc = kb * BK;
                if (el) {
                    mbar_arrive_expect_tx(&full[s], tl.cnt * C::UNIT_BYTES + C::X_BYTES);
                    if (tl.cnt == 4 && !glu)  // whole tiles in one copy
                        tma_load_5d(sW + s * C::W_BYTES, &tmW4, &full[s], kc, tl.n0 * 32, 0, 0, tl.e);
                    for (int n = tl.cnt == 4 && !glu ? 4 : 0; n < tl.cnt; ++n) {
                        const int first = (tl.n0 + n) * (glu ? 16 : 32);
                        tma_load_5d(sW + s * C::W_BYTES + n * C::UNIT_BYTES, &tmW, &full[s], kc, glu ? first & 127 : first, 0,
                                    glu ? first >> 7 : 0, tl.e);
                    }
                    tma_load_2d(sX + s * C::X_BYTES, &tmX, &full[s], kc, tl.row0);
                }
                __syncwarp();
                issued |= 1u << s;
                issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
                i += !met;
                if (++s == STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        if (!met) __syncthreads();
        if (!ok) {
            // Loads in flight land before the CTA can exit (bounded).
            const unsigned long long t0 = globaltimer_ns();
            for (int k = 0; k < STAGES; ++k) {
                if (!((issued >> k) & 1u)) continue;
                while (!mbar_try_wait(&full[k], (issued_ph >> k) & 1u) && globaltimer_ns() - t0 < 100000000ull) {
                }
            }
        }
    } else {
        if (warp == 1) {
            tmem_alloc(tmem_slot, C::TMEM_COLS);
            tmem_relinquish();
            tc_fence_before();
        }
        dep_wait();
        __syncthreads();
        tc_fence_after();
    }
    dep_release();  // (not before this CTA holds its tensor memory)
    const uint32_t tmem_base = warp == 0 ? 0u : *tmem_slot;

    if (warp == 1) {
        const bool el = elect_one();
        int s = 0, buf = 0;
        uint32_t ph = 0, bph = 0;
        bool ok = true;
        const uint64_t wd0 = sdesc_k128(sW), xd0 = sdesc_k128(sX);
        for (int t = (int)blockIdx.x; t < tiles() && ok; t += (int)gridDim.x) {
            for (int kb = 0; kb < a.num_k; ++kb) {
                ok = wait(&full[s], ph, ERR_SITE_BLOCKS_MMA_FULL);
                if (ok && (F8 ? kb % kScaleQuad : kb) == 0) ok = wait(&pempty[buf], bph ^ 1u, ERR_SITE_BLOCKS_MMA_EMPTY);
                if (!ok) break;
                tc_fence_after();
                const bool last = kb == a.num_k - 1 || (F8 && kb % kScaleQuad == kScaleQuad - 1);
                if (el) {
                    const uint64_t wd = wd0 + (uint64_t)(s * (C::W_BYTES >> 4)), xd = xd0 + (uint64_t)(s * (C::X_BYTES >> 4));
                    const uint32_t d = tmem_base + (uint32_t)(buf * C::ACC_COLS + (F8 ? kb % kScaleQuad * C::ROWS : 0));
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if constexpr (F8)
                            mma_f8kind(d, wd + 2 * kk, xd + 2 * kk, IDESC, kk != 0);
                        else
                            mma_f16kind(d, wd + 2 * kk, xd + 2 * kk, IDESC, (kb | kk) != 0);
                    }
                    if (last) mma_commit(&pfull[buf]);
                    mma_commit(&empty[s]);
                }
                __syncwarp();
                if (last && ++buf == NBUF) {
                    buf = 0;
                    bph ^= 1u;
                }
                if (++s == STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        // All MMAs issued by this warp have completed once `drain` fires (also on the abort path).
        if (el) {
            mma_commit(drain);
            const unsigned long long t0 = globaltimer_ns();
            while (!mbar_try_wait(drain, 0)) {
                if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
                    if (a.err) atomicCAS(a.err, 0, ERR_SITE_BLOCKS_DRAIN);
                    break;
                }
            }
        }
        __syncwarp();
    } else if (F8 && warp == 3) {
        int slot = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = (int)blockIdx.x; t < tiles() && ok; t += (int)gridDim.x) {
            const Tile tl = tile_at(t);
            const float *xs = a.xs + (int64_t)(tl.row0 + min(lane, tl.rows - 1)) * a.ld_xs;  // the last row's again past the end
            // lane = (unit, half of a gated unit, block of K)
            const int first = (tl.n0 + (lane >> 3)) * (glu ? 16 : 32);
            const int nb = glu ? (first >> 7) * 2 + ((lane >> 2) & 1) : first >> 7;
            const float *ws = a.ws + tl.e * a.ws_group + (int64_t)min(nb, a.ws_blocks - 1) * a.ld_ws;
            for (int kb = 0; kb < a.num_k; kb += kScaleQuad) {
                ok = wait(&sempty[slot], ph ^ 1u, ERR_SITE_BLOCKS_PRODUCER);
                if (!ok) break;
                uint8_t *d = smem + C::SCALE_OFF + slot * C::SLOT_BYTES;
                const int n = min(kScaleQuad, a.num_k - kb);  // past the last block its scales again
#pragma unroll
                for (int j = 0; j < kScaleQuad; ++j) cp_async_4(d + (j * C::ROWS + lane) * 4, xs + kb + min(j, n - 1));
                cp_async_4(d + kScaleQuad * C::ROWS * 4 + lane * 4, ws + kb + min(lane & 3, n - 1));
                cp_async_arrive(&sfull[slot]);
                if (++slot == SLOTS) {
                    slot = 0;
                    ph ^= 1u;
                }
            }
        }
        cp_async_wait_all();
    } else if (warp >= 4) {
        const int unit = warp & 3;  // of the tile; tensor-memory lanes [32 unit, 32 unit + 32)
        int buf = 0, slot = 0;
        uint32_t bph = 0, sph = 0;
        bool ok = true;
        auto release = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pempty[buf]);
            if (++buf == NBUF) {
                buf = 0;
                bph ^= 1u;
            }
        };
        const uint32_t scales = smem_u32(smem) + C::SCALE_OFF;
        for (int t = (int)blockIdx.x; t < tiles() && ok; t += (int)gridDim.x) {
            const Tile tl = tile_at(t);
            const bool mine = unit < tl.cnt;
            const int col = glu ? (tl.n0 + unit) * 16 + (lane & 15) : (tl.n0 + unit) * 32 + lane;
            const bool out = mine && col < a.ycols && (!glu || lane < 16);
            const float bias = out && a.bias ? a.bias[tl.e * a.N + col] : 0.0f;
            float v[32];
            auto tbase = [&]() { return tmem_base + ((uint32_t)(unit * 32) << 16) + (uint32_t)(buf * C::ACC_COLS); };
            if constexpr (F8) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0.0f;
                for (int kb = 0; kb < a.num_k && ok; kb += kScaleQuad) {
                    ok = wait(&sfull[slot], sph, ERR_SITE_BLOCKS_EPILOGUE) && wait(&pfull[buf], bph, ERR_SITE_BLOCKS_EPILOGUE);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sc = scales + slot * C::SLOT_BYTES;
                    const int n = min(kScaleQuad, a.num_k - kb);
                    // Four blocks of K a hand-over: one at a time, its waits and loads took 420 cycles each.
                    auto add = [&](auto count) {
                        constexpr int R = decltype(count)::value;
                        float p[kScaleQuad][R], w[4];
#pragma unroll
                        for (int j = 0; j < kScaleQuad; ++j) {
                            if constexpr (R == 32)
                                tmem_ld32f(tbase() + j * C::ROWS, p[j]);
                            else
                                tmem_ld8f(tbase() + j * C::ROWS, p[j]);
                        }
                        ld_shared_v4(sc + kScaleQuad * C::ROWS * 4 + (unit * 2 + (lane >> 4)) * 16, w);
                        tmem_wait_ld();
                        release();
#pragma unroll
                        for (int j = 0; j < kScaleQuad; ++j) {
                            if (j >= n) break;
#pragma unroll
                            for (int q = 0; q < R / 4; ++q) {
                                float x[4];
                                ld_shared_v4(sc + (j * C::ROWS + 4 * q) * 4, x);
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[4 * q + i] = fmaf(p[j][4 * q + i], w[j] * x[i], v[4 * q + i]);
                            }
                        }
                    };
                    // Whether the scale of one of them is wide: lane (j, q) looks at rows 4 q .. 4 q + 3 in block j.
                    auto any_wide = [&]() {
                        float x[4];
                        ld_shared_v4(sc + lane * 16, x);
                        const uint32_t at = sc + kScaleQuad * C::ROWS * 4 + unit * 32 + (lane >> 3) * 4;
                        const float w0 = ld_shared_f32(at), w1 = ld_shared_f32(at + 16);
                        float least = fabsf(x[0]), most = least;
#pragma unroll
                        for (int i = 1; i < 4; ++i) least = fminf(least, fabsf(x[i])), most = fmaxf(most, fabsf(x[i]));
                        least *= fminf(fabsf(w0), fabsf(w1));
                        most *= fmaxf(fabsf(w0), fabsf(w1));
                        if (__builtin_expect(__all_sync(0xffffffffu, ordinary_scales(least, most)), 1)) return false;
                        bool wide = false;
#pragma unroll
                        for (int i = 0; i < 4; ++i) wide = wide || wide_scale(x[i], w0) || wide_scale(x[i], w1);
                        return __any_sync(0xffffffffu, wide) != 0;
                    };
                    // Then, a block at a time, in 64 bits.
                    auto add_wide = [&]() {
#pragma unroll 1
                        for (int j = 0; j < n; ++j) {
                            float p[32];
                            tmem_ld32f(tbase() + j * C::ROWS, p);
                            const double w = ld_shared_f32(sc + kScaleQuad * C::ROWS * 4 + (unit * 2 + (lane >> 4)) * 16 + 4 * j);
                            tmem_wait_ld();
                            if (j == n - 1) release();
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                float x[4];
                                ld_shared_v4(sc + (j * C::ROWS + 4 * q) * 4, x);
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[4 * q + i] += (float)((double)p[4 * q + i] * (w * (double)x[i]));
                            }
                        }
                    };
                    if (!mine)
                        release();
                    else if (__builtin_expect(any_wide(), 0))
                        add_wide();
                    else if (tl.rows <= 8)
                        add(std::integral_constant<int, 8>{});
                    else
                        add(std::integral_constant<int, 32>{});
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sempty[slot]);
                    if (++slot == SLOTS) {
                        slot = 0;
                        sph ^= 1u;
                    }
                }
                if (!ok) break;
            } else {
                ok = wait(&pfull[buf], bph, ERR_SITE_BLOCKS_EPILOGUE);
                if (!ok) break;
                tc_fence_after();
                tmem_ld32f(tbase(), v);
                tmem_wait_ld();
                release();
            }
            if (!mine) continue;
            if (glu) {
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    if (r >= tl.rows) break;
                    v[r] *= silu_fast(__shfl_xor_sync(0xffffffffu, v[r], 16));
                }
            }
            auto store = [&](auto type) {
                using T = decltype(type);
                T *y = static_cast<T *>(a.y) + (int64_t)tl.row0 * a.ldy + col;
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    if (r >= tl.rows) break;
                    float f = v[r] + bias;
                    if (out) {
                        if constexpr (std::is_same<T, float>::value) {
                            if (a.accumulate) f += *y;
                        }
                        if (a.act == 1) f = fmaxf(f, 0.0f);
                        if constexpr (std::is_same<T, float>::value)
                            *y = f;
                        else if constexpr (std::is_same<T, __half>::value)
                            *y = __float2half_rn(f);
                        else
                            *y = __float2bfloat16_rn(f);
                    }
                    y += a.ldy;
                }
            };
            if (a.y_dtype == TSFM_DTYPE_F32)
                store(float{});
            else if (a.y_dtype == TSFM_DTYPE_F16)
                store(__half{});
            else
                store(__nv_bfloat16{});
        }
    }

    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

BlkArgs blk_args(const LinearBlocksCall &c, int n_tiles, int bk) {
    BlkArgs a = {};
    a.M = c.M;
    a.N = c.N;
    a.K = c.K;
    a.offsets = c.offsets;
    a.groups = (int)c.groups;
    a.n_tiles = n_tiles;
    a.n_inv = 0xffffffffu / (uint32_t)n_tiles;
    a.num_k = (int)((c.K + bk - 1) / bk);
    a.xs = c.xs;
    a.ws = c.ws;
    a.ld_xs = c.ld_xs;
    a.ld_ws = c.ld_ws;
    a.ws_group = c.ws_group;
    a.ws_blocks = (int)((c.N + 127) / 128);
    a.bias = c.bias;
    a.y = c.y;
    a.ldy = c.ldy;
    a.ycols = c.act == ACT_GLU ? c.N / 2 : c.N;
    a.y_dtype = c.y_dtype;
    a.accumulate = c.accumulate;
    a.act = c.act;
    a.err = c.err;
    return a;
}

// x by boxes of `rows` rows.
Status x_map(const LinearBlocksCall &c, int kind, uint32_t bk, uint32_t rows, CUtensorMap *tx) {
    const int64_t dx[2] = {c.K, c.M}, sx[2] = {1, c.ldx};
    const uint32_t bx[2] = {bk, rows};
    return make_tmap_nd(tx, c.x, kind, 2, dx, sx, bx);
}

// W [groups, N, K] by boxes of w_rows rows; for gated pairs W is [groups, N / 256, 2, 128, K] and a box holds
// w_rows rows of each of w_halves of them.
Status w_map(const LinearBlocksCall &c, int kind, uint32_t bk, uint32_t w_rows, uint32_t w_halves, CUtensorMap *tw) {
    const bool glu = c.act == ACT_GLU;
    const int64_t wg = c.groups > 1 ? c.w_group : c.N * c.ldw;
    const int64_t dw[5] = {c.K, glu ? 128 : c.N, glu ? 2 : 1, glu ? c.N / 256 : 1, c.groups};
    const int64_t sw[5] = {1, c.ldw, glu ? 128 * c.ldw : c.N * c.ldw, glu ? 256 * c.ldw : c.N * c.ldw, wg};
    const uint32_t bw[5] = {bk, w_rows, w_halves, 1, 1};
    return make_tmap_nd(tw, c.w, kind, 5, dw, sw, bw);
}

// At most this many tiles of `rows` rows: every group may end inside one.
int64_t most_row_tiles(const LinearBlocksCall &c, int rows) {
    return c.offsets ? c.M / rows + std::min(c.groups, c.M) : (c.M + rows - 1) / rows;
}

template <int KIND>
Status launch_few(const LinearBlocksCall &c, cudaStream_t stream) {
    using C = FewCfg<KIND>;
    constexpr int BK = C::F8 ? 128 : 64;
    alignas(64) CUtensorMap tx, tw, tw4;
    const bool glu = c.act == ACT_GLU;
    TSFM_TRY(x_map(c, KIND, BK, C::ROWS, &tx));
    // W by units (gated pairs, and the tiles of fewer than four) and by whole tiles: those of the two that
    // this N has.
    const int64_t units = (c.N + 31) / 32;
    const bool by_unit = glu || units % 4 != 0, by_tile = !glu && units >= 4;
    if (by_unit) TSFM_TRY(w_map(c, KIND, BK, glu ? 16 : 32, glu ? 2 : 1, &tw));
    if (by_tile) TSFM_TRY(w_map(c, KIND, BK, 128, 1, &tw4));
    if (!by_unit) tw = tw4;
    if (!by_tile) tw4 = tw;
    const BlkArgs a = blk_args(c, (int)((c.N + 127) / 128), BK);
    const int smem = C::smem(c.groups);
    TSFM_TRY(ensure_smem_attr(reinterpret_cast<const void *>(&linear_few_rows_kernel<KIND>), smem));
    const int64_t most = most_row_tiles(c, C::ROWS) * a.n_tiles;
    if (most > INT32_MAX / 16) return Status::fail(TSFM_ERR_UNSUPPORTED, "linear: too many tiles");
    DepLaunch l((unsigned)std::min<int64_t>(most, num_sms()), C::THREADS, smem, stream);
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, linear_few_rows_kernel<KIND>, tx, tw, tw4, a);
    return e == cudaSuccess ? Status::ok() : Status::cuda(e, "linear (few rows): launch");
}

// split: CTAs that share a tile's K (64-wide E4M3 tiles; one tile per cluster, the grid covers every tile).
template <int KIND, int BN>
Status launch_blk(const LinearBlocksCall &c, int split, cudaStream_t stream) {
    using C = BlkCfg<KIND, BN>;
    constexpr bool PAIR = C::PAIR;
    constexpr int BK = C::F8 ? 128 : 64;
    alignas(64) CUtensorMap ta, tb, ty;
    const bool glu = c.act == ACT_GLU;
    TSFM_TRY(x_map(c, KIND, BK, C::A_BOX, &ta));
    TSFM_TRY(w_map(c, KIND, BK, PAIR || glu ? BN / 2 : BN, !PAIR && glu ? 2 : 1, &tb));
    BlkArgs a = blk_args(c, (int)((c.N + BN - 1) / BN), BK);
    const int ysz = c.y_dtype == TSFM_DTYPE_F32 ? 4 : 2;
    a.vec = reinterpret_cast<uintptr_t>(c.y) % (4 * ysz) == 0 && c.ldy % 4 == 0;
    a.vec32 = reinterpret_cast<uintptr_t>(c.y) % 32 == 0 && (c.ldy * ysz) % 32 == 0;
    // A TMA store clips a row to whole 16 bytes: with other numbers of columns it would write the padding.
    a.y_tma = C::TMA_Y && ysz == 2 && !c.accumulate && reinterpret_cast<uintptr_t>(c.y) % 16 == 0 && c.ldy % 8 == 0 &&
              a.ycols % 8 == 0;
    ty = ta;
    if (a.y_tma) {
        const int64_t d[2] = {a.ycols, c.M}, st[2] = {1, c.ldy};
        const uint32_t box[2] = {64, 32};
        TSFM_TRY(make_tmap_nd(&ty, c.y, c.y_dtype == TSFM_DTYPE_F16 ? E_F16 : E_BF16, 2, d, st, box));
    }
    a.split = split;
    const int smem = C::smem(c.groups);
    const void *fn = reinterpret_cast<const void *>(&linear_blocks_kernel<KIND, BN>);
    TSFM_TRY(ensure_smem_attr(fn, smem));
    const int64_t most = most_row_tiles(c, C::TILE_M) * a.n_tiles;
    if (most > INT32_MAX / 16) return Status::fail(TSFM_ERR_UNSUPPORTED, "linear: too many tiles");
    const int cta = PAIR ? 2 : split;
    DepLaunch l((unsigned)(split > 1 ? most * split : cta * std::min<int64_t>(most, num_sms() / cta)), C::THREADS, smem, stream,
                cta);
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, linear_blocks_kernel<KIND, BN>, ta, tb, ty, a);
    if (e != cudaSuccess) return Status::cuda(e, "linear (blocks): launch");
    return Status::ok();
}

// The tile width by the time that its waves of tiles take: a start, and per wave a part per stage of
// K and one per tile (units of 100 ns, fitted to M 256-4096, N 768-4096, K 768-4096; the fit need only
// rank the widths). Groups: each is taken to end in the middle of a tile. Measured, E4M3, us for widths
// 64 / 128 / 256:
//   M 512  N 2304 K 768   6.3 /  6.9 / 11.0      M 4096 N 2304 K 768   26.9 / 18.4 / 16.5
//   M 1024 N 2304 K 768   9.1 /  7.1 / 11.2      M 2048 N 4096 K 1024  26.7 / 20.6 / 18.2
//   M 2048 N 1024 K 4096 22.7 / 15.8 / 23.0      M 4096 N 1024 K 4096  40.2 / 27.5 / 24.3
// Outside the fit it loses up to 4 % (M 3000 N 2500 K 1024: 24.5 on 128 columns, 25.4 on the 256 taken), and
// lost 10 to 12 % on three of twenty sizes.
template <int KIND>
int tile_width(const LinearBlocksCall &c) {
    struct Cost {
        int bn, rows, units;
        double start, stage, tile;
    };
    const int sms = num_sms();
    const bool f8 = KIND == E_U8;
    const Cost costs[3] = {{64, 128, sms, 0, f8 ? 2.3 : 2.2, f8 ? 16.4 : 3.0},
                           {128, 128, sms, 0, f8 ? 3.3 : 2.8, f8 ? 18.7 : 3.0},
                           {256, 256, sms / 2, f8 ? 32.0 : 35.0, f8 ? 4.8 : 3.6, f8 ? 20.0 : 5.0}};
    const int64_t stages = (c.K + (f8 ? 127 : 63)) / (f8 ? 128 : 64);
    int best = 128;
    double least = 1e300;
    for (const Cost &k : costs) {
        const int64_t ends = c.offsets ? std::min(c.groups, c.M) : 1;
        const int64_t row_tiles = std::max(ends, c.M / k.rows + (c.offsets ? ends / 2 : c.M % k.rows != 0));
        const double tiles = (double)row_tiles * (double)((c.N + k.bn - 1) / k.bn);
        const double t = k.start + std::ceil(tiles / k.units) * (k.stage * (double)stages + k.tile);
        if (t < least) {
            least = t;
            best = k.bn;
        }
    }
    return best;
}

// Whether a call's groups are taken to have few rows. Measured, us on 64- or 128-wide tiles / with the
// operands exchanged:
//   E4M3, N 2048 K 1024, 32 groups:  M 32 18.9 / 12.8   M 192 19.0 / 14.8   M 256 (gated) 16.5 / 18.9
//     all rows in one group:         M 32  7.5 /  7.8   M 128  8.0 /  8.0
//     4 groups:                      M  4  7.2 /  6.4   M  32  7.3 /  7.2
//   BF16, the same, 32 groups:       M 32 23.1 / 21.2   M 192 23.4 / 21.9   M 256 (gated) 22.9 / 24.0
//     4 groups (fewer tiles than SMs, where nothing waits for memory): M 4 8.2 / 8.9
//   E4M3, one product (N 2304 K 768): M 1 5.8 / 4.8      M 8 5.8 / 5.1       M 16 5.8 / 5.9
//     N 2304, longer K:              K 1024 M 1 6.1 / 5.7   M 8 6.1 / 6.0    K 1280 M 1 6.7 / 6.6   M 8 6.6 / 6.9
//     K 4096, which a cluster's CTAs share on 64-wide tiles (N 1024): M 1 7.0 / 12.0
// The host does not know the groups' rows. Rows spread over three quarters of the groups, and all of them in one
// group, E4M3: 256 groups, M 1536, N 1024, K 512 50.0 / 30.8 and 11.3 / 17.1; 1024 groups, M 6144, N 512, K 512
// 108 / 68 and 29 / 38: the loss is smaller than the gain. BF16: 43.6 / 41.9 and 11.9 / 17.5, 92 / 92 and 29 / 38.
template <int KIND>
bool few_rows(const LinearBlocksCall &c) {
    const bool f8 = KIND == E_U8;
    if (!c.offsets) return f8 && c.M <= 8 && c.K <= 1024;
    return c.M <= 6 * c.groups && (f8 || std::min(c.groups, c.M) * ((c.N + 127) / 128) > num_sms());
}

template <int KIND>
Status launch_kind(const LinearBlocksCall &c, cudaStream_t stream) {
    if (few_rows<KIND>(c)) return launch_few<KIND>(c, stream);
    const int bn = tile_width<KIND>(c);
    if (bn == 256) return launch_blk<KIND, 256>(c, 1, stream);
    if (bn == 128) return launch_blk<KIND, 128>(c, 1, stream);
    // Few tiles and a long K (one group, 16 blocks of K or more): 2, 4 or 8 CTAs of a cluster share a
    // tile's K, as many as leave all clusters on the card at once (of 8 CTAs, 16 clusters took two
    // turns). us for 1 / 2 / 4 / 8 CTAs: M 32 N 1024 K 4096 12.1 / 8.9 / 7.1 / 12.3, M 32 N 512 K 8192
    // 20.3 / 12.8 / 8.8 / 7.2. At K 768 the exchange costs more than it saves (N 2304: 5.8 / 5.9).
    int split = 1;
    if (KIND == E_U8 && !c.offsets && c.K >= 2048) {
        const int64_t tiles = ((c.M + 127) / 128) * ((c.N + 63) / 64);
        while (split < 8 && tiles * split * 2 <= (split == 4 ? 64 : 128)) split *= 2;
    }
    return launch_blk<KIND, 64>(c, split, stream);
}

}  // namespace

Status launch_linear_blocks(const LinearBlocksCall &c, cudaStream_t stream) {
    switch (c.dtype) {
        case E_U8: return launch_kind<E_U8>(c, stream);
        case E_F16: return launch_kind<E_F16>(c, stream);
        case E_BF16: return launch_kind<E_BF16>(c, stream);
        default: return Status::fail(TSFM_ERR_UNSUPPORTED_DTYPE, "linear: operand type");
    }
}

}  // namespace tsfm
