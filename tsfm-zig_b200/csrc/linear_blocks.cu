// Products over block-scaled E4M3 operands, and products grouped by expert on 16-bit or E4M3
// operands: y[r] (+)= act(x[r] W[e]^T + bias[e]) for the rows r of group e.
//
// E4M3 operands carry one FP32 scale per 128 elements of a row of x and per 128 x 128 block of W:
//   y[m, n] = sum_b xs[m, b] ws[n / 128, b] (sum_{k in block b} xq[m, k] wq[n, k]).
// The inner sums run on the tensor cores (kind::f8f6f4, FP32 accumulators) one 128-wide block of K
// at a time; the scales differ from block to block, so each block's sums leave tensor memory and
// are added, scaled, into FP32 registers. 16-bit operands have no scales: their sums stay in tensor
// memory over the whole of K.
//
// One CTA per SM walks tiles of 128 rows x BN columns (or a CTA pair, 256 x BN):
//   warp 0     TMA producer: K-major tiles of x and W with the 128-byte swizzle into a ring of
//              STAGES, 128 bytes of K a stage. W's tile comes as two boxes of BN / 2 rows, so that
//              for gated pairs ([g | u] blocks of 256 rows) a tile holds g and u of the same columns.
//   warp 1     tensor-memory allocation, MMA issue (one thread) into NBUF accumulators: one
//              accumulator per block of K (E4M3) or per tile (16 bits).
//   warps 2..  epilogue: a thread owns a row and BN (or BN / 2, with 8 warps) of its columns.
// Rows of a group that end inside a tile: the tile's other rows hold whatever follows in x (or the
// stage's old bytes), are computed and not stored.
//
// Groups: the offsets are device memory, so the tile list is made on the device: warp 0 scans the
// groups' row counts into shared memory before the roles start (32 groups a step). Offsets are
// clamped to [0, M] and to be nondecreasing, so no content of theirs reaches outside x and y.
// Every element is summed over K by one CTA in a fixed order: no atomics, results do not depend on
// the grid.
#include "kernels.h"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace tsfm {

namespace {

constexpr int kMaxGroups = 1024;  // two words of shared memory each

// KIND: element type of x and W (E_F16, E_BF16, E_U8 = E4M3).
template <int KIND, int BN, bool PAIR>
struct BlkCfg {
    static constexpr bool F8 = KIND == E_U8;
    static constexpr int EPI_WARPS = BN >= 128 ? 8 : 4;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int TILE_M = PAIR ? 256 : 128;
    static constexpr int A_BOX = BN >= 128 ? 128 : 32;  // rows of x per TMA box
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;   // rows of W in this CTA's shared memory
    static constexpr int B_BYTES = B_ROWS * 128;
    static constexpr int STAGES = BN == 64 ? 8 : BN == 256 && !PAIR ? 3 : 5;
    static constexpr int NBUF = F8 ? (512 / BN > 8 ? 8 : 512 / BN) : 2;
    static constexpr int TMEM_COLS = NBUF * BN;
    static constexpr int EPI_OFF = STAGES * (A_BYTES + B_BYTES);
    static constexpr int BAR_OFF = EPI_OFF + EPI_WARPS * 4096;
    static constexpr int GROUP_OFF = BAR_OFF + 512;
    static int smem(int64_t groups) { return 1024 + GROUP_OFF + 8 * (int)(groups + 1); }
};

struct BlkArgs {
    int64_t M, N, K;
    const int32_t *offsets;
    int groups, n_tiles, num_k;
    const float *xs, *ws;
    int64_t ld_xs, ld_ws, ws_group;
    int ws_blocks;  // blocks of N
    const float *bias;
    void *y;
    int64_t ldy, ycols;
    int y_dtype, accumulate, act, vec;
    int *err;
};

template <int DT>
__device__ __forceinline__ uint32_t pack2_dt(float a, float b) {
    return pack16<DT == TSFM_DTYPE_F16>(a, b);
}

__device__ __forceinline__ float silu_fast(float u) { return __fdividef(u, 1.0f + __expf(-u)); }

// Stores (or adds) one 32-row x 32-column chunk of a warp: lane = row in, rows leave contiguous.
// `box` is the warp's 4 KB of shared memory; row0 the chunk's first row, rows its valid rows.
__device__ __forceinline__ void store_chunk32(const BlkArgs &a, uint8_t *box, int lane, int64_t row0, int rows,
                                              int64_t col0, const float (&v)[32]) {
    const bool f32 = a.y_dtype == TSFM_DTYPE_F32;
    const int64_t left = a.ycols - col0;
    if (left <= 0 || rows <= 0) return;  // the same for the whole warp
    __syncwarp();
    if (f32) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4 *>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    } else {
        const bool h = a.y_dtype == TSFM_DTYPE_F16;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint4 p;
            p.x = h ? pack16<true>(v[8 * q], v[8 * q + 1]) : pack16<false>(v[8 * q], v[8 * q + 1]);
            p.y = h ? pack16<true>(v[8 * q + 2], v[8 * q + 3]) : pack16<false>(v[8 * q + 2], v[8 * q + 3]);
            p.z = h ? pack16<true>(v[8 * q + 4], v[8 * q + 5]) : pack16<false>(v[8 * q + 4], v[8 * q + 5]);
            p.w = h ? pack16<true>(v[8 * q + 6], v[8 * q + 7]) : pack16<false>(v[8 * q + 6], v[8 * q + 7]);
            *reinterpret_cast<uint4 *>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = p;
        }
    }
    __syncwarp();
    if (a.vec && left >= 32) {
        if (f32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 4 * i + (lane >> 3), q = lane & 7;
                if (r < rows) {
                    float4 t = *reinterpret_cast<const float4 *>(box + r * 128 + ((q ^ (r & 7)) << 4));
                    float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(a.y) + (row0 + r) * a.ldy + col0) + q;
                    if (a.accumulate) {
                        const float4 old = *o;
                        t.x += old.x, t.y += old.y, t.z += old.z, t.w += old.w;
                        if (a.act == 1) t = make_float4(fmaxf(t.x, 0.f), fmaxf(t.y, 0.f), fmaxf(t.z, 0.f), fmaxf(t.w, 0.f));
                    }
                    *o = t;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 8 * i + (lane >> 2), q = lane & 3;
                if (r < rows)
                    reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.y) + (row0 + r) * a.ldy + col0)[q] =
                        *reinterpret_cast<const uint4 *>(box + r * 128 + ((q ^ (r & 7)) << 4));
            }
        }
    } else if (lane < left) {
        // A column tail or an unaligned y: one element per lane.
        for (int r = 0; r < rows; ++r) {
            if (f32) {
                float t = *reinterpret_cast<const float *>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                float *o = static_cast<float *>(a.y) + (row0 + r) * a.ldy + col0 + lane;
                if (a.accumulate) {
                    t += *o;
                    if (a.act == 1) t = fmaxf(t, 0.0f);
                }
                *o = t;
            } else {
                static_cast<uint16_t *>(a.y)[(row0 + r) * a.ldy + col0 + lane] = *reinterpret_cast<const uint16_t *>(
                    box + r * 128 + (((lane >> 3) ^ (r & 7)) << 4) + (lane & 7) * 2);
            }
        }
    }
}

template <int KIND, int BN, bool PAIR>
__global__ void __launch_bounds__((BlkCfg<KIND, BN, PAIR>::THREADS), 1)
    linear_blocks_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, BlkArgs a) {
    using C = BlkCfg<KIND, BN, PAIR>;
    constexpr bool F8 = C::F8;
    constexpr int STAGES = C::STAGES, NBUF = C::NBUF;
    constexpr int BK = F8 ? 128 : 64;  // elements of K per stage
    constexpr uint32_t IDESC = idesc_f32acc(KIND == E_BF16 ? 1u : 0u, C::TILE_M, BN);
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    const int64_t unit = PAIR ? (int64_t)(blockIdx.x >> 1) : (int64_t)blockIdx.x;
    const int64_t units = PAIR ? (int64_t)(gridDim.x >> 1) : (int64_t)gridDim.x;

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem;
    uint8_t *sB = smem + STAGES * C::A_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);
    uint64_t *empty = full + STAGES;
    uint64_t *pfull = empty + STAGES;
    uint64_t *pempty = pfull + NBUF;
    uint64_t *drain = pempty + NBUF;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *g_row = reinterpret_cast<int *>(smem + C::GROUP_OFF);  // group e has rows [g_row[e], g_row[e + 1])
    int *g_tile = g_row + a.groups + 1;                         // and row tiles [g_tile[e], g_tile[e + 1])

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 32) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < NBUF; ++i) {
            mbar_init(&pfull[i], 1);
            mbar_init(&pempty[i], (PAIR ? 2 : 1) * C::EPI_WARPS);  // one arrival per epilogue warp
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 0) {
        const int M = (int)a.M;
        int end = a.offsets ? min(max(a.offsets[0], 0), M) : 0;  // running maximum of the offsets
        int tiles = 0;
        if (lane == 0) {
            g_row[0] = end;
            g_tile[0] = 0;
        }
        for (int base = 0; base < a.groups; base += 32) {
            const int e = base + lane;
            int o = e < a.groups ? (a.offsets ? min(max(a.offsets[e + 1], 0), M) : M) : 0;
            o = max(o, end);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int p = __shfl_up_sync(0xffffffffu, o, d);
                if (lane >= d) o = max(o, p);
            }
            int start = __shfl_up_sync(0xffffffffu, o, 1);
            if (lane == 0) start = end;
            int t = (o - start + C::TILE_M - 1) / C::TILE_M;
#pragma unroll
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
        }
    }
    if (warp == 1) {
        __syncwarp();
        if constexpr (PAIR) {
            tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, C::TMEM_COLS);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    struct Tile {
        int e, row0, row_end;  // group, first row of this CTA's 128 rows, end of the group
        int b0, b1;            // first W row of the tile's two boxes
        int ocol0, ocol1;      // the boxes' output columns
    };
    const int64_t tiles = (int64_t)g_tile[a.groups] * a.n_tiles;
    auto tile_at = [&](int64_t t) {
        Tile r;
        const int mt = (int)(t / a.n_tiles), nt = (int)(t - (int64_t)mt * a.n_tiles);
        int lo = 0, hi = a.groups - 1;  // the last e with g_tile[e] <= mt
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (g_tile[mid] <= mt)
                lo = mid;
            else
                hi = mid - 1;
        }
        r.e = lo;
        r.row0 = g_row[lo] + (mt - g_tile[lo]) * C::TILE_M + (int)rank * 128;
        r.row_end = g_row[lo + 1];
        if (a.act == ACT_GLU) {
            const int c = nt * (BN / 2);
            r.b0 = (c >> 7) * 256 + (c & 127);
            r.b1 = r.b0 + 128;
            r.ocol0 = r.ocol1 = c;
        } else {
            r.ocol0 = r.b0 = nt * BN;
            r.ocol1 = r.b1 = r.b0 + BN / 2;
        }
        return r;
    };
    auto slabs = [&](int row0, int row_end) {  // boxes of x that hold rows of the tile
        return min(128 / C::A_BOX, max(0, (row_end - row0 + C::A_BOX - 1) / C::A_BOX));
    };

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0, issued = 0, issued_ph = 0;
            bool ok = true;
            for (int64_t t = unit; t < tiles && ok; t += units) {
                const Tile tl = tile_at(t);
                const int na = PAIR ? 1 : slabs(tl.row0, tl.row_end);
                for (int kb = 0; kb < a.num_k; ++kb) {
                    ok = PAIR ? mbar_wait_cl(&empty[s], ph ^ 1u, abort_flag, a.err, ERR_SITE_BLOCKS_PRODUCER)
                              : mbar_wait(&empty[s], ph ^ 1u, abort_flag, a.err, ERR_SITE_BLOCKS_PRODUCER);
                    if (!ok) break;
                    const int32_t kc = kb * BK;
                    if constexpr (PAIR) {
                        // Each CTA loads its 128 rows of x and one of W's two boxes.
                        if (leader) mbar_arrive_expect_tx(&full[s], 2 * (C::A_BYTES + C::B_BYTES));
                        const uint32_t fb = mapa_shared(&full[s], 0);
                        tma_load_2d_pair(sA + s * C::A_BYTES, &tmA, fb, kc, tl.row0);
                        tma_load_3d_pair(sB + s * C::B_BYTES, &tmB, fb, kc, leader ? tl.b0 : tl.b1, tl.e);
                    } else {
                        mbar_arrive_expect_tx(&full[s], na * C::A_BOX * 128 + C::B_BYTES);
                        for (int i = 0; i < na; ++i)
                            tma_load_2d(sA + s * C::A_BYTES + i * C::A_BOX * 128, &tmA, &full[s], kc, tl.row0 + i * C::A_BOX);
                        tma_load_3d(sB + s * C::B_BYTES, &tmB, &full[s], kc, tl.b0, tl.e);
                        tma_load_3d(sB + s * C::B_BYTES + C::B_BYTES / 2, &tmB, &full[s], kc, tl.b1, tl.e);
                    }
                    issued |= 1u << s;
                    issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
                    if (++s == STAGES) {
                        s = 0;
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
                        while (!mbar_try_wait_cl(&full[i], (issued_ph >> i) & 1u) && globaltimer_ns() - t0 < 100000000ull) {
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            int s = 0, buf = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
                return PAIR ? mbar_wait_cl(bar, parity, abort_flag, a.err, site) : mbar_wait(bar, parity, abort_flag, a.err, site);
            };
            auto commit = [&](uint64_t *bar) {
                if constexpr (PAIR) {
                    mma_commit_pair(mapa_shared(bar, 0));
                    mma_commit_pair(mapa_shared(bar, 1));
                } else {
                    mma_commit(bar);
                }
            };
            for (int64_t t = unit; t < tiles && ok; t += units) {
                for (int kb = 0; kb < a.num_k; ++kb) {
                    if (F8 || kb == 0) {
                        ok = wait(&pempty[buf], bph ^ 1u, ERR_SITE_BLOCKS_MMA_EMPTY);
                        if (!ok) break;
                    }
                    ok = wait(&full[s], ph, ERR_SITE_BLOCKS_MMA_FULL);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem_base + (uint32_t)(buf * BN);
                    const uint64_t ad = sdesc_k128(sA + s * C::A_BYTES), bd = sdesc_k128(sB + s * C::B_BYTES);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint32_t accum = F8 ? kk != 0 : (kb | kk) != 0;
                        if constexpr (F8) {
                            if constexpr (PAIR)
                                mma_f8kind_pair(d, ad + 2 * kk, bd + 2 * kk, IDESC, accum);
                            else
                                mma_f8kind(d, ad + 2 * kk, bd + 2 * kk, IDESC, accum);
                        } else if constexpr (PAIR) {
                            mma_f16kind_pair(d, ad + 2 * kk, bd + 2 * kk, IDESC, accum);
                        } else {
                            mma_f16kind(d, ad + 2 * kk, bd + 2 * kk, IDESC, accum);
                        }
                    }
                    commit(&empty[s]);
                    if (F8 || kb == a.num_k - 1) {
                        commit(&pfull[buf]);
                        if (++buf == NBUF) {
                            buf = 0;
                            bph ^= 1u;
                        }
                    }
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
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
    } else {
        constexpr int PARTS = C::EPI_WARPS / 4;         // warps that share a row's columns
        constexpr int CPH = BN / 2 / PARTS / 32;        // 32-column chunks per thread of each box
        const int ew = warp - 2;
        const int eg = warp & 3, part = ew >> 2;        // tensor-memory lanes [32 eg, 32 eg + 32)
        uint8_t *box = smem + C::EPI_OFF + ew * 4096;
        int buf = 0;
        uint32_t bph = 0;
        bool ok = true;
        auto wait = [&]() {
            const bool got = PAIR ? mbar_wait_cl(&pfull[buf], bph, abort_flag, a.err, ERR_SITE_BLOCKS_EPILOGUE)
                                  : mbar_wait(&pfull[buf], bph, abort_flag, a.err, ERR_SITE_BLOCKS_EPILOGUE);
            return __all_sync(0xffffffffu, got) != 0;
        };
        auto release = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR)
                    mbar_arrive_cluster(mapa_shared(&pempty[buf], 0));
                else
                    mbar_arrive(&pempty[buf]);
            }
            if (++buf == NBUF) {
                buf = 0;
                bph ^= 1u;
            }
        };
        for (int64_t t = unit; t < tiles && ok; t += units) {
            const Tile tl = tile_at(t);
            const int wrow0 = tl.row0 + eg * 32;
            const int wrows = min(32, tl.row_end - wrow0);  // this warp's valid rows (may be <= 0)
            // Chunk c of this thread: columns [off(c), off(c) + 32) of the tile's accumulator; chunks
            // [0, CPH) belong to the first box, [CPH, 2 CPH) to the second.
            auto off = [&](int c) { return (c / CPH) * (BN / 2) + (part * CPH + c % CPH) * 32; };
            float acc[F8 ? 2 * CPH * 32 : 32];
            uint32_t tbase = 0;
            if constexpr (F8) {
#pragma unroll
                for (int i = 0; i < 2 * CPH * 32; ++i) acc[i] = 0.0f;
                const float *xs = a.xs + (int64_t)min(wrow0 + lane, tl.row_end - 1) * a.ld_xs;
                const float *ws0 = a.ws + tl.e * a.ws_group + (int64_t)min(tl.b0 >> 7, a.ws_blocks - 1) * a.ld_ws;
                const float *ws1 = a.ws + tl.e * a.ws_group + (int64_t)min(tl.b1 >> 7, a.ws_blocks - 1) * a.ld_ws;
                float sx = __ldg(xs), w0 = __ldg(ws0), w1 = __ldg(ws1);
                for (int kb = 0; kb < a.num_k; ++kb) {
                    const float s0 = sx * w0, s1 = sx * w1;
                    if (kb + 1 < a.num_k) {
                        sx = __ldg(xs + kb + 1);
                        w0 = __ldg(ws0 + kb + 1);
                        w1 = __ldg(ws1 + kb + 1);
                    }
                    ok = wait();
                    if (!ok) break;
                    tc_fence_after();
                    if (wrows > 0) {
                        tbase = tmem_base + ((uint32_t)(eg * 32) << 16) + (uint32_t)(buf * BN);
#pragma unroll
                        for (int c = 0; c < 2 * CPH; ++c) {
                            float p[32];
                            tmem_ld32(tbase + off(c), p);
                            tmem_wait_ld();
                            const float sc = c < CPH ? s0 : s1;
#pragma unroll
                            for (int j = 0; j < 32; ++j) acc[c * 32 + j] = fmaf(p[j], sc, acc[c * 32 + j]);
                        }
                    }
                    release();
                }
                if (!ok) break;
            } else {
                ok = wait();
                if (!ok) break;
                tc_fence_after();
                tbase = tmem_base + ((uint32_t)(eg * 32) << 16) + (uint32_t)(buf * BN);
            }
            auto chunk = [&](int c, float (&v)[32]) {
                if constexpr (F8) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = acc[c * 32 + j];
                } else {
                    tmem_ld32(tbase + off(c), v);
                    tmem_wait_ld();
                }
            };
            if (wrows > 0) {
                if (a.act == ACT_GLU) {
#pragma unroll
                    for (int c = 0; c < CPH; ++c) {
                        float g[32], u[32];
                        chunk(c, g);
                        chunk(CPH + c, u);
#pragma unroll
                        for (int j = 0; j < 32; ++j) g[j] *= silu_fast(u[j]);
                        store_chunk32(a, box, lane, wrow0, wrows, tl.ocol0 + off(c), g);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 2 * CPH; ++c) {
                        float v[32];
                        chunk(c, v);
                        const int64_t col0 = (int64_t)tl.b0 + off(c);
                        if (a.bias) {
                            const float *b = a.bias + tl.e * a.N + col0;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (col0 + j < a.N) v[j] += __ldg(b + j);
                        }
                        if (a.act == 1 && !a.accumulate) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = fmaxf(v[j], 0.0f);
                        }
                        store_chunk32(a, box, lane, wrow0, wrows, col0, v);
                    }
                }
            }
            if constexpr (!F8) release();
        }
    }

    __syncthreads();
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

template <int KIND, int BN, bool PAIR>
Status launch_blk(const LinearBlocksCall &c, cudaStream_t stream) {
    using C = BlkCfg<KIND, BN, PAIR>;
    constexpr int BK = C::F8 ? 128 : 64;
    alignas(64) CUtensorMap ta, tb;
    TSFM_TRY(make_tmap_3d(&ta, c.x, KIND, c.K, c.M, 0, c.ldx, 0, BK, C::A_BOX));
    TSFM_TRY(make_tmap_3d(&tb, c.w, KIND, c.K, c.N, c.groups, c.ldw, c.groups > 1 ? c.w_group : c.N * c.ldw, BK, BN / 2));
    BlkArgs a;
    a.M = c.M;
    a.N = c.N;
    a.K = c.K;
    a.offsets = c.offsets;
    a.groups = (int)c.groups;
    a.n_tiles = (int)((c.N + BN - 1) / BN);
    a.num_k = (int)((c.K + BK - 1) / BK);
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
    const int ysz = c.y_dtype == TSFM_DTYPE_F32 ? 4 : 2;
    a.vec = (reinterpret_cast<uintptr_t>(c.y) & 15) == 0 && (c.ldy * ysz) % 16 == 0;
    a.err = c.err;
    const int smem = C::smem(c.groups);
    const void *fn = reinterpret_cast<const void *>(&linear_blocks_kernel<KIND, BN, PAIR>);
    TSFM_TRY(ensure_smem_attr(fn, smem));
    // At most this many row tiles: every group may end inside one.
    const int64_t row_tiles = c.offsets ? c.M / C::TILE_M + std::min(c.groups, c.M) : (c.M + C::TILE_M - 1) / C::TILE_M;
    const int64_t most = row_tiles * a.n_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(PAIR ? 2 * std::min<int64_t>(most, num_sms() / 2) : std::min<int64_t>(most, num_sms())));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_blocks_kernel<KIND, BN, PAIR>, ta, tb, a);
    if (e != cudaSuccess) return Status::cuda(e, "linear (blocks): launch");
    return Status::ok();
}

template <int KIND>
Status launch_kind(const LinearBlocksCall &c, cudaStream_t stream) {
    return launch_blk<KIND, 128, false>(c, stream);
}

}  // namespace

Status launch_linear_blocks(const LinearBlocksCall &c, cudaStream_t stream) {
    if (c.groups > kMaxGroups) return Status::fail(TSFM_ERR_UNSUPPORTED, "linear: more than 1024 groups");
    switch (c.dtype) {
        case E_U8: return launch_kind<E_U8>(c, stream);
        case E_F16: return launch_kind<E_F16>(c, stream);
        case E_BF16: return launch_kind<E_BF16>(c, stream);
        default: return Status::fail(TSFM_ERR_UNSUPPORTED_DTYPE, "linear: operand type");
    }
}

}  // namespace tsfm
