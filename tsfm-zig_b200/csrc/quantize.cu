// Block-scaled E4M3 operands: q = e4m3(x / s) with one FP32 scale s per block of 1 x 128 (an
// activation's row) or 128 x 128 (a weight) elements.
//
// s is the smallest power of two with max|x| / s <= 448, so x / s is exact and the only rounding
// is E4M3's own (half a step, 2^-4 of a normal value): a floating format loses nothing to a scale
// that is a power of two, and the result does not depend on how a division rounds. With
// max|x| = m 2^e, 1 <= m < 2, and 448 = 1.75 * 2^8: s = 2^(e - 8) for m <= 1.75, else 2^(e - 7),
// at least 2^-126 (FP32's smallest normal, so that 1 / s is finite). The maximum is taken over the
// bit patterns of |x|: infinities and NaN order above every number, and a block that holds one gets
// s = NaN and q = NaN throughout, so that a product over it shows it.
//
// Every input is read once and every code written once.
#include "kernels.h"
#include "ptx.cuh"

#include <algorithm>
#include <climits>

namespace tsfm {

namespace {

struct BlockScale {
    float scale, inv;
};

// From the bits of the block's largest |x|.
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) {
        const float nan = __uint_as_float(0x7fc00000u);
        return {nan, nan};
    }
    int e = (int)(amax_bits >> 23);                               // biased; 0 for zero and subnormals
    e += (amax_bits & 0x7fffffu) > 0x600000u ? -7 : -8;           // mantissa of 1.75
    e = max(e, 1);
    return {__uint_as_float((uint32_t)e << 23), __uint_as_float((uint32_t)(254 - e) << 23)};
}

// Sixteen consecutive elements of a row as they are stored (a lane's share of a block's row: eight
// lanes of 16); elements at or past `n` read as zero.
template <int DT>
struct Raw16 {
    static constexpr int W = DT == E_F32X ? 4 : 2;
    uint4 w[W];
};

template <int DT>
__device__ __forceinline__ Raw16<DT> load16(const void *row, int col, int n, bool vec) {
    Raw16<DT> r;
    constexpr int W = Raw16<DT>::W;
    if (vec && n >= 16) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(row) + (int64_t)col * (DT == E_F32X ? 4 : 2));
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = __ldcs(p + i);
    } else {
        uint32_t w[4 * W];
#pragma unroll
        for (int j = 0; j < 4 * W; ++j) {
            if constexpr (DT == E_F32X) {
                w[j] = j < n ? static_cast<const uint32_t *>(row)[col + j] : 0u;
            } else {
                const uint16_t *p = static_cast<const uint16_t *>(row) + col;
                w[j] = (2 * j < n ? (uint32_t)p[2 * j] : 0u) | (2 * j + 1 < n ? (uint32_t)p[2 * j + 1] << 16 : 0u);
            }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    return r;
}

// The largest |x| of 16 elements as bits: two 16-bit maxima packed, or one of 32 bits. Reduced
// across lanes with amax_of, then turned into FP32 bits.
template <int DT>
__device__ __forceinline__ uint32_t amax_of(uint32_t a, uint32_t b, uint32_t c = 0u) {
    if constexpr (DT == E_F32X)
        return __vimax3_u32(a, b, c);
    else
        return __vimax3_u16x2(a, b, c);
}

template <int DT>
__device__ __forceinline__ uint32_t amax16(const Raw16<DT> &r) {
    constexpr uint32_t m = DT == E_F32X ? 0x7fffffffu : 0x7fff7fffu;
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < Raw16<DT>::W; ++i) {
        a = amax_of<DT>(a, r.w[i].x & m, r.w[i].y & m);
        a = amax_of<DT>(a, r.w[i].z & m, r.w[i].w & m);
    }
    return a;
}

template <int DT>
__device__ __forceinline__ uint32_t amax_bits(uint32_t m) {
    if constexpr (DT == E_F32X) return m;
    m = max(m & 0xffffu, m >> 16);
    if constexpr (DT == E_F16)
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    else
        return m << 16;
}

// Four of the elements, scaled and rounded, as one word of codes.
template <int DT>
__device__ __forceinline__ uint32_t codes4(const Raw16<DT> &r, int i, float inv) {
    float v[4];
    if constexpr (DT == E_F32X) {
        const uint4 w = r.w[i];
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    } else {
        const uint4 q = r.w[i >> 1];
        const uint32_t w[2] = {i & 1 ? q.z : q.x, i & 1 ? q.w : q.y};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if constexpr (DT == E_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                v[2 * j] = f.x, v[2 * j + 1] = f.y;
            } else {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
    return e4m3x2(v[0] * inv, v[1] * inv) | (e4m3x2(v[2] * inv, v[3] * inv) << 16);
}

template <int DT>
__device__ __forceinline__ void store16(uint8_t *p, int n, bool vec, const Raw16<DT> &r, float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = codes4<DT>(r, i, inv);
    if (vec && n >= 16) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < n) p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
}

// One row x 128 columns per eight lanes. Eight lanes take U blocks, 32 apart, whose loads are all
// under way before the first maximum; the CTA's 32 U blocks are consecutive. 36928 x 2048 BF16 takes
// 38.0 us, 6.03 TB/s of the 6.46 TB/s of a copy. Instructions bound it as much as memory: eight
// elements a lane with 64-bit indices and a division per block took 69 us, with packed maxima and one
// division a thread 51 us, sixteen elements a lane (half the reductions and scales) 38 us.
template <int DT, int U>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeCall c, int64_t blocks, uint32_t per_row, bool vx,
                                                            bool vq) {
    constexpr int esz = DT == E_F32X ? 4 : 2;
    dep_wait();
    dep_release();
    const int lane = threadIdx.x & 7, at = threadIdx.x >> 3;
    const int64_t first = (int64_t)blockIdx.x * (32 * U);
    const int64_t r0 = first / per_row;
    uint32_t kb = (uint32_t)(first - r0 * per_row) + at;
    int64_t row = r0 + kb / per_row;
    kb %= per_row;
    const uint32_t rows32 = 32 / per_row, kb32 = 32 % per_row;  // 32 blocks further on
    const int left = (int)min((int64_t)U, (blocks - first - at + 31) / 32);  // these lanes' blocks
    Raw16<DT> raw[U];
    int64_t rr[U];
    int col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        rr[u] = row;
        col[u] = (int)kb * 128 + lane * 16;
        raw[u] = load16<DT>(static_cast<const char *>(c.x) + row * c.ldx * esz, col[u], u < left ? (int)c.cols - col[u] : 0, vx);
        row += rows32;
        kb += kb32;
        if (kb >= per_row) {
            kb -= per_row;
            ++row;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        uint32_t m = amax16<DT>(raw[u]);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = amax_of<DT>(m, __shfl_xor_sync(0xffffffffu, m, o));
        const BlockScale s = block_scale(amax_bits<DT>(m));
        if (u < left) {
            if (lane == 0) c.scale[rr[u] * c.ld_scale + (col[u] >> 7)] = s.scale;
            store16<DT>(c.q + rr[u] * c.ldq + col[u], (int)c.cols - col[u], vq, raw[u], s.inv);
        }
    }
}

// One 128 x 128 block per CTA: 256 threads of 4 rows (32 apart) x 16 columns, held in registers
// between the maximum and the conversion.
template <int DT>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(QuantizeCall c, bool vx, bool vq) {
    __shared__ uint32_t warp_max[8];
    constexpr int esz = DT == E_F32X ? 4 : 2;
    dep_wait();
    dep_release();
    const int lane = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    const int col = (int)blockIdx.x * 128 + lane * 16, n = (int)c.cols - col;
    for (int64_t br = blockIdx.y; br * 128 < c.rows; br += gridDim.y) {
        Raw16<DT> raw[4];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = br * 128 + i * 32 + r0;
            raw[i] = load16<DT>(static_cast<const char *>(c.x) + r * c.ldx * esz, col, r < c.rows ? n : 0, vx);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) m = amax_of<DT>(m, amax16<DT>(raw[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = amax_of<DT>(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) m = amax_of<DT>(m, warp_max[i]);
        __syncthreads();
        const BlockScale s = block_scale(amax_bits<DT>(m));
        if (threadIdx.x == 0) c.scale[br * c.ld_scale + blockIdx.x] = s.scale;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = br * 128 + i * 32 + r0;
            if (r < c.rows) store16<DT>(c.q + r * c.ldq + col, n, vq, raw[i], s.inv);
        }
    }
}

template <int DT>
Status launch_dt(const QuantizeCall &c, cudaStream_t stream) {
    constexpr int esz = DT == E_F32X ? 4 : 2;
    const bool vx = (reinterpret_cast<uintptr_t>(c.x) & 15) == 0 && (c.ldx * esz) % 16 == 0;
    const bool vq = (reinterpret_cast<uintptr_t>(c.q) & 15) == 0 && c.ldq % 16 == 0;
    const int64_t per_row = (c.cols + 127) / 128;
    cudaError_t e;
    if (c.block_rows == 1) {
        const int64_t blocks = c.rows * per_row;
        constexpr int U = DT == E_F32X ? 1 : 2;  // 64 bytes a thread in flight
        const int64_t ctas = (blocks + 32 * U - 1) / (32 * U);
        if (ctas > INT32_MAX) return Status::fail(TSFM_ERR_UNSUPPORTED, "quantize: too many blocks");
        DepLaunch l((unsigned)ctas, 256, 0, stream);
        e = cudaLaunchKernelEx(&l.cfg, quantize_rows_kernel<DT, U>, c, blocks, (uint32_t)per_row, vx, vq);
    } else {
        const int64_t tiles = (c.rows + 127) / 128;
        const dim3 grid((unsigned)per_row, (unsigned)std::min<int64_t>(tiles, 65535));
        DepLaunch l(grid, 256, 0, stream);
        e = cudaLaunchKernelEx(&l.cfg, quantize_tiles_kernel<DT>, c, vx, vq);
    }
    return e == cudaSuccess ? Status::ok() : Status::cuda(e, "quantize: launch");
}

}  // namespace

Status launch_quantize_e4m3(const QuantizeCall &c, cudaStream_t stream) {
    if (c.rows == 0) return Status::ok();
    switch (c.x_dtype) {
        case E_F32X: return launch_dt<E_F32X>(c, stream);
        case E_F16: return launch_dt<E_F16>(c, stream);
        default: return launch_dt<E_BF16>(c, stream);
    }
}

}  // namespace tsfm
