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
// Bound by memory: every input is read once and every code written once.
#include "kernels.h"
#include "ptx.cuh"

#include <algorithm>

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

// Eight consecutive elements of a row as FP32; elements at or past `n` read as zero.
template <int DT>
__device__ __forceinline__ void load8(const void *row, int64_t col, int n, bool vec, float (&v)[8]) {
    if constexpr (DT == E_F32X) {
        const float *p = static_cast<const float *>(row) + col;
        if (vec && n >= 8) {
            const float4 a = __ldcs(reinterpret_cast<const float4 *>(p));
            const float4 b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.0f;
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(row) + col;
        uint32_t w[4];
        if (vec && n >= 8) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(p));
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = (2 * j < n ? (uint32_t)p[2 * j] : 0u) | (2 * j + 1 < n ? (uint32_t)p[2 * j + 1] << 16 : 0u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == E_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                v[2 * j] = f.x, v[2 * j + 1] = f.y;
            } else {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
}

__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}

__device__ __forceinline__ void store8(uint8_t *p, int n, bool vec, const float (&v)[8], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        w[h] = e4m3x2(v[4 * h] * inv, v[4 * h + 1] * inv) | (e4m3x2(v[4 * h + 2] * inv, v[4 * h + 3] * inv) << 16);
    if (vec && n >= 8) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
}

// One row x 128 columns per half warp: 16 lanes of 8 elements.
template <int DT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeCall c, int64_t blocks, int64_t per_row, bool vx,
                                                            bool vq) {
    const int lane = threadIdx.x & 15;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x / 16);
    for (int64_t b = (int64_t)blockIdx.x * (blockDim.x / 16) + (threadIdx.x >> 4); b < blocks; b += step) {
        const int64_t r = b / per_row, kb = b - r * per_row;
        const int64_t col = kb * 128 + lane * 8;
        const int n = (int)max((int64_t)0, min((int64_t)8, c.cols - col));
        constexpr int esz = DT == E_F32X ? 4 : 2;
        float v[8];
        load8<DT>(static_cast<const char *>(c.x) + r * c.ldx * esz, col, n, vx, v);
        uint32_t m = amax8(v);
        const uint32_t half = 0xffffu << (threadIdx.x & 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half, m, o));
        const BlockScale s = block_scale(m);
        if (lane == 0) c.scale[r * c.ld_scale + kb] = s.scale;
        store8(c.q + r * c.ldq + col, n, vq, v, s.inv);
    }
}

// One 128 x 128 block per CTA: 256 threads of 8 rows (16 apart) x 8 columns, held in registers
// between the maximum and the conversion.
template <int DT>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(QuantizeCall c, bool vx, bool vq) {
    __shared__ uint32_t warp_max[8];
    const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 128 + lane * 8;
    const int n = (int)max((int64_t)0, min((int64_t)8, c.cols - col));
    constexpr int esz = DT == E_F32X ? 4 : 2;
    for (int64_t br = blockIdx.y; br * 128 < c.rows; br += gridDim.y) {
        float v[8][8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = br * 128 + i * 16 + r0;
            load8<DT>(static_cast<const char *>(c.x) + r * c.ldx * esz, col, r < c.rows ? n : 0, vx, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, amax8(v[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, warp_max[i]);
        __syncthreads();
        const BlockScale s = block_scale(m);
        if (threadIdx.x == 0) c.scale[br * c.ld_scale + blockIdx.x] = s.scale;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = br * 128 + i * 16 + r0;
            if (r < c.rows) store8(c.q + r * c.ldq + col, n, vq, v[i], s.inv);
        }
    }
}

template <int DT>
Status launch_dt(const QuantizeCall &c, cudaStream_t stream) {
    constexpr int esz = DT == E_F32X ? 4 : 2;
    const bool vx = (reinterpret_cast<uintptr_t>(c.x) & 15) == 0 && (c.ldx * esz) % 16 == 0;
    const bool vq = (reinterpret_cast<uintptr_t>(c.q) & 7) == 0 && c.ldq % 8 == 0;
    const int64_t per_row = (c.cols + 127) / 128;
    if (c.block_rows == 1) {
        const int64_t blocks = c.rows * per_row;
        const int64_t ctas = (blocks + 15) / 16;
        const unsigned grid = (unsigned)std::min<int64_t>(ctas, (int64_t)num_sms() * 8);
        quantize_rows_kernel<DT><<<grid, 256, 0, stream>>>(c, blocks, per_row, vx, vq);
    } else {
        const int64_t tiles = (c.rows + 127) / 128;
        const dim3 grid((unsigned)per_row, (unsigned)std::min<int64_t>(tiles, 65535));
        quantize_tiles_kernel<DT><<<grid, 256, 0, stream>>>(c, vx, vq);
    }
    const cudaError_t e = cudaGetLastError();
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
