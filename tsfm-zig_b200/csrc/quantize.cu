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

// Eight consecutive elements of a row as they are stored; elements at or past `n` read as zero.
template <int DT>
struct Raw8 {
    uint4 w[DT == E_F32X ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void *row, int64_t col, int n, bool vec) {
    Raw8<DT> r;
    constexpr int W = DT == E_F32X ? 2 : 1;
    if (vec && n >= 8) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(row) + col * (DT == E_F32X ? 4 : 2));
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

template <int DT>
__device__ __forceinline__ void to_f32(const Raw8<DT> &r, float (&v)[8]) {
    if constexpr (DT == E_F32X) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v[4 * i] = __uint_as_float(r.w[i].x), v[4 * i + 1] = __uint_as_float(r.w[i].y);
            v[4 * i + 2] = __uint_as_float(r.w[i].z), v[4 * i + 3] = __uint_as_float(r.w[i].w);
        }
    } else {
        const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
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

// One row x 128 columns per half warp: 16 lanes of 8 elements. A half warp takes U blocks, all of
// whose loads are under way before the first maximum; the CTA's 16 U blocks are consecutive.
template <int DT, int U>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeCall c, int64_t blocks, uint32_t per_row, bool vx,
                                                            bool vq) {
    constexpr int esz = DT == E_F32X ? 4 : 2;
    const int lane = threadIdx.x & 15;
    const int64_t first = (int64_t)blockIdx.x * (16 * U);
    const int64_t r0 = first / per_row;
    const uint32_t kb0 = (uint32_t)(first - r0 * per_row);
    Raw8<DT> raw[U];
    int64_t row[U];
    uint32_t kb[U];
    int n[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t b = u * 16 + (threadIdx.x >> 4), k = kb0 + b, q = k / per_row;
        row[u] = r0 + q;
        kb[u] = k - q * per_row;
        const int64_t col = (int64_t)kb[u] * 128 + lane * 8;
        n[u] = first + b < blocks ? (int)max((int64_t)0, min((int64_t)8, c.cols - col)) : 0;
        raw[u] = load8<DT>(static_cast<const char *>(c.x) + (n[u] > 0 ? row[u] : 0) * c.ldx * esz, col, n[u], vx);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float v[8];
        to_f32<DT>(raw[u], v);
        uint32_t m = amax8(v);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const BlockScale s = block_scale(m);
        if (n[u] > 0) {
            if (lane == 0) c.scale[row[u] * c.ld_scale + kb[u]] = s.scale;
            store8(c.q + row[u] * c.ldq + kb[u] * 128 + lane * 8, n[u], vq, v, s.inv);
        }
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
        Raw8<DT> raw[8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = br * 128 + i * 16 + r0;
            raw[i] = load8<DT>(static_cast<const char *>(c.x) + r * c.ldx * esz, col, r < c.rows ? n : 0, vx);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v[8];
            to_f32<DT>(raw[i], v);
            m = max(m, amax8(v));
        }
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
            float v[8];
            to_f32<DT>(raw[i], v);
            if (r < c.rows) store8(c.q + r * c.ldq + col, n, vq, v, s.inv);
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
        constexpr int U = DT == E_F32X ? 2 : 4;  // 64 bytes a thread in flight
        const int64_t ctas = (blocks + 16 * U - 1) / (16 * U);
        if (ctas > INT32_MAX) return Status::fail(TSFM_ERR_UNSUPPORTED, "quantize: too many blocks");
        quantize_rows_kernel<DT, U><<<(unsigned)ctas, 256, 0, stream>>>(c, blocks, (uint32_t)per_row, vx, vq);
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
