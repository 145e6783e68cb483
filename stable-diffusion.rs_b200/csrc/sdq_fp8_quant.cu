// sdq_fp8_quant.cu -- quantise to and from block-scaled e4m3 (sdq_fp8.cuh).
//
//   s = 2^e, e = least integer >= -126 with max|x| <= 448 * 2^e;  q = rn_e4m3(x / s)
//
// over the 128 values of a row's group (activations) or a 128 x 128 block (weights).  x / s is
// exact in f32 (a shift of the exponent), so each value is rounded exactly once.  An infinity or
// a NaN makes its whole group NaN: the scale byte is 255 and every code 0x7F.
//
// All of it is bound by memory: 2 or 4 bytes in and one out per value, each touched once; the
// group stays in registers between its maximum and its rounding.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "sdq_dequant.cuh"
#include "sdq_fp8.cuh"
#include "sdq_internal.h"
#include "sdq_ptx.cuh"

namespace sdq {
namespace {

// 16 consecutive values of a row held by one thread, and their largest |bits|.
template <bool BF16>
struct Sixteen;
template <>
struct Sixteen<true> {
    uint32_t w[8];
    __device__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ void load(const void* p, int64_t e) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e);
        const uint4 a = s[0], b = s[1];
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ float get(int i) const {
        return i & 1 ? __uint_as_float(w[i >> 1] & 0xFFFF0000u) : __uint_as_float(w[i >> 1] << 16);
    }
};
template <>
struct Sixteen<false> {
    uint32_t w[16];
    __device__ void zero() {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = 0;
    }
    __device__ void load(const void* p, int64_t e) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 a = s[i];
            w[4 * i] = a.x; w[4 * i + 1] = a.y; w[4 * i + 2] = a.z; w[4 * i + 3] = a.w;
        }
    }
    __device__ float get(int i) const { return __uint_as_float(w[i]); }
};

// Fours of rows that a warp of fp8_quantize_rows takes.
template <bool BF16>
__host__ __device__ constexpr int row_quads() { return BF16 ? 2 : 1; }

template <class V>
__device__ __forceinline__ uint32_t largest(const V& v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v.get(i)) & 0x7FFFFFFFu);
    return m;
}
template <class V>
__device__ __forceinline__ uint4 encode(const V& v, float inv) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = e4m3x2(v.get(4 * i) * inv, v.get(4 * i + 1) * inv) |
               (e4m3x2(v.get(4 * i + 2) * inv, v.get(4 * i + 3) * inv) << 16);
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// Activations: eight lanes take the 128 values of one group, a warp the same group of four
// consecutive rows, so that the four scale bytes, which lie [group, row], share a sector; of bf16
// it takes eight rows, for as many bytes under way as of f32.  A dozen calls in a graph, at full clocks:
// 4608 x 12288 bf16 27 us (6.3 TB/s), four rows 28.6, sixteen 29.5; f32 42 us (6.7 TB/s).  Call after call
// the bf16 case takes 28.5 us (6.0 TB/s).
template <bool BF16>
__global__ void __launch_bounds__(256) fp8_quantize_rows(const void* x, int64_t m, int64_t k, uint8_t* q,
                                                         uint8_t* scales) {
    constexpr int NQ = row_quads<BF16>();
    const int lane = threadIdx.x & 31;
    const uint32_t kb = (uint32_t)((k + kFp8Block - 1) / kFp8Block);
    const uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 5);      // below 2^32: m <= 2^30, and memory's size
    const uint32_t part = u / kb, g = u - part * kb;
    const int64_t row0 = (int64_t)4 * NQ * part + (lane >> 3);
    const int64_t c = g * kFp8Block + 16 * (lane & 7);
    Sixteen<BF16> v[NQ];
    griddep_wait();
    griddep_launch_dependents();
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        v[i].zero();
        if (row0 + 4 * i < m && c < k) v[i].load(x, (row0 + 4 * i) * k + c);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int64_t row = row0 + 4 * i;
        uint32_t a = largest(v[i]);
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, d));
        const uint32_t byte = e8m0_of(a);
        if (row < m && c < k) *reinterpret_cast<uint4*>(q + row * k + c) = encode(v[i], e8m0_inverse(byte));
        if ((lane & 7) == 0 && row < m) scales[g * m + row] = (uint8_t)byte;
    }
}

// Weights: one CTA per 128 x 128 block, four rows of 16 values per thread.  32768 x 5120 bf16: 80 us call
// after call (6.3 TB/s), 75 in a few calls at full clocks.
template <bool BF16>
__global__ void __launch_bounds__(256) fp8_quantize_blocks(const void* __restrict__ w, int64_t n, int64_t k,
                                                           uint8_t* __restrict__ q, uint8_t* __restrict__ scales) {
    __shared__ uint32_t part[8];
    const int64_t kb = (k + kFp8Block - 1) / kFp8Block;
    const int64_t nb = blockIdx.x / kb, g = blockIdx.x - nb * kb;
    const int64_t c = g * kFp8Block + 16 * (threadIdx.x & 7);
    const int64_t r0 = nb * kFp8Block + (threadIdx.x >> 3);
    Sixteen<BF16> v[4];
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i].zero();
        if (r0 + 32 * i < n && c < k) v[i].load(w, (r0 + 32 * i) * k + c);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) a = max(a, largest(v[i]));
    a = __reduce_max_sync(0xFFFFFFFFu, a);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, part[i]);
    const uint32_t byte = e8m0_of(a);
    const float inv = e8m0_inverse(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r0 + 32 * i < n && c < k) *reinterpret_cast<uint4*>(q + (r0 + 32 * i) * k + c) = encode(v[i], inv);
    if (threadIdx.x == 0) scales[blockIdx.x] = (uint8_t)byte;
}

// The values that codes and scales stand for (tests, and layers without an fp8 product): 16 per
// thread.  Scale of value (r, c): scales[(c / 128) * rows + r] for activations,
// scales[(r / 128) * ceil(k / 128) + c / 128] for weights.
template <bool OUT_F32>
__global__ void __launch_bounds__(256) fp8_dequantize_kernel(const uint8_t* __restrict__ q,
                                                             const uint8_t* __restrict__ scales, int64_t rows,
                                                             int64_t k, int weight, void* __restrict__ out) {
    const int64_t per_row = k / 16, total = rows * per_row, kb = (k + kFp8Block - 1) / kFp8Block;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / per_row, c = 16 * (i - r * per_row), g = c / kFp8Block;
        const float s = e8m0_value(scales[weight ? (r / kFp8Block) * kb + g : g * rows + r]);
        const uint4 v = *reinterpret_cast<const uint4*>(q + r * k + c);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        float f[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[j >> 1] >> (16 * (j & 1))), __NV_E4M3);
            const float2 p = __half22float2(__half2(h));
            f[2 * j] = p.x * s;
            f[2 * j + 1] = p.y * s;
        }
        if (OUT_F32) {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + r * k + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
        } else {
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                o[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + r * k + c);
            dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
            dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
}

}  // namespace

cudaError_t launch_fp8_quantize(const void* x, bool bf16, int64_t m, int64_t k, uint8_t* q, uint8_t* scales,
                                cudaStream_t st) {
    const int64_t kb = (k + kFp8Block - 1) / kFp8Block, rows = 4 * (bf16 ? row_quads<true>() : row_quads<false>());
    const int64_t warps = (m + rows - 1) / rows * kb;
    const unsigned grid = (unsigned)((warps + 7) / 8);
    return launch_programmatic(bf16 ? fp8_quantize_rows<true> : fp8_quantize_rows<false>, dim3(grid), 256, 0, st, x, m, k, q,
                               scales);
}

cudaError_t launch_fp8_quantize_weight(const void* w, bool bf16, int64_t n, int64_t k, uint8_t* q,
                                       uint8_t* scales, cudaStream_t st) {
    const unsigned grid = (unsigned)(((n + kFp8Block - 1) / kFp8Block) * ((k + kFp8Block - 1) / kFp8Block));
    if (bf16) fp8_quantize_blocks<true><<<grid, 256, 0, st>>>(w, n, k, q, scales);
    else fp8_quantize_blocks<false><<<grid, 256, 0, st>>>(w, n, k, q, scales);
    return cudaGetLastError();
}

cudaError_t launch_fp8_dequantize(const uint8_t* q, const uint8_t* scales, int64_t rows, int64_t k, bool weight,
                                  void* out, bool out_f32, cudaStream_t st) {
    const int64_t want = (rows * (k / 16) + 255) / 256, cap = (int64_t)num_sms() * 16;
    const int grid = (int)(want < cap ? want : cap);
    if (out_f32) fp8_dequantize_kernel<true><<<grid, 256, 0, st>>>(q, scales, rows, k, weight ? 1 : 0, out);
    else fp8_dequantize_kernel<false><<<grid, 256, 0, st>>>(q, scales, rows, k, weight ? 1 : 0, out);
    return cudaGetLastError();
}

}  // namespace sdq
