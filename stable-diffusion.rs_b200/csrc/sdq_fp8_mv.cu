// sdq_fp8_mv.cu -- product of block-scaled e4m3 operands for a few tokens (m <= 32), bound by the
// weight's bytes.
//
// The formula is sdq_fp8_mm.cu's.  There a step of 128 values of K takes 300 cycles however few tokens
// there are, one step after another; here the steps of a tile are spread over eight warps.  A CTA takes
// 16 features (one weight scale a step); warp w takes the steps w, w + 8, ... and multiplies the codes
// as they lie, mma.sync m16n8k32 (e4m3, f32 sums), features on the rows and tokens on the columns.
// The order of the values of K within a step does not matter as long as both operands share it, so a
// lane feeds its fragments from 16-byte pieces: bytes 16 j .. 16 j + 15 (and those 64 further) of its
// two feature rows and its token row, j = lane % 4.  Nothing is unpacked and nothing passes through
// shared memory on the way.  Each step's sums are scaled by 2^(ex + ew) and added up in f32; the
// eight warps' sums meet in shared memory in a fixed order.
#include <cstdint>
#include <cuda_runtime.h>

#include "sdq_dequant.cuh"
#include "sdq_epilogue.cuh"
#include "sdq_fp8.cuh"
#include "sdq_internal.h"
#include "sdq_ptx.cuh"

namespace sdq {
namespace {

constexpr int kRows = 16;                  // features of a CTA
constexpr int kWarps = 8;

// 16 bytes of the weight, which nothing reads again soon.
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// v 2^(ex + ew - 254) in two steps, so that neither overflows unless the result does.
__device__ __forceinline__ float scaled(float v, uint32_t ex, uint32_t ew) {
    if (ex == 255u || ew == 255u) return __uint_as_float(0x7FFFFFFFu);
    const int e = (int)(ex + ew) - 254, h = e >> 1;
    return v * e8m0_value((uint32_t)(h + 127)) * e8m0_value((uint32_t)(e - h + 127));
}

// NT: tokens in eights.  U: steps whose loads a warp has under way at once.
template <int NT, int U>
__global__ void __launch_bounds__(32 * kWarps)
    fp8_mv_kernel(const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, int m, int k,
                  const uint8_t* __restrict__ wq, const uint8_t* __restrict__ ws, int n, const EpiArgs epi, void* y) {
    __shared__ float part[kWarps][NT * 8][kRows + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int f0 = blockIdx.x * kRows, kt = (k + kFp8Block - 1) / kFp8Block;
    // Rows and tokens that are not there read the last one's: what they give is not stored.
    const uint8_t* w0 = wq + (int64_t)min(f0 + g, n - 1) * k + 16 * j;
    const uint8_t* w1 = wq + (int64_t)min(f0 + g + 8, n - 1) * k + 16 * j;
    const uint8_t* x[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = xq + (int64_t)min(8 * t + g, m - 1) * k + 16 * j;
    const uint8_t* wscale = ws + (int64_t)(f0 / kFp8Block) * kt;
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
    griddep_wait();
    griddep_launch_dependents();
    for (int s0 = warp; s0 < kt; s0 += kWarps * U) {
        uint4 a[U][2][2], b[U][2][NT];
        uint32_t ew[U], ex[U][NT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * kWarps;
            const int at = min(s, kt - 1) * kFp8Block;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool in = s < kt && at + 64 * h + 16 * j < k;
                const uint4 zero = make_uint4(0, 0, 0, 0);
                a[u][h][0] = in ? ld_stream(w0 + at + 64 * h) : zero;
                a[u][h][1] = in ? ld_stream(w1 + at + 64 * h) : zero;
#pragma unroll
                for (int t = 0; t < NT; ++t) b[u][h][t] = in ? __ldg(reinterpret_cast<const uint4*>(x[t] + at + 64 * h)) : zero;
            }
            ew[u] = __ldg(wscale + min(s, kt - 1));
            const uint8_t* row = xs + (int64_t)min(s, kt - 1) * m;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) ex[u][t][i] = __ldg(row + min(8 * t + 2 * j + i, m - 1));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u * kWarps >= kt) break;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mma_e4m3(c, a[u][h][0].x, a[u][h][1].x, a[u][h][0].y, a[u][h][1].y, b[u][h][t].x, b[u][h][t].y);
                    mma_e4m3(c, a[u][h][0].z, a[u][h][1].z, a[u][h][0].w, a[u][h][1].w, b[u][h][t].z, b[u][h][t].w);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] += scaled(c[i], ex[u][t][i & 1], ew[u]);
            }
        }
    }
    // c[0], c[1]: feature g, tokens 2j and 2j + 1; c[2], c[3]: feature g + 8.
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[warp][8 * t + 2 * j + (i & 1)][g + 8 * (i >> 1)] = acc[t][i];
    __syncthreads();
    for (int o = threadIdx.x; o < NT * 8 * kRows; o += 32 * kWarps) {
        const int t = o / kRows, r = o % kRows, f = f0 + r;
        if (t >= m || f >= n) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += part[w][t][r];
        const int64_t at = (int64_t)t * n + f;
        if (epi.f32) {
            if (epi.bias != nullptr) v += reinterpret_cast<const float*>(epi.bias)[f];
            static_cast<float*>(y)[at] = v;
        } else {
            if (epi.bias != nullptr) v += bf16_bits_to_f32(epi.bias[f]);
            v = epi_activation(v, epi.act);
            if (epi.gate != nullptr) v *= bf16_bits_to_f32(epi.gate[f]);
            if (epi.resid != nullptr) v += bf16_bits_to_f32(epi.resid[at]);
            static_cast<uint16_t*>(y)[at] = (uint16_t)(pack_bf16x2(v, 0.f) & 0xFFFFu);
        }
    }
}

}  // namespace

int fp8_mv_tokens() { return 32; }

cudaError_t launch_fp8_mv(const uint8_t* xq, const uint8_t* xs, int64_t m, int64_t k, const uint8_t* wq,
                          const uint8_t* ws, int64_t n, const EpiArgs& epi, void* y, cudaStream_t st) {
    const dim3 grid((unsigned)((n + kRows - 1) / kRows));
    auto go = [&](auto kernel) {
        return launch_programmatic(kernel, grid, 32 * kWarps, 0, st, xq, xs, (int)m, (int)k, wq, ws, (int)n, epi, y);
    };
    if (m <= 8) return go(fp8_mv_kernel<1, 2>);
    if (m <= 16) return go(fp8_mv_kernel<2, 2>);
    return go(fp8_mv_kernel<4, 1>);
}

}  // namespace sdq
