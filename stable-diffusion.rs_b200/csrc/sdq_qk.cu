// sdq_qk.cu -- queries, keys and values made ready for attention in one pass.
//
// For every head vector x of d values at (batch b, token t):
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (queries and keys; no w: y = x)
//   rotate the first R values of y by the angles of row p of the tables, p = t or positions[b, t]:
//     interleaved  (y[2i], y[2i+1])      halves  (y[i], y[i + R/2])
//     -> (a cos_i - b sin_i, a sin_i + b cos_i)
//   write it at [b, head, t], whatever strides input and output have; values are copied
//
// in f32 from the loaded to the stored value, rounded once.  This is the reference's split_qkv,
// qk_norm, concatenation of the text and image streams (through the output's strides) and rotate
// (crates/sd-models/src/mlx/flux.rs:302-329, 165-212), and the q / k norm and half-split rotation
// of its decoder-only encoders (llm.rs:226-291).
//
// Bound by memory: every value is read and written once.  A vector lies in the registers of the
// fewest lanes (a power of two) that hold it at 8 values each: 16-byte accesses for bf16, sums and
// the halves' partners by shuffles.  A block takes one token's heads (or several tokens when there
// are few heads), so the table row is read once and kept in registers for all of them, and each
// lane has kBatch vectors' loads under way at once.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "sdq_internal.h"

namespace sdq {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;      // vectors a lane loads before it works on the first

template <bool BF16>
struct Eight {
    float f[8];
    __device__ __forceinline__ void load(const void* p, int64_t e) {
        if (BF16) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        } else {
            const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + e);
            const float4 a = __ldcs(s), b = __ldcs(s + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
            f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t e) const {
        if (BF16) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                o[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + e) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
            float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + e);
            d[0] = make_float4(f[0], f[1], f[2], f[3]);
            d[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
    }
};

// LPV lanes hold one vector; `per_token` vector slots of the block work on the same token.
template <bool BF16, bool INTER, int LPV>
__global__ void __launch_bounds__(kThreads) qk_kernel(const __grid_constant__ QkArgs a, int per_token) {
    constexpr int kSlots = kThreads / LPV;
    const int slot = threadIdx.x / LPV, l = threadIdx.x % LPV;
    const int64_t bt = (int64_t)blockIdx.x * (kSlots / per_token) + slot / per_token;
    const bool live = bt < a.batch * a.tokens && 8 * l < a.d;
    const int64_t b = live ? bt / a.tokens : 0, t = live ? bt - b * a.tokens : 0;
    const int all = a.heads[0] + a.heads[1] + a.heads[2];

    // This lane's cosines and sines, if its values are in the rotated part (whole lanes are: R is
    // a multiple of 16).  A position outside the tables reads nothing and makes the token's
    // queries and keys NaN.
    constexpr int NC = INTER ? 4 : 8;
    float c[NC], s[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) c[i] = s[i] = 0.f;
    const int half = a.rope / 2;
    const int e = 8 * l;
    const bool low = e < half;                           // halves: in the first half of the pair
    const bool turns = e < a.rope;
    if (live && turns) {
        int64_t row = t;
        if (a.positions != nullptr) {
            const int64_t at = b * a.pos_batch_stride + t;
            row = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
        }
        if (row < 0 || row >= a.table_rows) {
#pragma unroll
            for (int i = 0; i < NC; ++i) c[i] = s[i] = __uint_as_float(0x7FFFFFFFu);
        } else {
            const int64_t at = row * half + (INTER ? e / 2 : (low ? e : e - half));
#pragma unroll
            for (int i = 0; i < NC / 4; ++i) {
                const float4 cc = __ldg(reinterpret_cast<const float4*>(a.cos + at) + i);
                const float4 ss = __ldg(reinterpret_cast<const float4*>(a.sin + at) + i);
                c[4 * i] = cc.x; c[4 * i + 1] = cc.y; c[4 * i + 2] = cc.z; c[4 * i + 3] = cc.w;
                s[4 * i] = ss.x; s[4 * i + 1] = ss.y; s[4 * i + 2] = ss.z; s[4 * i + 3] = ss.w;
            }
        }
    }

    // Every lane of the block makes the same number of trips: the shuffles below need them all.
    const int step = per_token * gridDim.y;
    for (int h0 = blockIdx.y * per_token; h0 < all; h0 += kBatch * step) {
        Eight<BF16> v[kBatch];
        int kind[kBatch], head[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            int h = h0 + j * step + slot % per_token;
            kind[j] = -1;
            if (live && h < all) {
                kind[j] = 0;
                if (h >= a.heads[0]) { h -= a.heads[0]; kind[j] = 1; }
                if (kind[j] == 1 && h >= a.heads[1]) { h -= a.heads[1]; kind[j] = 2; }
                head[j] = h;
                const QkTensor& x = a.in[kind[j]];
                v[j].load(x.data, b * x.batch_stride + t * x.token_stride + h * x.head_stride + e);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j].f[i] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            float* f = v[j].f;
            const void* w = kind[j] == 0 ? a.weight[0] : (kind[j] == 1 ? a.weight[1] : nullptr);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
#pragma unroll
            for (int m = 1; m < LPV; m <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
            if (w != nullptr) {
                const float r = rsqrtf(sum * a.inv_d + a.eps);
                Eight<BF16> g;
                g.load(w, e);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = f[i] * r * g.f[i];
            }
            if (INTER) {
                if (turns && kind[j] != 2) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = f[2 * i], q = f[2 * i + 1];
                        f[2 * i] = p * c[i] - q * s[i];
                        f[2 * i + 1] = p * s[i] + q * c[i];
                    }
                }
            } else {
                // The partner of value i lies R/2 further on: half / 8 lanes up, or down.
                const int from = (threadIdx.x & 31) + (turns ? (low ? half / 8 : -(half / 8)) : 0);
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xFFFFFFFFu, f[i], from);
                if (turns && kind[j] != 2) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = f[i] * c[i] + (low ? -o[i] : o[i]) * s[i];
                }
            }
            if (kind[j] >= 0) {
                const QkTensor& y = a.out[kind[j]];
                v[j].store(y.data, b * y.batch_stride + t * y.token_stride + head[j] * y.head_stride + e);
            }
        }
    }
}

template <bool BF16, bool INTER, int LPV>
cudaError_t go(const QkArgs& a, cudaStream_t st) {
    constexpr int kSlots = kThreads / LPV;
    const int all = a.heads[0] + a.heads[1] + a.heads[2];
    int per_token = kSlots;
    while (per_token > 1 && per_token / 2 >= all) per_token /= 2;
    const int64_t blocks = (a.batch * a.tokens + kSlots / per_token - 1) / (kSlots / per_token);
    // Few tokens: their heads are spread over blocks, one vector per slot, rather than queued.
    const int trips = (all + per_token - 1) / per_token;
    const int spread = blocks * 4 < num_sms() ? trips : 1;
    qk_kernel<BF16, INTER, LPV><<<dim3((unsigned)blocks, (unsigned)spread), kThreads, 0, st>>>(a, per_token);
    return cudaGetLastError();
}

template <bool BF16, bool INTER>
cudaError_t by_width(const QkArgs& a, cudaStream_t st) {
    const int lanes = (a.d + 7) / 8;
    if (lanes <= 1) return go<BF16, INTER, 1>(a, st);
    if (lanes <= 2) return go<BF16, INTER, 2>(a, st);
    if (lanes <= 4) return go<BF16, INTER, 4>(a, st);
    if (lanes <= 8) return go<BF16, INTER, 8>(a, st);
    if (lanes <= 16) return go<BF16, INTER, 16>(a, st);
    return go<BF16, INTER, 32>(a, st);
}

}  // namespace

cudaError_t launch_qk_norm_rope(const QkArgs& a, bool bf16, bool interleaved, cudaStream_t st) {
    if (bf16) return interleaved ? by_width<true, true>(a, st) : by_width<true, false>(a, st);
    return interleaved ? by_width<false, true>(a, st) : by_width<false, false>(a, st);
}

}  // namespace sdq
