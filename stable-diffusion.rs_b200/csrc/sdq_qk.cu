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
// the halves' partners by shuffles.  A warp takes one token and, for each vector's worth of its
// lanes, kBatch heads of one of the three tensors, all loads issued before the first is worked on;
// the warps of a block take neighbouring tokens of the same heads, which lie side by side in the
// output.  The norm's weights are multiplied into the cosines and sines once for all the heads:
// a c - b s becomes r (x0 (w0 c) - x1 (w1 s)), three operations a value.
// 4608 tokens, 72 heads of 128: a block a token, looping over its heads, took 63 us (49 KB a SM
// under way); this layout 40 with the norm and the rotation one after the other, now 30.4 (5.6 TB/s).
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "sdq_internal.h"
#include "sdq_ptx.cuh"

namespace sdq {
namespace {

// A block: 8 warps took 34 us for the case above, 4 and 2 30.3 (2 10 % longer at 4096 x 18 heads of
// 80), 1 43.8; plain loads 3 % less than streaming ones.
constexpr int kWarps = 4;
// Heads a lane group loads before it works on the first: 2 took 10 % longer than 4, 8 20 %; one, for
// calls of a few tokens, gained 4 % up to 16 tokens and lost 15 % at 128.
constexpr int kBatch = 4;

// Eight values as they are loaded.
template <bool BF16>
struct Raw;
template <>
struct Raw<true> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const void* p, int64_t e) {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ float get(int i) const {
        return i & 1 ? __uint_as_float(w[i >> 1] & 0xFFFF0000u) : __uint_as_float(w[i >> 1] << 16);
    }
    static __device__ __forceinline__ void store(void* p, int64_t e, const float (&f)[8]) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            o[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + e) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __device__ __forceinline__ void put(void* p, int64_t e) const {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + e) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static constexpr int N = 4;
};
template <>
struct Raw<false> {
    uint32_t w[8];
    __device__ __forceinline__ void load(const void* p, int64_t e) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + e);
        const uint4 a = s[0], b = s[1];
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(w[i]); }
    static __device__ __forceinline__ void store(void* p, int64_t e, const float (&f)[8]) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + e);
        d[0] = make_float4(f[0], f[1], f[2], f[3]);
        d[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    __device__ __forceinline__ void put(void* p, int64_t e) const {
        uint4* d = reinterpret_cast<uint4*>(static_cast<float*>(p) + e);
        d[0] = make_uint4(w[0], w[1], w[2], w[3]);
        d[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    static constexpr int N = 8;
};

// LPV lanes hold one vector.  blockIdx.y counts pieces of the queries' heads, then the keys', then
// the values'.
template <bool BF16, bool INTER, int LPV>
__global__ void __launch_bounds__(32 * kWarps) qk_kernel(const __grid_constant__ QkArgs a) {
    constexpr int kSide = 32 / LPV, kHeads = kSide * kBatch;      // vectors side by side; heads a piece
    const int lane = threadIdx.x & 31, l = lane % LPV, e = 8 * l;
    const uint32_t bt = blockIdx.x * kWarps + (threadIdx.x >> 5);      // batch * tokens < 2^31
    if (bt >= (uint32_t)(a.batch * a.tokens)) return;    // whole warps
    const int64_t b = bt / (uint32_t)a.tokens, t = bt - (uint32_t)b * (uint32_t)a.tokens;
    int piece = blockIdx.y, kind = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int n = (a.heads[i] + kHeads - 1) / kHeads;
        if (kind == i && piece >= n) { piece -= n; kind = i + 1; }
    }
    const QkTensor& x = a.in[kind];
    const QkTensor& y = a.out[kind];
    // Vectors this lane takes part in (a head of 80 values fills 10 of 16 lanes).
    const int h0 = piece * kHeads + lane / LPV;
    const int count = e < a.d ? a.heads[kind] - h0 : 0;  // vector j is there when j * kSide < count
    int64_t from = b * x.batch_stride + t * x.token_stride + h0 * x.head_stride + e;
    int64_t to = b * y.batch_stride + t * y.token_stride + h0 * y.head_stride + e;

    Raw<BF16> v[kBatch];
    griddep_wait();
    griddep_launch_dependents();
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
        if (j * kSide < count) {
            v[j].load(x.data, from + j * kSide * x.head_stride);
        } else {
#pragma unroll
            for (int i = 0; i < Raw<BF16>::N; ++i) v[j].w[i] = 0;
        }
    }
    if (kind == 2) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (j * kSide < count) v[j].put(y.data, to + j * kSide * y.head_stride);
        return;
    }

    // The norm's weights of this lane's values and, in halves, of their partners' (1 without a norm).
    const void* weight = a.weight[kind];
    const int half = a.rope / 2;
    const bool turns = e < a.rope;                       // whole lanes turn or stay: R is a multiple of 16
    const bool low = e < half;                           // halves: in the first half of the pair
    const int partner = turns && !INTER ? (low ? e + half : e - half) : e;
    float w[8], wp[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = wp[i] = 1.f;
    if (weight != nullptr && e < a.d) {
        Raw<BF16> g;
        g.load(weight, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = g.get(i);
        if (!INTER) {
            g.load(weight, partner);
#pragma unroll
            for (int i = 0; i < 8; ++i) wp[i] = g.get(i);
        }
    }
    // What each value, and its partner's, is multiplied by.  A position outside the tables reads
    // nothing and makes the token's queries and keys NaN.
    float own[8], other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { own[i] = w[i]; other[i] = 0.f; }
    if (turns) {
        int64_t row = t;
        if (a.positions != nullptr) {
            const int64_t at = b * a.pos_batch_stride + t;
            row = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
        }
        if (row < 0 || row >= a.table_rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i) own[i] = other[i] = __uint_as_float(0x7FFFFFFFu);
        } else {
            constexpr int NC = INTER ? 4 : 8;
            float c[NC], s[NC];
            const int64_t at = row * half + (INTER ? e / 2 : (low ? e : e - half));
#pragma unroll
            for (int i = 0; i < NC / 4; ++i) {
                const float4 cc = __ldg(reinterpret_cast<const float4*>(a.cos + at) + i);
                const float4 ss = __ldg(reinterpret_cast<const float4*>(a.sin + at) + i);
                c[4 * i] = cc.x; c[4 * i + 1] = cc.y; c[4 * i + 2] = cc.z; c[4 * i + 3] = cc.w;
                s[4 * i] = ss.x; s[4 * i + 1] = ss.y; s[4 * i + 2] = ss.z; s[4 * i + 3] = ss.w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (INTER) {                             // even values: a c - b s; odd ones: b c + a s
                    own[i] = w[i] * c[i / 2];
                    other[i] = w[i ^ 1] * (i & 1 ? s[i / 2] : -s[i / 2]);
                } else {
                    own[i] = w[i] * c[i];
                    other[i] = wp[i] * (low ? -s[i] : s[i]);
                }
            }
        }
    }

    float r[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
        r[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[j] = fmaf(v[j].get(i), v[j].get(i), r[j]);
    }
#pragma unroll
    for (int m = 1; m < LPV; m <<= 1) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) r[j] += __shfl_xor_sync(0xFFFFFFFFu, r[j], m);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
        Raw<BF16> o;                                     // halves: the partner's values
        if (!INTER) {
            const int lp = lane + (partner - e) / 8;
#pragma unroll
            for (int i = 0; i < Raw<BF16>::N; ++i) o.w[i] = __shfl_sync(0xFFFFFFFFu, v[j].w[i], lp);
        }
        if (j * kSide < count) {
            const float rj = weight != nullptr ? rsqrtf(r[j] * a.inv_d + a.eps) : 1.f;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = v[j].get(i) * own[i];
                if (turns) f[i] = fmaf(INTER ? v[j].get(i ^ 1) : o.get(i), other[i], f[i]);
                f[i] *= rj;
            }
            Raw<BF16>::store(y.data, to + j * kSide * y.head_stride, f);
        }
    }
}

template <bool BF16, bool INTER, int LPV>
cudaError_t go(const QkArgs& a, cudaStream_t st) {
    constexpr int kSide = 32 / LPV;
    const unsigned blocks = (unsigned)((a.batch * a.tokens + kWarps - 1) / kWarps);
    unsigned pieces = 0;
    for (int h : a.heads) pieces += (unsigned)((h + kBatch * kSide - 1) / (kBatch * kSide));
    return launch_programmatic(qk_kernel<BF16, INTER, LPV>, dim3(blocks, pieces), 32 * kWarps, 0, st, a);
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
