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
// the halves' partners by shuffles.  A warp works on one of the three tensors.  The vectors that fit
// its lanes side by side are heads of one token, or, of tensors with fewer heads than that, the heads
// of several tokens; for each of them it takes BATCH heads, all loads issued before the first is
// worked on.  The warps of a block take neighbouring tokens of the same heads, which lie side by side
// in the output.  The norm's weights are multiplied into the cosines and sines once for all the heads:
// a c - b s becomes r (x0 (w0 c) - x1 (w1 s)), three operations a value.
// 4608 tokens, 72 heads of 128: a block a token, looping over its heads, took 63 us (49 KB a SM
// under way); this layout 40 with the norm and the rotation one after the other, now 30.9 in a graph and
// 31.8 call after call (5.4 TB/s).
// 4 x 8192 tokens with one query and one key head of 64: 35 us with a token a warp, 7.9 with four.
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
// BATCH, the heads a lane group loads before it works on the first: 4 (2 took 10 % longer for the case
// above, 8 20 %), or 1 or 2 where no tensor has more for it, which leaves registers for more warps
// (8192 tokens with 4 query and 2 key heads of 128: 12.1 us by 4, 9.5 by 2).

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

// What go() has settled for a launch: for each tensor the logarithm of how many heads lie side by side
// in a warp (the other lanes take further tokens) and the pieces that its heads come in.
struct QkPlan {
    int log_side[3], pieces[3];
};

// LPV lanes hold one vector.  blockIdx.y counts the pieces of the queries, then the keys', then the
// values'; tokens go along x (the pieces of one token next to one another took 6 % longer).
template <bool BF16, bool INTER, int LPV, int BATCH>
__global__ void __launch_bounds__(32 * kWarps) qk_kernel(const __grid_constant__ QkArgs a, const __grid_constant__ QkPlan p) {
    const int lane = threadIdx.x & 31, l = lane % LPV, e = 8 * l;
    int piece = blockIdx.y, kind = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (kind == i && piece >= p.pieces[i]) { piece -= p.pieces[i]; kind = i + 1; }
    const int log_side = p.log_side[kind], side = 1 << log_side, apart = (32 / LPV) >> log_side;   // heads, tokens of a warp
    const int group = lane / LPV, which = group & (side - 1);
    const uint64_t first = (uint64_t)(blockIdx.x * kWarps + (threadIdx.x >> 5)) * apart;
    const uint32_t all = (uint32_t)(a.batch * a.tokens);                 // < 2^31
    if (first >= all) return;                            // whole warps
    const uint32_t bt = (uint32_t)first + (group >> log_side);
    const bool there = bt < all;
    const uint32_t at0 = there ? bt : 0;
    const int64_t b = at0 / (uint32_t)a.tokens, t = at0 - (uint32_t)b * (uint32_t)a.tokens;
    const QkTensor& x = a.in[kind];
    const QkTensor& y = a.out[kind];
    // Vectors this lane takes part in (a head of 80 values fills 10 of 16 lanes).
    const int h0 = piece * side * BATCH + which;
    const int count = there && e < a.d ? a.heads[kind] - h0 : 0;         // vector j is there when j * side < count
    int64_t from = b * x.batch_stride + t * x.token_stride + h0 * x.head_stride + e;
    int64_t to = b * y.batch_stride + t * y.token_stride + h0 * y.head_stride + e;

    Raw<BF16> v[BATCH];
    griddep_wait();
    griddep_launch_dependents();
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
        if (j * side < count) {
            v[j].load(x.data, from + j * side * x.head_stride);
        } else {
#pragma unroll
            for (int i = 0; i < Raw<BF16>::N; ++i) v[j].w[i] = 0;
        }
    }
    if (kind == 2) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (j * side < count) v[j].put(y.data, to + j * side * y.head_stride);
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
    // nothing and makes what it turns of the token's queries and keys NaN.
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
                const float4 cc = reinterpret_cast<const float4*>(a.cos + at)[i];
                const float4 ss = reinterpret_cast<const float4*>(a.sin + at)[i];
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

    float r[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
        r[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[j] = fmaf(v[j].get(i), v[j].get(i), r[j]);
    }
#pragma unroll
    for (int m = 1; m < LPV; m <<= 1) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) r[j] += __shfl_xor_sync(0xFFFFFFFFu, r[j], m);
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
        Raw<BF16> o;                                     // halves: the partner's values
        if (!INTER) {
            const int lp = lane + (partner - e) / 8;
#pragma unroll
            for (int i = 0; i < Raw<BF16>::N; ++i) o.w[i] = __shfl_sync(0xFFFFFFFFu, v[j].w[i], lp);
        }
        if (j * side < count) {
            const float rj = weight != nullptr ? rsqrtf(r[j] * a.inv_d + a.eps) : 1.f;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = v[j].get(i) * own[i];
                if (turns) f[i] = fmaf(INTER ? v[j].get(i ^ 1) : o.get(i), other[i], f[i]);
                f[i] *= rj;
            }
            Raw<BF16>::store(y.data, to + j * side * y.head_stride, f);
        }
    }
}

template <bool BF16, bool INTER, int LPV>
cudaError_t go(const QkArgs& a, cudaStream_t st) {
    constexpr int kGroups = 32 / LPV;
    const int64_t all = a.batch * a.tokens;
    QkPlan p{};
    int batch = 1;
    for (int i = 0; i < 3; ++i) {
        while ((1 << p.log_side[i]) < kGroups && (1 << p.log_side[i]) < a.heads[i]) ++p.log_side[i];
        while (batch < 4 && a.heads[i] > batch << p.log_side[i]) batch *= 2;
    }
    // Tensors with fewer heads have further tokens in a warp and leave the last blocks of x idle.
    int64_t blocks = 0;
    unsigned pieces = 0;
    for (int i = 0; i < 3; ++i) {
        const int heads = (1 << p.log_side[i]) * batch, tokens = kWarps * (kGroups >> p.log_side[i]);
        p.pieces[i] = (a.heads[i] + heads - 1) / heads;
        pieces += (unsigned)p.pieces[i];
        if (a.heads[i] > 0 && (all + tokens - 1) / tokens > blocks) blocks = (all + tokens - 1) / tokens;
    }
    const dim3 grid((unsigned)blocks, pieces);
    if (batch == 1) return launch_programmatic(qk_kernel<BF16, INTER, LPV, 1>, grid, 32 * kWarps, 0, st, a, p);
    if (batch == 2) return launch_programmatic(qk_kernel<BF16, INTER, LPV, 2>, grid, 32 * kWarps, 0, st, a, p);
    return launch_programmatic(qk_kernel<BF16, INTER, LPV, 4>, grid, 32 * kWarps, 0, st, a, p);
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
