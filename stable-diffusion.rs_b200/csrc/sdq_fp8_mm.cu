// sdq_fp8_mm.cu -- product of block-scaled e4m3 matrices on the tensor cores.
//
//   y[t, f] = resid + gate[f] * act( sum_kb xs[kb, t] ws[f/128, kb] sum_{k in kb} xq[t,k] wq[f,k] + bias[f] )
//
// The tile is D[f, t] = W[f, :] . X[t, :]^T: 128 features (MMA M) by BT tokens (MMA N), f32 in
// tensor memory.  One step is one scale block of K (128 values, 128 bytes): W's 128 rows and X's
// BT rows arrive by TMA with the 128-byte swizzle, four block-scaled MMAs (K = 32 each) consume
// them, and the scales are multiplied in by the tensor core, from tensor memory, where a warpgroup
// has laid them: row r of A has its byte in lane r % 32 of column r / 32 (and so for B), repeated
// in each of the four 32-lane quarters.  All four MMAs of a step use the same byte.
//
// Warp roles (384 threads, one CTA per SM, persistent over tiles):
//   warp 0       TMA producer of the operand ring
//   warp 1       tensor memory allocator and MMA issuer
//   warps 4-7    scale bytes: global -> registers (four steps ahead) -> tensor memory ring
//   warps 8-11   output stage: accumulator -> registers -> y, while the next tile accumulates in
//                the other buffer (BT <= 224)
// Every mbarrier wait is bounded; on expiry the kernel records a status bit, drains its own copies
// and MMAs, frees its tensor memory and returns.
#include <cstdint>
#include <cstring>
#include <cuda.h>
#include <cuda_runtime.h>

#include "sdq_dequant.cuh"
#include "sdq_epilogue.cuh"
#include "sdq_fp8.cuh"
#include "sdq_internal.h"
#include "sdq_ptx.cuh"

namespace sdq {

__device__ unsigned int g_fp8_status = 0;

namespace {

constexpr int kMmThreads = 384;

template <int BT>
struct MmCfg {
    static constexpr int BF = 128;                                 // features per tile
    static constexpr int W_STAGE = BF * kFp8Block;                 // bytes
    static constexpr int X_STAGE = BT * kFp8Block;
    static constexpr int STAGE = W_STAGE + X_STAGE;
    static constexpr int STAGES = (kQmvMaxSmem - 2048) / STAGE < 8 ? (kQmvMaxSmem - 2048) / STAGE : 8;
    static constexpr int D_BUFS = BT <= 224 ? 2 : 1;
    static constexpr int D_COLS = (BT + 31) / 32 * 32;             // columns of one accumulator
    static constexpr int SB_COLS = (BT + 127) / 128 * 4;           // columns of X's scales (a multiple of 4)
    static constexpr int SLOT = 4 + SB_COLS;                       // W's four, then X's
    static constexpr int SF_COL = D_BUFS * D_COLS;
    static constexpr int SLOTS = (512 - SF_COL) / SLOT < STAGES ? (512 - SF_COL) / SLOT : STAGES;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + 1024;
    static_assert(BT % 16 == 0 && BT >= 16 && BT <= 256, "MMA N");
    static_assert(SLOTS >= 3 && STAGES >= 3, "rings too short");
};

template <int BT, bool FUSED, bool YF32>
__global__ void __launch_bounds__(kMmThreads, 1)
    fp8_mm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                  const uint8_t* __restrict__ xs, const uint8_t* __restrict__ ws, const EpiArgs epi, void* y, int M,
                  int N, int K, int group) {
    using C = MmCfg<BT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);
    // Step s uses stage s % STAGES and scale slot s % SLOTS.
    uint64_t* full = bars;                       // operands landed            count 1 + tx
    uint64_t* done = full + C::STAGES;           // the step's MMAs finished   count 1 (commit); frees stage and slot
    uint64_t* sfull = done + C::STAGES;          // scale slot written         count 128
    uint64_t* dfull = sfull + C::SLOTS;          // accumulator complete       count 1 (commit)
    uint64_t* dempty = dfull + 2;                // accumulator drained        count 128
    uint64_t* drain = dempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    unsigned int* status = &g_fp8_status;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(full + i, 1); mbar_init(done + i, 1); }
        for (int i = 0; i < C::SLOTS; ++i) mbar_init(sfull + i, 128);
        for (int i = 0; i < 2; ++i) { mbar_init(dfull + i, 1); mbar_init(dempty + i, 128); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int KT = (K + kFp8Block - 1) / kFp8Block;
    const int nft = (N + C::BF - 1) / C::BF, ntt = (M + BT - 1) / BT, ntiles = nft * ntt;
    // Tiles go in groups of `group` token tiles: within a group, the tokens of one feature tile
    // first, so that the CTAs at work share W's tiles and the group's X stays in L2 while W
    // streams past it once per group.
    auto place = [&](int tile, int& ft, int& tt) {
        const int per = group * nft, g = tile / per, r = tile - g * per;
        const int h = ntt - g * group < group ? ntt - g * group : group;
        ft = r / h;
        tt = g * group + (r - ft * h);
    };

    if (warp == 0) {
        // ------------------------------------------------------------ operand producer
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            const bool withhold = g_withhold_first_copy != 0;      // testing hook, normally false
            for (int tile = blockIdx.x; ok && tile < ntiles; tile += gridDim.x) {
                int ft, tt;
                place(tile, ft, tt);
                for (int kt = 0; kt < KT; ++kt, ++it) {
                    const int s = it % C::STAGES;
                    if (!mbar_wait_sleep(done + s, ((it / C::STAGES) & 1) ^ 1, abort_flag, status, 1u, 20)) { ok = false; break; }
                    if (withhold && it == 0) continue;
                    mbar_arrive_expect_tx(full + s, C::STAGE);
                    tma_load_2d(smem + s * C::STAGE, &tmW, full + s, kt * kFp8Block, ft * C::BF);
                    tma_load_2d(smem + s * C::STAGE + C::W_STAGE, &tmX, full + s, kt * kFp8Block, tt * BT);
                }
            }
            // Whatever stopped the loop, no copy may outlive the CTA's shared memory: the last
            // STAGES steps that were started are waited for.
            if (!ok)
                for (int j = it - 1; j >= 0 && j >= it - C::STAGES; --j)
                    if (!(withhold && j == 0)) mbar_wait_drain(full + j % C::STAGES, (uint32_t)((j / C::STAGES) & 1));
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t idesc = idesc_mx_e4m3(C::BF, BT);
        int it = 0, tc = 0;
        bool ok = true, any = false;
        for (int tile = blockIdx.x; ok && tile < ntiles; tile += gridDim.x, ++tc) {
            const int buf = tc % C::D_BUFS;
            if (!mbar_wait_warp(dempty + buf, ((tc / C::D_BUFS) & 1) ^ 1, abort_flag, status, 2u)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d = tmem + buf * C::D_COLS;
            for (int kt = 0; kt < KT; ++kt, ++it) {
                const int s = it % C::STAGES, f = it % C::SLOTS;
                if (!mbar_wait_warp(sfull + f, (it / C::SLOTS) & 1, abort_flag, status, 2u) ||
                    !mbar_wait_warp(full + s, (it / C::STAGES) & 1, abort_flag, status, 2u)) { ok = false; break; }
                tc_fence_after();
                const uint64_t adesc = smem_desc_sw128(smem_u32(smem + s * C::STAGE));
                const uint64_t bdesc = smem_desc_sw128(smem_u32(smem + s * C::STAGE + C::W_STAGE));
                const uint32_t sf = tmem + C::SF_COL + f * C::SLOT;
                // Past the end of K both operands are zeros: whole MMAs of them are left out.
                const int nj = K - kt * kFp8Block < kFp8Block ? (K - kt * kFp8Block + 31) / 32 : 4;
                for (int j = 0; j < nj; ++j)
                    tc_mma_mx_elect(d, adesc + 2ull * j, bdesc + 2ull * j, idesc, sf, sf + 4, (kt | j) != 0);
                tc_commit_elect(done + s);
                any = true;
            }
            if (!ok) break;
            tc_commit_elect(dfull + buf);
        }
        if (!ok && any) {
            tc_commit_elect(drain);
            mbar_wait_drain(drain, 0);
        }
    } else if (warp >= 4 && warp < 8) {
        // ------------------------------------------------------------ scales
        // Lane l of each of the four warps holds, per step, W's scale (the same for all 128
        // features) and those of tokens l, l + 32, ...: the columns of its quarter.
        constexpr int NX = C::SB_COLS, AHEAD = 4;
        const uint32_t quarter = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        uint32_t next[AHEAD][NX + 1];
        auto fetch = [&](int tile, int kt0) {
            int ft, tt;
            place(tile, ft, tt);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int kt = kt0 + i;
                if (kt < KT) {
                    next[i][0] = __ldg(ws + (int64_t)ft * KT + kt);
                    const uint8_t* row = xs + (int64_t)kt * M;
#pragma unroll
                    for (int c = 0; c < NX; ++c) {
                        const int t = 32 * c + lane;
                        next[i][1 + c] = t < BT && (int64_t)tt * BT + t < M ? __ldg(row + (int64_t)tt * BT + t) : 127u;
                    }
                }
            }
        };
        int it = 0;
        bool ok = true;
        if ((int)blockIdx.x < ntiles) fetch(blockIdx.x, 0);
        for (int tile = blockIdx.x; ok && tile < ntiles; tile += gridDim.x) {
            for (int kt0 = 0; ok && kt0 < KT; kt0 += AHEAD) {
                uint32_t cur[AHEAD][NX + 1];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (int c = 0; c <= NX; ++c) cur[i][c] = next[i][c] * 0x01010101u;
                if (kt0 + AHEAD < KT) fetch(tile, kt0 + AHEAD);
                else if (tile + (int)gridDim.x < ntiles) fetch(tile + gridDim.x, 0);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    if (ok && kt0 + i < KT) {
                        const int f = it % C::SLOTS;
                        if (it >= C::SLOTS) {                        // the step that used the slot last
                            const int prev = it - C::SLOTS;
                            ok = mbar_wait_warp(done + prev % C::STAGES, (prev / C::STAGES) & 1, abort_flag, status, 4u);
                        }
                        if (ok) {
                            tc_fence_after();
                            const uint32_t at = tmem + quarter + C::SF_COL + f * C::SLOT;
                            tmem_st4(at, cur[i][0], cur[i][0], cur[i][0], cur[i][0]);
#pragma unroll
                            for (int c = 0; c < NX; c += 4)
                                tmem_st4(at + 4 + c, cur[i][1 + c], cur[i][2 + c], cur[i][3 + c], cur[i][4 + c]);
                            tc_wait_st();
                            tc_fence_before();
                            mbar_arrive(sfull + f);
                            ++it;
                        }
                    }
                }
            }
        }
    } else if (warp >= 8) {
        // ------------------------------------------------------------ output stage
        // Thread = feature: 16 tokens of the accumulator at a time.  A warp's 32 features are 64
        // (f32: 128) consecutive bytes of a token's row.
        const int fl = 32 * (warp & 3) + lane;
        const uint32_t quarter = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        int tc = 0;
        for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x, ++tc) {
            int ft, tt;
            place(tile, ft, tt);
            const int buf = tc % C::D_BUFS;
            const int f = ft * C::BF + fl;
            float badd = 0.f, gmul = 1.f;
            if (epi.bias != nullptr && f < N)
                badd = YF32 ? reinterpret_cast<const float*>(epi.bias)[f] : bf16_bits_to_f32(epi.bias[f]);
            if (FUSED && epi.gate != nullptr && f < N) gmul = bf16_bits_to_f32(epi.gate[f]);
            if (!__all_sync(0xffffffffu, mbar_wait_sleep(dfull + buf, (tc / C::D_BUFS) & 1, abort_flag, status, 8u, 64))) break;
            tc_fence_after();
            const int64_t t0 = (int64_t)tt * BT;
            for (int c = 0; c < BT / 16; ++c) {
                uint32_t v[16];
                __syncwarp();
                tmem_ld16(tmem + quarter + buf * C::D_COLS + 16 * c, v);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int64_t t = t0 + 16 * c + j;
                    if (t < M && f < N) {
                        float a = __uint_as_float(v[j]) + badd;
                        if (FUSED) {
                            a = epi_activation(a, epi.act) * gmul;
                            if (epi.resid != nullptr) a += bf16_bits_to_f32(epi.resid[t * N + f]);
                        }
                        if (YF32) static_cast<float*>(y)[t * N + f] = a;
                        else static_cast<uint16_t*>(y)[t * N + f] = (uint16_t)(pack_bf16x2(a, 0.f) & 0xFFFFu);
                    }
                }
            }
            __syncwarp();
            tc_fence_before();
            mbar_arrive(dempty + buf);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------- host side
bool byte_map(CUtensorMap* map, const uint8_t* p, int64_t rows, int64_t k, int box_rows) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)k};
    cuuint32_t box[2] = {(cuuint32_t)kFp8Block, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BT, bool FUSED, bool YF32>
cudaError_t launch_mm_t(const uint8_t* xq, const uint8_t* xs, int64_t m, int64_t k, const uint8_t* wq,
                        const uint8_t* ws, int64_t n, const EpiArgs& epi, void* y, cudaStream_t st, const char** msg) {
    using C = MmCfg<BT>;
    CUtensorMap tmX, tmW;
    if (!byte_map(&tmX, xq, m, k, BT) || !byte_map(&tmW, wq, n, k, C::BF)) {
        *msg = "cuTensorMapEncodeTiled rejected an fp8 operand's tensor map";
        return cudaErrorInvalidValue;
    }
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static bool configured[64] = {};
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        e = cudaFuncSetAttribute(fp8_mm_kernel<BT, FUSED, YF32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    const int64_t nft = (n + C::BF - 1) / C::BF, ntt = (m + BT - 1) / BT, tiles = nft * ntt;
    const int64_t fit = (32ll << 20) / ((int64_t)BT * k);          // token tiles whose X is 32 MB
    const int64_t group = fit < 1 ? 1 : (fit < ntt ? fit : ntt);
    const int grid = (int)(tiles < num_sms() ? tiles : num_sms());
    fp8_mm_kernel<BT, FUSED, YF32><<<grid, kMmThreads, C::SMEM, st>>>(tmX, tmW, xs, ws, epi, y, (int)m, (int)n, (int)k,
                                                                      (int)group);
    return cudaGetLastError();
}

template <int BT>
cudaError_t launch_mm_f(const uint8_t* xq, const uint8_t* xs, int64_t m, int64_t k, const uint8_t* wq,
                        const uint8_t* ws, int64_t n, const EpiArgs& epi, void* y, cudaStream_t st, const char** msg) {
    if (epi.fused()) return launch_mm_t<BT, true, false>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
    if (epi.f32) return launch_mm_t<BT, false, true>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
    return launch_mm_t<BT, false, false>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
}

}  // namespace

cudaError_t launch_fp8_mm(const uint8_t* xq, const uint8_t* xs, int64_t m, int64_t k, const uint8_t* wq,
                          const uint8_t* ws, int64_t n, const EpiArgs& epi, void* y, cudaStream_t st,
                          const char** msg) {
    if (m <= 16) return launch_mm_f<16>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
    if (m <= 64) return launch_mm_f<64>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
    if (m <= 128) return launch_mm_f<128>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
    return launch_mm_f<224>(xq, xs, m, k, wq, ws, n, epi, y, st, msg);
}

cudaError_t read_and_clear_fp8_status(unsigned int* out, cudaStream_t st) {
    cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_fp8_status, sizeof(unsigned int), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && *out != 0) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbolAsync(g_fp8_status, &zero, sizeof(unsigned int), 0, cudaMemcpyHostToDevice, st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    }
    return e;
}

cudaError_t set_wait_hook_fp8(unsigned long long limit_ns, int withhold, cudaStream_t st) {
    cudaError_t e = cudaMemcpyToSymbolAsync(g_wait_limit_ns, &limit_ns, sizeof(limit_ns), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess)
        e = cudaMemcpyToSymbolAsync(g_withhold_first_copy, &withhold, sizeof(withhold), 0, cudaMemcpyHostToDevice, st);
    return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}

}  // namespace sdq
