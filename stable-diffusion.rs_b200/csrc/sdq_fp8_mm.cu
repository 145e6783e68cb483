// sdq_fp8_mm.cu -- product of block-scaled e4m3 matrices on the tensor cores.
//
//   y[t, f] = resid + gate[f] * act( sum_kb xs[kb, t] ws[f/128, kb] sum_{k in kb} xq[t,k] wq[f,k] + bias[f] )
//
// A tile is 128 tokens (MMA M; 256 for a CTA pair, 128 in each) by `bn` features (MMA N, 16 .. 224),
// f32 in tensor memory, double-buffered.  One step is one scale block of K: 128 values, 128 bytes.
// X's rows and W's rows (a pair's CTAs load half of W's each) arrive by TMA with the 128-byte
// swizzle; four block-scaled MMAs (K = 32) consume them.  The tensor core multiplies the scales in
// from tensor memory: row r of an operand has its scale in lane r % 32 of column r / 32, the same
// in each of the four 32-lane quarters; the four bytes of a 32-bit cell are the scales of four
// consecutive steps, chosen by the instruction, so they are laid once for 512 values of K.
//
// Tokens lie on the lanes, so that a thread of the output stage holds consecutive features of one
// token and stores whole 32-byte sectors.  (The other way round each thread held one feature and
// stored 2 bytes a time, which cost more than the product at K = 4096.)
//
// Where the tiles leave SMs idle and K is long, a cluster of 2, 4 or 8 CTAs shares one tile's K (SPLIT):
// each accumulates its steps, then they exchange pieces of 16 features through one another's shared
// memory, each adding up (in the order of K) and storing its own.  1 x 9728 x 2560: 14.8 -> 9.2 us.
//
// One kernel for every number of tokens.  For a few of them a stream of the weight through mma.sync
// was measured beside it and is not kept: its e4m3 form is emulated on sm_100a (170 cycles each), and
// with the codes turned into f16 the conversion sets the pace (1 x 2560 x 9728: 14.3 us by the
// conversion instruction, 18.7 by shifts, 7.1 here, where nothing is unpacked).
//
// Warp roles (512 threads, one CTA per SM, persistent over tiles):
//   warp 0       TMA producer of the operand ring (one thread)
//   warp 1       tensor memory allocator and MMA issuer (one thread; in a pair, rank 0's)
//   warps 4-7    scale bytes: global -> registers, four groups ahead -> shared memory
//   warps 8-15   output stage, two groups of four warps, a half of the tile's features each
// Every mbarrier wait is bounded; on expiry the kernel records a status bit, waits for its own
// copies and MMAs, frees its tensor memory and returns.
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

constexpr int kMmThreads = 512;
constexpr int kTokens = 128;                       // per CTA
constexpr int kMaxBn = 224;                        // two accumulators and the scales fill 512 columns
constexpr int kXStage = kTokens * kFp8Block;       // bytes
constexpr int kMaxStages = 12;
constexpr int kSlots = 4;                          // scale groups in tensor memory, one for each scale warp
constexpr int kCells = 3 * 512;                    // bytes of a group's scales in shared memory
static_assert(2 * kMaxBn + kSlots * 12 <= 512, "tensor memory");
constexpr int kMaxPitch = 43;                      // words per token of a warp's transposing buffer
constexpr int kFixedSmem = 1024 /* alignment */ + 512 /* barriers */ + 4 * 256 * 4 /* two tiles' bias and gate */ +
                           kSlots * kCells;
constexpr int kTransposeSmem = 8 * 32 * kMaxPitch * 4;
constexpr size_t fixed_smem(bool aligned) { return kFixedSmem + (aligned ? 0 : kTransposeSmem); }

// Quotients of numbers below 2^31 by a settled divisor d, 2^(l-1) < d <= 2^l: n / d is the upper half of
// n * ceil(2^(31+l) / d), l - 1 places down.  (A tile's place took 400 cycles by division.)
struct Divisor {
    uint32_t mul, shift;
    Divisor(uint32_t d = 1) {
        uint32_t l = 0;
        while ((1ull << l) < d) ++l;
        mul = l == 0 ? 0 : (uint32_t)(((1ull << (31 + l)) + d - 1) / d);      // d = 1: n itself
        shift = l == 0 ? 0 : l - 1;
    }
    __device__ __forceinline__ int of(int n) const { return mul == 0 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
};

// What the host has settled for a launch.
struct MmPlan {
    int m, n, k;
    int kt;                // steps: blocks of K
    int bn;                // features per tile
    int nft, ntt;          // feature tiles, token tiles
    int stages;            // ring depth
    int group;             // token tiles that are walked together (see place)
    Divisor by_tiles, by_group, by_rest;   // group * nft; group; the last group's token tiles
    int split;             // CTAs that share a tile's K
    int x_rows;            // rows of X a CTA loads (128, or M rounded up to 8)
    int aligned;           // rows of y (and resid) start on 32 bytes and hold whole 16-feature pieces
    int resid_like_y;      // resid lies at y's offset within 16 bytes
    int pitch;             // of the transposing buffer
};

__device__ __forceinline__ uint64_t pack2(float2 a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)), "l"(pack2(c)));
    return unpack2(r);
}
// Both activations are a / (1 + 2^x): SiLU with x = -a log2 e, GELU (tanh form), a (1 + tanh u) / 2 with
// u = sqrt(2/pi) (a + 0.044715 a^3), with x = -2u log2 e.  Nothing cancels, so a value keeps its relative
// accuracy.  (1 + tanh u by the hardware's tanh does: at a = -4 its 2^-11 is fourteen times 1 + tanh u.
// It takes two special functions for two values, this three: GELU of 3116 x 48 x 4176 15.4 us, 16.9 here, and
// 18.2 with a reciprocal for each value, which needs no LEAST.)
// For two values, with the hardware's exponential and one reciprocal for both, 1 / d0 = d1 (1 / (d0 d1)):
// the special function unit sets the output stage's pace.  So that the product stays finite an a below LEAST,
// where 2^x is 2^62, stands for LEAST; the value there is under 10^-17 either way.
template <class F>
__device__ __forceinline__ float2 over_one_plus_exp2(float2 a, float least, F exponent) {
    float2 d = exponent(make_float2(fmaxf(a.x, least), fmaxf(a.y, least)));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a.x) : "f"(least));         // a NaN stays, but out of d, which the two share
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a.y) : "f"(least));
    float r;
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d.y));
    d = add2(d, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d.x * d.y));
    return mul2(a, mul2(make_float2(d.y, d.x), make_float2(r, r)));
}
__device__ __forceinline__ float2 gelu2(float2 a) {
    return over_one_plus_exp2(a, -7.6f, [](float2 v) {
        const float c = -2.f * 0.7978845608028654f * 1.4426950408889634f, k = 0.044715f * c;
        return mul2(v, fma2(mul2(v, v), make_float2(k, k), make_float2(c, c)));
    });
}
__device__ __forceinline__ float2 silu2(float2 a) {
    return over_one_plus_exp2(a, -43.f, [](float2 v) { return mul2(v, make_float2(-1.4426950408889634f, -1.4426950408889634f)); });
}
// The activation of N pairs of values; one decision a piece, not one a value.
template <int N>
__device__ __forceinline__ void activate(float2 (&o)[N], int act) {
    if (act == SDQ_ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = gelu2(o[j]);
    } else if (act == SDQ_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = silu2(o[j]);
    }
}

// ANY: rows of y that do not start on 32 bytes (a kernel of its own: the two output stages in one cost
// the aligned one 3 %).
template <bool PAIR, bool SPLIT, bool FUSED, bool YF32, bool ANY>
__global__ void __launch_bounds__(kMmThreads, 1)
    fp8_mm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                  const uint8_t* xs, const uint8_t* ws, const EpiArgs epi, void* y,
                  const __grid_constant__ MmPlan p) {
    constexpr int CG = PAIR ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    // (An offset, not a cast of the rounded address: from that the compiler made generic accesses.)
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const int w_rows = p.bn / CG;                               // rows of W this CTA loads
    const int stage_bytes = kXStage + w_rows * kFp8Block;       // both parts multiples of 1024
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.stages * stage_bytes);
    // Step s uses stage s % stages; a group of up to four steps of a tile uses one scale slot.
    uint64_t* full = bars;                       // operands of the pair landed   count 1 + tx
    uint64_t* done = full + kMaxStages;          // the step's MMAs finished      count 1 (commit); frees the stage
    uint64_t* sfull = done + kMaxStages;         // a group's scales in smem      count CG
    uint64_t* sempty = sfull + kSlots;        // the group's MMAs finished     count 1 (commit); frees the slot
    uint64_t* dfull = sempty + kSlots;        // accumulator complete          count 1 (commit)
    uint64_t* dempty = dfull + 2;                // accumulator drained           count 8 (a warp each) x CG
    uint64_t* drain = dempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* started = reinterpret_cast<int*>(tmem_slot + 2);       // steps whose copies this CTA has issued
    float* sbias = reinterpret_cast<float*>(bars + 64);         // [2][256], a tile's in turn
    float* sgate = sbias + 512;                                 // [2][256]
    // [slots][3 column quads][32 lanes][4 columns][4 steps], X's quad first
    uint8_t* sscale = reinterpret_cast<uint8_t*>(sgate + 512);
    float* stage32 = reinterpret_cast<float*>(sscale + kSlots * kCells);    // the transposing buffers, if any
    unsigned int* status = &g_fp8_status;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const int hook = g_withhold_first_copy;      // testing hook, normally 0; read here, where nothing waits for it yet
    const bool withhold = PAIR ? hook == 1 : hook != 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) { mbar_init(full + i, 1); mbar_init(done + i, 1); }
        for (int i = 0; i < kSlots; ++i) { mbar_init(sfull + i, CG); mbar_init(sempty + i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(dfull + i, 1); mbar_init(dempty + i, 8 * CG); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
    }
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(tmem_slot, 512);
        } else {
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();                    // the peer's barriers are initialised too
    tc_fence_after();
    // Launched with programmatic stream serialisation: all of the above may run while the kernel
    // before this one finishes; nothing that it may have written is read, and nothing is written,
    // before this.
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tmem = *tmem_slot;

    // This CTA's steps: all of them, or its share of the cluster's.
    const int share = SPLIT ? (int)cluster_rank() : 0;
    const int kbase = SPLIT ? p.kt * share / p.split : 0, KT = SPLIT ? p.kt * (share + 1) / p.split - kbase : p.kt;
    const int d_cols = (p.bn + 31) / 32 * 32, sf_col = 2 * d_cols;
    const int sb_cols = (p.bn + 127) / 128 * 4, slot_cols = 4 + sb_cols;   // X's four columns, then W's
    const int nft = p.nft, ntt = p.ntt, ntiles = nft * ntt;
    const int per_tile_ctas = SPLIT ? p.split : CG;
    const int first = blockIdx.x / per_tile_ctas, stride = gridDim.x / per_tile_ctas;
    // Tiles go in groups of `group` token tiles; within a group, the tokens of one feature tile
    // first.  So the CTAs at work share W's rows, and the group's X stays in L2 while W streams
    // past it once per group.
    auto place = [&](int tile, int& ft, int& tt) {
        const int g = p.by_tiles.of(tile), r = tile - g * p.group * nft;
        const int h = ntt - g * p.group < p.group ? ntt - g * p.group : p.group;
        ft = h == p.group ? p.by_group.of(r) : p.by_rest.of(r);
        tt = g * p.group + (r - ft * h);
    };

    // The bias and gate of a tile, a feature for each of the output stage's 256 threads: fetched a tile
    // ahead, then put into shared memory as f32 (half b of sbias and sgate).  (Fetched when the tile
    // began, they took 900 cycles of a tile whose output is 3500.)
    uint32_t bias_bits = 0, gate_bits = 0x3F80;  // as loaded: a conversion would wait for the load
    auto fetch_bias = [&](int tile) {
        int ft, tt;
        place(tile, ft, tt);
        const int i = threadIdx.x - 256, f = ft * p.bn + i;
        if (i < p.bn && f < p.n) {
            if (epi.bias != nullptr) bias_bits = YF32 ? reinterpret_cast<const uint32_t*>(epi.bias)[f] : epi.bias[f];
            if (FUSED && epi.gate != nullptr) gate_bits = epi.gate[f];
        }
    };
    auto put_bias = [&](int b) {
        const int i = 256 * b + threadIdx.x - 256;
        sbias[i] = YF32 ? __uint_as_float(bias_bits) : bf16_bits_to_f32(bias_bits);
        if (FUSED) sgate[i] = bf16_bits_to_f32(gate_bits);
    };
    bool complete = false;                       // SPLIT: this warp has seen the accumulator complete
    if (warp == 0) {
        // ------------------------------------------------------------ operand producer
        if (elect_one()) {
            const uint32_t my_bytes = (uint32_t)((p.x_rows + w_rows) * kFp8Block);
            const uint32_t full0 = PAIR ? cluster_addr(full, 0) : 0;
            int it = 0, s = 0;
            uint32_t phase = 1;
            bool ok = !(PAIR && hook == (rank == 0 ? 3 : 2));
            for (int tile = first; ok && tile < ntiles; tile += stride) {
                int ft, tt;
                place(tile, ft, tt);
                const int xr = (tt * CG + (int)rank) * kTokens, wr = ft * p.bn + (int)rank * w_rows;
                for (int kt = 0; kt < KT; ++kt, ++it) {
                    if (!mbar_wait(done + s, phase, abort_flag, status, 1u)) { ok = false; break; }
                    uint8_t* at = smem + s * stage_bytes;
                    if (!(withhold && it == 0)) {
                        if (PAIR) {
                            if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * my_bytes);
                            tma_load_2d_pair(at, &tmX, full0 + 8 * s, kt * kFp8Block, xr);
                            tma_load_2d_pair(at + kXStage, &tmW, full0 + 8 * s, kt * kFp8Block, wr);
                        } else {
                            mbar_arrive_expect_tx(full + s, my_bytes);
                            tma_load_2d(at, &tmX, full + s, (kbase + kt) * kFp8Block, xr);
                            tma_load_2d(at + kXStage, &tmW, full + s, (kbase + kt) * kFp8Block, wr);
                        }
                    }
                    if (++s == p.stages) { s = 0; phase ^= 1; }
                }
            }
            *started = it;
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        // One thread does all of it: one wait, four MMAs and one commit per step.  (The whole warp
        // waiting and an election per MMA took 820 cycles a step, whatever the tile's width.)
        if (rank == 0 && elect_one()) {
            const uint32_t idesc0 = idesc_mx_e4m3(CG * kTokens, p.bn);
            const uint64_t adesc0 = smem_desc_sw128(smem_u32(smem));
            auto commit = [&](uint64_t* bar) {
                if (PAIR) tc_commit_pair(bar);
                else tc_commit(bar);
            };
            int s = 0, slot = 0, tc = 0;
            uint32_t phase = 0, sphase = 0;
            bool ok = true, any = false;
            for (int tile = first; ok && tile < ntiles; tile += stride, ++tc) {
                const int buf = tc & 1;
                if (!mbar_wait(dempty + buf, ((tc >> 1) & 1) ^ 1, abort_flag, status, 2u)) { ok = false; break; }
                const uint32_t d = tmem + buf * d_cols;
                for (int kt0 = 0; kt0 < KT; kt0 += 4) {
                    if (!mbar_wait(sfull + slot, sphase, abort_flag, status, 2u)) { ok = false; break; }
                    const uint32_t sf = tmem + sf_col + slot * slot_cols;
                    const uint64_t cells = smem_desc_rows16(smem_u32(sscale + slot * kCells));
                    tc_cp_32x16_x4<PAIR>(sf, cells);
                    tc_cp_32x16_x4<PAIR>(sf + 4, cells + 32);
                    if (sb_cols > 4) tc_cp_32x16_x4<PAIR>(sf + 8, cells + 64);
                    const int left = p.k - (kbase + kt0) * kFp8Block;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (kt0 + q >= KT) break;
                        if (!mbar_wait(full + s, phase, abort_flag, status, 2u)) { ok = false; break; }
                        tc_fence_after();
                        const uint64_t adesc = adesc0 + (uint32_t)(s * (stage_bytes >> 4));
                        const uint64_t bdesc = adesc + (kXStage >> 4);
                        const uint32_t idesc = idesc0 | ((uint32_t)q << 29) | ((uint32_t)q << 4);   // scale byte q of A and B
                        // A 32-value piece is 32 bytes along the swizzled rows: +2 in the
                        // descriptors' 16-byte units.  Pieces past the end of K are zeros: left out.
                        tc_mma_mx<PAIR>(d, adesc, bdesc, idesc, sf, sf + 4, q != 0 || kt0 != 0);
                        if (left > q * kFp8Block + 32) tc_mma_mx<PAIR>(d, adesc + 2, bdesc + 2, idesc, sf, sf + 4, 1);
                        if (left > q * kFp8Block + 64) tc_mma_mx<PAIR>(d, adesc + 4, bdesc + 4, idesc, sf, sf + 4, 1);
                        if (left > q * kFp8Block + 96) tc_mma_mx<PAIR>(d, adesc + 6, bdesc + 6, idesc, sf, sf + 4, 1);
                        commit(done + s);
                        any = true;
                        if (++s == p.stages) { s = 0; phase ^= 1; }
                    }
                    if (!ok) break;
                    commit(sempty + slot);
                    if (++slot == kSlots) { slot = 0; sphase ^= 1; }
                }
                if (!ok) break;
                commit(dfull + buf);
            }
            if (!ok && any) {
                commit(drain);
                mbar_wait_drain(drain, 0);
            }
        }
    } else if (warp >= 4 && warp < 8) {
        // ------------------------------------------------------------ scales
        // Warp w lays groups w, w + 4, ... of the CTA's steps, all in scale slot w: lane l fetches
        // the bytes of rows l, l + 32, ... (X's 128 rows of this CTA, and W's bn, all of them in each
        // CTA of a pair) for the group's four steps and puts them into the slot's cells in shared
        // memory; the MMA thread has them copied to tensor memory in order with its MMAs.  A fence or
        // an arrival waits for the loads before it, so a warp has the time of four groups for one
        // (when the four worked on every group together, that latency set the pace of the MMAs).
        const uint32_t sfull0 = PAIR ? cluster_addr(sfull, 0) : 0;
        const int w = warp & 3, per_tile = (KT + 3) / 4;
        const int groups = first < ntiles ? ((ntiles - 1 - first) / stride + 1) * per_tile : 0;
        uint32_t raw[48];
        // Rows and steps that are not there read the last one's byte: what it scales is never stored
        // or never multiplied, and loads without conditions all issue at once (48 guarded ones took
        // 2600 cycles to).
        auto fetch = [&](int g) {
            const int i = g / per_tile, kt0 = 4 * (g - i * per_tile);
            int ft, tt;
            place(first + i * stride, ft, tt);
            const int t = (tt * CG + (int)rank) * kTokens + lane, f = ft * p.bn + lane;
            int step[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) step[q] = kt0 + q < KT ? q : KT - 1 - kt0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint8_t* x = xs + (int64_t)(kbase + kt0) * p.m + (t + 32 * c < p.m ? t + 32 * c : p.m - 1);
#pragma unroll
                for (int q = 0; q < 4; ++q) raw[4 * c + q] = x[(int64_t)step[q] * p.m];
            }
#pragma unroll
            for (int c = 4; c < 12; ++c) {
                if (c >= 8 && sb_cols == 4) break;
                const int fc = f + 32 * (c - 4) < p.n ? f + 32 * (c - 4) : p.n - 1;
                const uint8_t* row = ws + (int64_t)(fc / kFp8Block) * p.kt + kbase + kt0;
#pragma unroll
                for (int q = 0; q < 4; ++q) raw[4 * c + q] = row[step[q]];
            }
        };
#pragma unroll
        for (int c = 0; c < 48; ++c) raw[c] = 0;
        uint32_t phase = 1;
        if (w < groups) fetch(w);
        for (int g = w; g < groups; g += kSlots, phase ^= 1) {
            if (!mbar_wait_warp(sempty + w, phase, abort_flag, status, 4u)) break;
            uint4* cells = reinterpret_cast<uint4*>(sscale + w * kCells) + lane;
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t* b = raw + 4 * (4 * c + j);
                    o[j] = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
                }
                cells[32 * c] = make_uint4(o[0], o[1], o[2], o[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_at(sfull0 + 8 * w);
                else mbar_arrive(sfull + w);
            }
            if (g + kSlots < groups) fetch(g + kSlots);
        }
    } else if (SPLIT && warp >= 8) {
        fetch_bias(first);
        put_bias(0);
        complete = __all_sync(0xffffffffu, mbar_wait_sleep(dfull, 0, abort_flag, status, 8u, 32));
    } else if (warp >= 8) {
        // ------------------------------------------------------------ output stage
        // Thread = token (its quarter of the lanes); group e of four warps takes one half of the tile's
        // features, 32 at a time.
        const int e = (warp - 8) >> 2;
        const uint32_t quarter = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t dempty0 = PAIR ? cluster_addr(dempty, 0) : 0;
        const bool resid = FUSED && epi.resid != nullptr;
        // Rows that do not start on 32 bytes: the warp turns 32 tokens x 32 features around in shared
        // memory, and a lane stores a chunk, the CHUNK values of an aligned 16 bytes of y; LANES lanes
        // take a token's piece.  What is over of a piece (row t's chunks start `over` values before
        // feature c) waits for the next one in front of it.  What the half's ends leave of a chunk is
        // stored by a lane a token.  (All of it by 2 bytes a lane, 64 bytes of a token a warp,
        // took much longer: 3907 x 320 x 8597 with gate and residual 112 us, 65 this way.)
        constexpr int CHUNK = YF32 ? 4 : 8, LANES = 32 / CHUNK, TOKENS = 32 / LANES;
        float* mine = stage32 + (warp - 8) * 32 * kMaxPitch;
        const uint32_t y_off = (uint32_t)(reinterpret_cast<uintptr_t>(y) / (YF32 ? 4 : 2));
        // The residual tile on its way to L2, a tile ahead: group e, sixteen of the warp's rows, four
        // lanes a row, 64 features (128 bytes) each.
        auto prefetch_resid = [&](int tile) {
            int ft, tt;
            place(tile, ft, tt);
            const int left = p.n - ft * p.bn < p.bn ? p.n - ft * p.bn : p.bn;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = (tt * CG + (int)rank) * kTokens + 32 * (warp & 3) + 16 * e + 8 * i + (lane >> 2), c = 64 * (lane & 3);
                if (c < left && t < p.m) prefetch_l2(epi.resid + (int64_t)t * p.n + ft * p.bn + c);
            }
        };
        if (first < ntiles) {
            fetch_bias(first);
            if (resid) prefetch_resid(first);
        }
        int tc = 0;
        for (int tile = first; tile < ntiles; tile += stride, ++tc) {
            int ft, tt;
            place(tile, ft, tt);
            const int buf = tc & 1, f0 = ft * p.bn;
            const int width = p.n - f0 < p.bn ? p.n - f0 : p.bn;
            const int half = (width + 63) / 64 * 32, h0 = e * half, h1 = e == 0 && half < width ? half : width;
            const int row0 = (tt * CG + (int)rank) * kTokens + 32 * (warp & 3);      // the warp's first token
            const int row = row0 + lane, rows = p.m - row0 < 32 ? p.m - row0 : 32;
            put_bias(buf);                                          // read by all after the barrier below
            if (tile + stride < ntiles) {
                fetch_bias(tile + stride);
                if (resid) prefetch_resid(tile + stride);
            }
            // How many values before a piece's first feature token t's first chunk of it starts.
            auto over = [&](int t) { return (int)((y_off + (uint32_t)(row0 + t) * (uint32_t)p.n) & (CHUNK - 1)); };
            // The residual of a piece: 32 features of this thread's token, or those of its chunks.  The
            // first piece's is fetched while the accumulator fills.
            uint32_t r[16];
            auto fetch_resid = [&](int c) {
                if (!ANY) {
                    if (row < p.m) {
                        const uint16_t* from = epi.resid + (int64_t)row * p.n + f0 + c;
                        ld_global_32(reinterpret_cast<uint32_t(&)[8]>(r[0]), from);
                        if (h1 - c > 16) ld_global_32(reinterpret_cast<uint32_t(&)[8]>(r[8]), from + 16);
                    }
                } else if (p.resid_like_y) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int t = TOKENS * u + lane / LANES, cs = c - over(t) + CHUNK * (lane % LANES);
                        if (t < rows && cs >= h0 && cs + CHUNK <= h1) {
                            const uint4 z = *reinterpret_cast<const uint4*>(epi.resid + (int64_t)(row0 + t) * p.n + f0 + cs);
                            r[4 * u] = z.x; r[4 * u + 1] = z.y; r[4 * u + 2] = z.z; r[4 * u + 3] = z.w;
                        }
                    }
                }
            };
            // `count` < CHUNK values of this thread's token from feature c on, up to a chunk's start (`head`) or
            // from one on: as 2, 4 and 8 bytes, each as far as it is due.
            auto put_cut = [&](int c, int count, float* from, bool head) {
                const int64_t at = (int64_t)row * p.n + f0 + c;
                if (YF32) {
                    float* to = static_cast<float*>(y) + at;
                    const int e4 = head ? 0 : count & 2, e8 = head ? count & 1 : 0;
                    if (count & 1) to[e4] = from[e4];
                    if (count & 2) *reinterpret_cast<float2*>(to + e8) = make_float2(from[e8], from[e8 + 1]);
                } else {
                    uint16_t* to = static_cast<uint16_t*>(y) + at;
                    const uint16_t* add = epi.resid + at;
                    const int e2 = head ? 0 : count & 6, e4 = head ? count & 1 : count & 4, e8 = head ? count & 3 : 0;
                    const bool wide = resid && p.resid_like_y;
                    uint32_t r2 = 0, r4 = 0;
                    uint2 r8 = make_uint2(0, 0);
                    if (wide) {
                        if (count & 1) r2 = add[e2];
                        if (count & 2) r4 = *reinterpret_cast<const uint32_t*>(add + e4);
                        if (count & 4) r8 = *reinterpret_cast<const uint2*>(add + e8);
                    } else if (resid) {
#pragma unroll 1
                        for (int j = 0; j < count; ++j) from[j] += bf16_bits_to_f32(add[j]);
                    }
                    auto two = [&](int e, uint32_t r) {
                        float2 z = make_float2(from[e], from[e + 1]);
                        if (wide) z = add2(z, make_float2(bf16_bits_to_f32(r & 0xFFFFu), bf16_bits_to_f32(r >> 16)));
                        return pack_bf16x2(z.x, z.y);
                    };
                    if (count & 1) to[e2] = (uint16_t)(pack_bf16x2(wide ? from[e2] + bf16_bits_to_f32(r2) : from[e2], 0.f) & 0xFFFFu);
                    if (count & 2) *reinterpret_cast<uint32_t*>(to + e4) = two(e4, r4);
                    if (count & 4) *reinterpret_cast<uint2*>(to + e8) = make_uint2(two(e8, r8.x), two(e8 + 2, r8.y));
                }
            };
            if (resid && row0 < p.m && h0 < h1) fetch_resid(h0);
            const bool ok = __all_sync(0xffffffffu, mbar_wait_sleep(dfull + buf, (tc >> 1) & 1, abort_flag, status, 8u, 32));
            // All eight warps go on or none does: none is left at a barrier.
            if (!named_barrier_and(1, 256, ok)) break;
            tc_fence_after();
            if (row0 < p.m) {                                       // warps of tokens that are not there rest
                const uint32_t acc = tmem + quarter + buf * d_cols;
                for (int c = h0; c < h1; c += 32) {
                    if (resid && c != h0) fetch_resid(c);
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(acc + c, v);
                    tc_wait_ld();
                    float2 o[16];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float4 b = *reinterpret_cast<const float4*>(sbias + 256 * buf + c + 2 * j);
                        o[j] = add2(make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), make_float2(b.x, b.y));
                        o[j + 1] = add2(make_float2(__uint_as_float(v[2 * j + 2]), __uint_as_float(v[2 * j + 3])), make_float2(b.z, b.w));
                    }
                    if (FUSED) {
                        activate(o, epi.act);
                        if (epi.gate != nullptr) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = mul2(o[j], *reinterpret_cast<const float2*>(sgate + 256 * buf + c + 2 * j));
                        }
                    }
                    if constexpr (!ANY) {
                        const int64_t at = (int64_t)row * p.n + f0 + c;
                        if (row < p.m) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (h == 1 && h1 - c <= 16) break;  // 32 features of this piece, or 16
                                uint32_t w[8];
                                if (YF32) {
#pragma unroll
                                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                                        for (int j = 0; j < 4; ++j) {
                                            w[2 * j] = __float_as_uint(o[8 * h + 4 * u + j].x);
                                            w[2 * j + 1] = __float_as_uint(o[8 * h + 4 * u + j].y);
                                        }
                                        st_global_32(static_cast<float*>(y) + at + 16 * h + 8 * u, w);
                                    }
                                } else {
#pragma unroll
                                    for (int j = 0; j < 8; ++j) {
                                        float2 z = o[8 * h + j];
                                        if (resid)
                                            z = add2(z, make_float2(bf16_bits_to_f32(r[8 * h + j] & 0xFFFFu),
                                                                    bf16_bits_to_f32(r[8 * h + j] >> 16)));
                                        w[j] = pack_bf16x2(z.x, z.y);
                                    }
                                    st_global_32(static_cast<uint16_t*>(y) + at + 16 * h, w);
                                }
                            }
                        }
                    } else {
                        float* to = mine + lane * p.pitch;          // [CHUNK of the last piece, 32]
                        __syncwarp();
                        if (c != h0) {
#pragma unroll
                            for (int j = 0; j < CHUNK; ++j) to[j] = to[32 + j];
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            to[CHUNK + 2 * j] = o[j].x;
                            to[CHUNK + 2 * j + 1] = o[j].y;
                        }
                        __syncwarp();
#pragma unroll
                        for (int u = 0; u < LANES; ++u) {
                            const int t = TOKENS * u + lane / LANES, before = over(t), i = CHUNK * (lane % LANES);
                            const int cs = c - before + i;
                            if (t < rows && cs >= h0 && cs + CHUNK <= h1) {
                                const float* from = mine + t * p.pitch + CHUNK - before + i;
                                const int64_t at = (int64_t)(row0 + t) * p.n + f0 + cs;
                                float z[CHUNK];
                                uint32_t w[4];
#pragma unroll
                                for (int j = 0; j < CHUNK; ++j) z[j] = from[j];
                                if (resid) {
#pragma unroll
                                    for (int j = 0; j < CHUNK; ++j)
                                        z[j] += !p.resid_like_y ? bf16_bits_to_f32(epi.resid[at + j])
                                                : bf16_bits_to_f32(j & 1 ? r[(4 * u + j / 2) & 15] >> 16 : r[(4 * u + j / 2) & 15] & 0xFFFFu);
                                }
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    w[j] = YF32 ? __float_as_uint(z[j]) : pack_bf16x2(z[(2 * j) % CHUNK], z[(2 * j + 1) % CHUNK]);
                                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(y) + at * (16 / CHUNK)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                        // Of this thread's token, values before the half's first chunk, and where the last one ends.
                        const int mine_over = over(lane), lead = -mine_over & (CHUNK - 1), end = h1 - ((h1 - h0 + mine_over) & (CHUNK - 1));
                        if (lane < rows && lead <= h1 - h0) {
                            if (c == h0) put_cut(h0, lead, to + CHUNK, true);
                            if (c + 32 >= h1) put_cut(end, h1 - end, to + CHUNK + end - c, false);
                        } else if (lane < rows) {                   // no chunk starts here
#pragma unroll 1
                            for (int f = h0; f < h1; ++f) put_cut(f, 1, to + CHUNK + f - h0, true);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_at(dempty0 + 8 * buf);
                else mbar_arrive(dempty + buf);
            }
        }
    }

    // After an abort, whichever role's, no copy may outlive shared memory: each stage's last step started is
    // waited for.  (The steps before it have landed: their MMAs are what freed the stage.)  The CTAs of a
    // pair may have stopped at different steps, up to a ring apart: rank 0, whose barriers count both,
    // expects the peer's bytes of a step that only the peer has started, and counts off those of one that
    // only itself has.
    auto drain_copies = [&](int mine, int peers) {
        const uint32_t bytes = (uint32_t)((p.x_rows + w_rows) * kFp8Block);
        const int last = mine > peers ? mine : peers;
        for (int j = last < p.stages ? 0 : last - p.stages; j < last; ++j) {
            if (j == 0 && withhold) continue;
            uint64_t* bar = full + j % p.stages;
            if (j >= peers) mbar_complete_tx(bar, bytes);
            else if (j >= mine) mbar_arrive_expect_tx(bar, bytes);
            mbar_wait_drain(bar, (uint32_t)((j / p.stages) & 1));
        }
    };
    tc_fence_before();
    __syncthreads();
    if (!PAIR && *abort_flag) {
        if (threadIdx.x == 0) drain_copies(*started, *started);
        __syncthreads();
    }
    if constexpr (SPLIT) {
        // ------------------------------------------------------------ output of a shared tile
        // Every CTA's copies and MMAs are done: the operand rings are free for the exchange.  Piece
        // c / 16 belongs to CTA (c / 16) % split; what the others have of it goes into its ring, one
        // place a sender, four features of 128 tokens at a time (16 bytes a lane, side by side).
        cluster_sync_relaxed();
        tc_fence_after();
        const int e = (warp - 8) >> 2, S = p.split;
        int ft, tt;
        place(first, ft, tt);
        const int f0 = ft * p.bn, width = p.n - f0 < p.bn ? p.n - f0 : p.bn;
        const int row0 = tt * kTokens + 32 * (warp & 3), row = row0 + lane, token = 32 * (warp & 3) + lane;
        const uint32_t acc = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        const int places = (p.bn / 16 + S - 1) / S;                      // pieces a CTA owns at most
        auto slot_of = [&](int sender, int piece) { return (uint32_t)((sender * places + piece / S) * 4 * kTokens * 16); };
        if (warp >= 8 && complete && row0 < p.m) {
            for (int piece = e; 16 * piece < width; piece += 2) {
                const int owner = piece % S;
                if (owner == share) continue;
                uint32_t v[16];
                __syncwarp();
                tmem_ld16(acc + 16 * piece, v);
                tc_wait_ld();
                const uint32_t to = cluster_addr(smem, owner) + slot_of(share, piece) + 16 * token;
                if (row < p.m) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        st_cluster_16(to + q * kTokens * 16, make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]),
                                                                         __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3])));
                }
            }
        }
        // Its own pieces; the residual of the first is on its way while the others' sums arrive.  Where rows
        // do not start on 32 bytes, a warp turns its 32 tokens x 16 features around, so that 16 lanes
        // load and store a token's features side by side (a lane a token: 2 to 4 us more).
        const bool resid = FUSED && epi.resid != nullptr;
        uint32_t r[16];
        auto fetch_resid = [&](int piece) {
            const int f = f0 + 16 * piece;
            if (p.aligned) {
                if (row < p.m) ld_global_32(reinterpret_cast<uint32_t(&)[8]>(r[0]), epi.resid + (int64_t)row * p.n + f);
            } else {
                const uint16_t* from = epi.resid + (f + (lane & 15) < p.n ? f + (lane & 15) : p.n - 1);
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    const int t = row0 + 2 * u + (lane >> 4);
                    r[u] = from[(int64_t)(t < p.m ? t : p.m - 1) * p.n];
                }
            }
        };
        const int mine = (share & 1) == e ? share : width;              // S is even: one group has them all
        const bool there = warp >= 8 && complete && row0 < p.m;
        float* turned = stage32 + (warp - 8) * 32 * kMaxPitch;          // pitch 17
        if (resid && there && 16 * mine < width) fetch_resid(mine);
        cluster_sync();
        if (there) {
            for (int piece = mine; 16 * piece < width; piece += S) {
                uint32_t v[16];
                __syncwarp();
                tmem_ld16(acc + 16 * piece, v);
                tc_wait_ld();
                if (resid && piece != mine) fetch_resid(piece);
                float2 o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = make_float2(0.f, 0.f);
                for (int from = 0; from < S; ++from) {
                    const float4* at = reinterpret_cast<const float4*>(smem + slot_of(from, piece)) + token;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 z = from == share ? make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]),
                                                                     __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]))
                                                       : at[q * kTokens];
                        o[2 * q] = add2(o[2 * q], make_float2(z.x, z.y));
                        o[2 * q + 1] = add2(o[2 * q + 1], make_float2(z.z, z.w));
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = add2(o[j], *reinterpret_cast<const float2*>(sbias + 16 * piece + 2 * j));
                if (FUSED) {
                    activate(o, epi.act);
                    if (epi.gate != nullptr) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) o[j] = mul2(o[j], *reinterpret_cast<const float2*>(sgate + 16 * piece + 2 * j));
                    }
                }
                if (p.aligned) {
                    if (row >= p.m) continue;
                    const int64_t to = (int64_t)row * p.n + f0 + 16 * piece;
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (resid) o[j] = add2(o[j], make_float2(bf16_bits_to_f32(r[j] & 0xFFFFu), bf16_bits_to_f32(r[j] >> 16)));
                        if (YF32) { w[2 * j] = __float_as_uint(o[j].x); w[2 * j + 1] = __float_as_uint(o[j].y); }
                        else w[j] = pack_bf16x2(o[j].x, o[j].y);
                    }
                    if (YF32) {
                        st_global_32(static_cast<float*>(y) + to, reinterpret_cast<uint32_t(&)[8]>(w[0]));
                        st_global_32(static_cast<float*>(y) + to + 8, reinterpret_cast<uint32_t(&)[8]>(w[8]));
                    } else {
                        st_global_32(static_cast<uint16_t*>(y) + to, reinterpret_cast<uint32_t(&)[8]>(w[0]));
                    }
                } else {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        turned[17 * lane + 2 * j] = o[j].x;
                        turned[17 * lane + 2 * j + 1] = o[j].y;
                    }
                    __syncwarp();
                    if ((lane & 15) < width - 16 * piece) {
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const int t = 2 * u + (lane >> 4);
                            const int64_t to = (int64_t)(row0 + t) * p.n + f0 + 16 * piece + (lane & 15);
                            if (row0 + t < p.m) {
                                float z = turned[17 * t + (lane & 15)];
                                if (resid) z += bf16_bits_to_f32(r[u]);
                                if (YF32) static_cast<float*>(y)[to] = z;
                                else static_cast<uint16_t*>(y)[to] = (uint16_t)(pack_bf16x2(z, 0.f) & 0xFFFFu);
                            }
                        }
                    }
                }
            }
        }
        tc_fence_before();
        __syncthreads();
    }
    if constexpr (PAIR) {
        // An abort of one CTA is the pair's; both end when its copies have landed.
        if (threadIdx.x == 0 && *abort_flag) st_cluster_4(cluster_addr(const_cast<int*>(abort_flag), rank ^ 1), 1);
        cluster_sync();                          // no MMA or arrival still needs the peer
        if (*abort_flag) {
            if (rank == 0 && threadIdx.x == 0) drain_copies(*started, ld_cluster_4(cluster_addr(started, 1)));
            cluster_sync();
        }
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
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

template <bool PAIR, bool SPLIT, bool FUSED, bool YF32, bool ANY>
cudaError_t launch_mm_t(const CUtensorMap& tmX, const CUtensorMap& tmW, const uint8_t* xs, const uint8_t* ws,
                        const EpiArgs& epi, void* y, const MmPlan& p, int grid, size_t smem, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static bool configured[64] = {};
    auto kernel = fp8_mm_kernel<PAIR, SPLIT, FUSED, YF32, ANY>;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kQmvMaxSmem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kMmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = PAIR ? 2 : p.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR || SPLIT ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, tmX, tmW, xs, ws, epi, y, p);
}

// Clusters of `ctas` CTAs of the kernel that the device runs at once (those of 4 and 8 do not reach
// every SM: 132 and 120 of 148).
int clusters_at_once(int ctas) {
    static int known[64][9] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int& n = known[dev][ctas];
    if (n == 0) {
        auto kernel = fp8_mm_kernel<false, true, false, false, false>;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(ctas * num_sms()));
        cfg.blockDim = dim3(kMmThreads);
        cfg.dynamicSmemBytes = kQmvMaxSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)ctas;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int at_once = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kQmvMaxSmem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&at_once, kernel, &cfg) != cudaSuccess || at_once < 1) {
            cudaGetLastError();                  // then no tile is shared that way
            at_once = -1;
        }
        n = at_once;
    }
    return n;
}

// The tile: a CTA, a pair or a cluster that shares it, and the width, by the cycles of the longest SM:
// whole waves of tiles, each KT steps of the longest of the MMAs (2 cycles a feature, 300 at least) and
// the copies (64 bytes a cycle from L2), not less than the weight's way from DRAM (3500 bytes a cycle);
// beside them, a tile behind, the output stage (750 cycles for 64 features, as much again for an
// activation, gate or residual, 1000 more for rows of any pitch), which of many short tiles sets the
// pace; the last tile's, and a pair's later start or the exchange, on top.  Measured in a graph, us: 512 x
// 4096 x 10240 with GELU pairs by 144 20.6 (CTAs by 144 22.3); 1 x 9728 x 2560 fours by 80 9.2 (CTAs by 48
// 14.7, twos by 48 11.8, eights by 176 9.7); 16 x 8192 x 128 eights by 16 5.4 (fours 6.5, CTAs 12.3); 3116 x
// 48 x 4181 with SiLU CTAs by 192 25.7 (by 80 35.2, pairs by 192 24.5).  Over 54 shapes from 1 to 4608
// tokens, timed at every width and kind, its choice is at the best's time for half
// of them, within 5 % for all but five and within 9 % for all.
void choose(int64_t m, int64_t n, int64_t k, bool fused, bool aligned, bool& pair, int& bn, int& split) {
    const int64_t kt = (k + kFp8Block - 1) / kFp8Block, sms = num_sms();
    const int64_t dram = n * k / 3500;
    int64_t best = -1;
    for (int cg = 1; cg <= (m > kTokens ? 2 : 1); ++cg) {
        const int64_t ntt = (m + kTokens * cg - 1) / (kTokens * cg);
        const int64_t x_rows = m < kTokens ? m : kTokens;
        for (int w = 16; w <= kMaxBn; w += 16) {
            const int64_t tiles = ntt * ((n + w - 1) / w), waves = (tiles + sms / cg - 1) / (sms / cg);
            const int64_t copy = (x_rows + w / cg) * kFp8Block / 64;
            int64_t step = 2 * w > copy ? 2 * w : copy;
            step = step < 300 ? 300 : step;
            const int64_t out = 900 + (w + 63) / 64 * (750 + (fused ? 750 : 0) + (aligned ? 0 : 1000)), tile = kt * step > out ? kt * step : out;
            const int64_t all = kt * step + (waves - 1) * tile, cost = (all > dram ? all : dram) + out + (cg == 2 ? 700 : 0);
            if (best < 0 || cost < best) {
                best = cost;
                pair = cg == 2;
                bn = w;
                split = 1;
            }
            // Shared tiles: all clusters at once, a step at least for every CTA, its own pieces of 16
            // features and the exchange.
            for (int s = 2; cg == 1 && s <= 8 && s <= kt; s *= 2) {
                if (tiles > clusters_at_once(s)) break;
                const int64_t steps = (kt + s - 1) / s * step, exchange = 3000 + 150 * s + w * (15 + x_rows / 12);
                const int64_t own = 900 + (w / 16 + s - 1) / s * (500 + (fused ? 250 : 0) + (aligned ? 0 : 300));
                const int64_t shared = (steps > dram ? steps : dram) + own + exchange;
                if (shared < best) {
                    best = shared;
                    pair = false;
                    bn = w;
                    split = s;
                }
            }
        }
    }
}

// All that a launch depends on but its pointers; `aligned` as in MmPlan.  grid: CTAs.
MmPlan plan_for(int64_t m, int64_t n, int64_t k, bool fused, bool aligned, bool& pair, int& grid) {
    MmPlan p{};
    p.aligned = aligned;
    choose(m, n, k, fused, aligned, pair, p.bn, p.split);
    const int cg = pair ? 2 : 1;
    p.m = (int)m;
    p.n = (int)n;
    p.k = (int)k;
    p.kt = (int)((k + kFp8Block - 1) / kFp8Block);
    p.x_rows = m < kTokens ? (int)((m + 7) / 8 * 8) : kTokens;
    // Odd, so that a lane a token writes without bank conflicts; lanes that read a chunk each, of rows
    // whose chunks start n values further back each time, then meet in pairs at most.
    p.pitch = n % 4 == 1 ? kMaxPitch : kMaxPitch - 2;
    const size_t stage = kXStage + (size_t)(p.bn / cg) * kFp8Block;
    const int fit = (int)((kQmvMaxSmem - fixed_smem(aligned)) / stage);
    p.stages = fit < kMaxStages ? fit : kMaxStages;
    const int64_t nft = (n + p.bn - 1) / p.bn, ntt = (m + cg * kTokens - 1) / (cg * kTokens), tiles = nft * ntt;
    p.nft = (int)nft;
    p.ntt = (int)ntt;
    const int64_t fit_tt = (32ll << 20) / ((int64_t)cg * kTokens * k);     // token tiles whose X is 32 MB
    p.group = (int)(fit_tt < 1 ? 1 : (fit_tt < ntt ? fit_tt : ntt));
    p.by_tiles = Divisor((uint32_t)(p.group * p.nft));
    p.by_group = Divisor((uint32_t)p.group);
    p.by_rest = Divisor((uint32_t)(ntt % p.group ? ntt % p.group : p.group));
    const int64_t places = num_sms() / cg;
    grid = p.split > 1 ? (int)tiles * p.split : (int)(tiles < places ? tiles : places) * cg;
    return p;
}

}  // namespace

cudaError_t launch_fp8_mm(const uint8_t* xq, const uint8_t* xs, int64_t m, int64_t k, const uint8_t* wq,
                          const uint8_t* ws, int64_t n, const EpiArgs& epi, void* y, cudaStream_t st,
                          const char** msg) {
    const uintptr_t bases = reinterpret_cast<uintptr_t>(y) | (epi.resid ? reinterpret_cast<uintptr_t>(epi.resid) : 0);
    bool pair = false;
    int grid = 0;
    MmPlan p = plan_for(m, n, k, epi.fused(), n % 16 == 0 && bases % 32 == 0, pair, grid);
    p.resid_like_y = (reinterpret_cast<uintptr_t>(y) - reinterpret_cast<uintptr_t>(epi.resid)) % 16 == 0;
    CUtensorMap tmX, tmW;
    const int w_rows = p.bn / (pair ? 2 : 1);
    if (!byte_map(&tmX, xq, m, k, p.x_rows) || !byte_map(&tmW, wq, n, k, w_rows)) {
        *msg = "cuTensorMapEncodeTiled rejected an fp8 operand's tensor map";
        return cudaErrorInvalidValue;
    }
    // More than half of an SM's shared memory, so that no second CTA waits there for tensor memory.
    size_t smem = fixed_smem(p.aligned) + (size_t)p.stages * (kXStage + w_rows * kFp8Block);
    if (smem < 120 * 1024) smem = 120 * 1024;
    auto go = [&](auto pr, auto sp, auto any) {
        constexpr bool P = decltype(pr)::value, S = decltype(sp)::value, A = decltype(any)::value;
        if (epi.fused()) return launch_mm_t<P, S, true, false, A>(tmX, tmW, xs, ws, epi, y, p, grid, smem, st);
        if (epi.f32) return launch_mm_t<P, S, false, true, A>(tmX, tmW, xs, ws, epi, y, p, grid, smem, st);
        return launch_mm_t<P, S, false, false, A>(tmX, tmW, xs, ws, epi, y, p, grid, smem, st);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (p.split > 1) return go(No{}, Yes{}, No{});
    if (pair) return p.aligned ? go(Yes{}, No{}, No{}) : go(Yes{}, No{}, Yes{});
    return p.aligned ? go(No{}, No{}, No{}) : go(No{}, No{}, Yes{});
}

void fp8_mm_plan(int64_t m, int64_t k, int64_t n, bool fused, bool aligned, int32_t (&out)[6]) {
    bool pair = false;
    int grid = 0;
    const MmPlan p = plan_for(m, n, k, fused, aligned, pair, grid);
    const int ctas = pair ? 2 : p.split;
    const int32_t v[6] = {pair ? 2 : 1, p.split, p.bn, p.nft * p.ntt, grid / ctas, p.group};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
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
