// sdq_fp8.cuh -- the block-scaled 8-bit floating-point format shared by the fp8 kernels.
//
// A value is e4m3 (1 sign, 4 exponent, 3 mantissa bits; largest 448, no infinities, 0x7F NaN)
// times a scale 2^(byte - 127) held as one e8m0 byte (255 stands for NaN).  A scale covers 128
// values of a row (activations) or a 128 x 128 block (weights).  Powers of two are used because
// dividing by one is exact: a value is rounded once, to e4m3, and the tensor cores multiply the
// scales in themselves (tcgen05 block_scale), so the product needs no pass over its partial sums.
#pragma once

#include <cstdint>
#include <cuda_fp8.h>

namespace sdq {

constexpr int kFp8Block = 128;

// The e8m0 byte of 2^e, e the least integer with amax <= 448 * 2^e and e >= -126; 255 (NaN) when
// amax is infinite or NaN.  With amax = 1.f * 2^E and 448 = 1.75 * 2^8 that is E - 8, one more
// when 1.f > 1.75.  `amax_bits` are the bits of |amax| in f32 (ordered like the values, NaN last,
// so the bits themselves can be reduced with an integer maximum).
__device__ __forceinline__ uint32_t e8m0_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return 255u;
    const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t)(b < 1 ? 1 : b);
}
// 2^-(byte - 127) as f32 (bytes 1 .. 247, all that e8m0_of gives), NaN for 255.
__device__ __forceinline__ float e8m0_inverse(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127) as f32 for any byte (0 is the subnormal 2^-127), NaN for 255.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    if (byte == 255u) return __uint_as_float(0x7FFFFFFFu);
    return byte == 0u ? __uint_as_float(0x400000u) : __uint_as_float(byte << 23);
}
// Two floats to two e4m3 bytes (a in the low one), nearest even, saturating; NaN -> 0x7F.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace sdq
