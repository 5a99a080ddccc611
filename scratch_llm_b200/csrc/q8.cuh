// Numbers of a cache held in 8 bits (sm_100a).
//
// A value is an e4m3 number times its block's power of two: v = q * 2^(b - 127), b an e8m0 byte.  A block
// is `block` neighbouring places of a page, for one plane (keys or values) and one kv head.  With
// powers of two a value is exact in bfloat16 and in 32 bits (q has 4 significant bits), and a block whose
// scale grows only shifts exponents: its earlier values stay as they are, but for those that become
// subnormal.  A finer scale would gain at most a binade of e4m3's range, which its own exponents cover.
//
// b is the smallest byte of 1 and more with amax <= 448 * 2^(b - 127), amax over the block's finite values, so
// that nothing saturates.  e4m3 has no infinity: infinities and NaN are stored as NaN and leave b alone.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace sllm {

// n / d for 0 <= n < 2^31: 2 n * ceil(2^(31 + s) / d) / 2^(32 + s), 2^s >= d
struct Divisor {
    uint32_t magic; int shift, d;
    __device__ __forceinline__ int quotient(int n) const { return (int)(__umulhi(2u * (uint32_t)n, magic) >> shift); }
};
static Divisor divisor(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s, d};
}

// 448 = 1.75 * 2^8: with amax = m * 2^(E - 127), 1 <= m < 2, b = E - 8, one more where m > 1.75.
__device__ __forceinline__ int q8_scale_byte(float amax) {
    const int bits = __float_as_int(amax);
    return max(1, (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0));
}
// 2^(b - 127); 0 stands for 2^-127 and 255 for NaN, as in e8m0 (neither is ever written here)
__device__ __forceinline__ float q8_power(int b) {
    return __int_as_float(b == 0 ? 0x00400000 : b == 255 ? 0x7fffffff : b << 23);
}
// 2^(127 - b) for b from 1 to 253
__device__ __forceinline__ float q8_inverse(int b) { return __int_as_float((254 - b) << 23); }

__device__ __forceinline__ bool q8_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// two scaled values to e4m3 (to nearest, ties to even; |a|, |b| <= 448 or no number)
__device__ __forceinline__ uint32_t q8_pack2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d) {
    return q8_pack2(a, b) | q8_pack2(c, d) << 16;
}
// two e4m3 numbers (the low 16 bits) as two halves, exactly
__device__ __forceinline__ uint32_t q8_half2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ float2 q8_float2(uint32_t two) {
    const uint32_t h = q8_half2(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace sllm
