// The 8-bit cache: a row (head_dim values of one token and kv head) is kept as e4m3 codes c_i and one power of two 2^e, the
// least with max |x_i| <= 448 * 2^e over the row's finite values (448: the largest e4m3 value; e >= -126).  A value is
// c_i * 2^e.  Scaling by a power of two rounds nothing, so a code is off by half an e4m3 step at most (2^-4 of the value, or
// 2^-10 * 2^e below the least normal code), and what is read back is exact in bfloat16 and in 32 bits.  One exponent a row
// (1 byte beside head_dim) and not one for every 32 values: it is a factor of a key's score and of a key's weight, so
// neither product of the attention has to touch it per element.
// Pages: codes [pages, kv heads, 64, head_dim], exponents e + 127 [pages, kv heads, 64], both bytes.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

// e for a row's largest finite magnitude, given as float bits: x = m 2^k, 1 <= m < 2, and 448 = 1.75 * 2^8.
__device__ __forceinline__ int c8_exponent(uint32_t top_bits) {
  const int k = (int)(top_bits >> 23) - 127;                                 // (zero and subnormal rows: -127)
  const int e = (top_bits & 0x7fffffu) <= 0x600000u ? k - 8 : k - 7;         // (mantissa bits of 1.75)
  return max(e, -126);
}
// 2^p for -126 <= p <= 127
__device__ __forceinline__ float c8_pow2(int p) { return __uint_as_float((uint32_t)(p + 127) << 23); }
// Two e4m3 codes (the first in the low byte); values beyond 448 do not occur, NaN gives NaN.
__device__ __forceinline__ uint32_t c8_pack2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// Four codes as two pairs of halves (every e4m3 value is a half): one instruction a pair.
__device__ __forceinline__ void c8_half4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
// Two codes.
__device__ __forceinline__ uint32_t c8_half2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
