// Rows of numbers in 8 bits: e4m3 numbers q and, for every 128 consecutive numbers of a row, a power of two 2^E.
//
//   x[r, k] ~ q[r, k] * 2^E[r, k / 128]      E: the least integer >= -127 with max |x| of the block <= 448 * 2^E
//
// 448 is the largest e4m3 number. Dividing by a power of two is exact, so a number is rounded once (to nearest, ties to even: by at
// most 2^-4 of itself, or 2^-10 * 2^E where e4m3 is subnormal). Scales are stored as E8M0 bytes (E + 127), laid out
// [ceil(K / 512), rows, 4]: the scales of 512 numbers of a row are one 32-bit word, which is what the tensor memory takes for a row
// (gemm_fp8.cu). Bytes past a row's last block are 0. A NaN or an infinity becomes the NaN of e4m3: it comes out of a product as NaN.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

constexpr int F8_BLOCK = 128;      // numbers of a row that share a scale
constexpr int F8_WORD = 512;       // numbers whose scales make up a word

// E + 127 for a block's largest magnitude (finite or not; never above 247).
__device__ __forceinline__ uint32_t f8_scale_byte(float top) {
  // top = 1.m * 2^(e - 127): the quotient of top and 448 = 1.75 * 2^8 is at most 2^(e - 127 - 8) where 1.m <= 1.75, else at
  // most twice that. Zero and subnormal numbers give the least scale.
  const uint32_t bits = __float_as_uint(top) & 0x7fffffffu, e = bits >> 23, m = bits & 0x7fffffu;
  const int byte = (int)e - 8 + (m > 0x600000u ? 1 : 0);
  return byte < 0 ? 0u : (byte > 247 ? 247u : (uint32_t)byte);
}
// 2^-E of a scale byte up to 247: exact, and a normal number.
__device__ __forceinline__ float f8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Two numbers, already divided by their scale, as e4m3 (the lower byte is the first). An infinity would become 448: a block whose
// maximum is one goes through f8_pack2_any.
__device__ __forceinline__ uint32_t f8_pack2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
static __device__ __noinline__ uint32_t f8_pack2_any(float a, float b) {
  uint32_t r = f8_pack2(a, b);
  if (isinf(a)) r |= 0x7fu;
  if (isinf(b)) r |= 0x7f00u;
  return r;
}
