// int8_blocks.cuh - the 8-bit form in which activations are kept for the
// backward pass: whole numbers in [-127, 127] with one power of two for each
// 32 neighbours of a row (the block form of the OCP Microscaling formats).
//
//   value = q 2^(e - 133),  e = 0 .. 254 one byte per block, 255: not a number
//
// e is the least with round(max / 2^(e - 133)) <= 127, so a value is off by
// at most half a step, 2^-7 of the block's largest value. Multiplying by a
// power of two is exact, so the only rounding is the one to whole numbers
// (nearest, ties to even), and a value read back has seven significant bits:
// it is a bf16 number, whatever the block. A block that holds an infinity or
// a NaN reads back as NaN.
#pragma once

#include "common.cuh"

namespace tnops {
namespace {

constexpr int kInt8Block = 32;

// Exponent byte of a block from its largest magnitude. Adding 2^16 to the
// fp32 bits carries into the exponent when the mantissa is at least 127/64
// steps of 64, i.e. when 127.5 steps or more would be needed.
__device__ __forceinline__ uint32_t int8Exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u >= 0x7f800000u) return 255u;
  const uint32_t e = (u + 0x10000u) >> 23;
  return e < 254u ? e : 254u;
}
// 1 / step as two factors (the second is 1 but for the smallest exponents,
// whose inverse passes the fp32 range).
struct Int8Inverse {
  float a, b;
};
__device__ __forceinline__ Int8Inverse int8Inverse(uint32_t e) {
  const uint32_t c = e < 6u ? 6u : e > 254u ? 254u : e;
  return {__uint_as_float((260u - c) << 23), __uint_as_float((127u + c - (e < 6u ? e : c)) << 23)};
}
// q as a two's complement byte. Only fp32 values above 127.5 2^121 can reach
// 128 (e stops at 254): they keep 127.
__device__ __forceinline__ uint32_t int8Quantize(float x, Int8Inverse inv) {
  const int q = __float2int_rn(x * inv.a * inv.b);
  return (uint32_t)max(-127, min(127, q)) & 0xffu;
}
__device__ __forceinline__ float int8Step(uint32_t e) {
  if (e == 255u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(e >= 7u ? (e - 6u) << 23 : 1u << (e + 16u));
}
// Four bytes to four values.
__device__ __forceinline__ float4 int8x4(uint32_t q, float step) {
  return make_float4((float)(int8_t)(q & 0xff) * step, (float)(int8_t)((q >> 8) & 0xff) * step,
                     (float)(int8_t)((q >> 16) & 0xff) * step, (float)(int8_t)(q >> 24) * step);
}

}  // namespace
}  // namespace tnops
