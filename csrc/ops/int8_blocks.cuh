// int8_blocks.cuh - the 8-bit form in which activations are kept for the
// backward pass: whole numbers in [-127, 127] with one power of two for each
// 32 neighbours of a row (the block form of the OCP Microscaling formats).
//
//   value = q 2^(e - 133),  e = 0 .. 254 one byte per block, 255: not a number
//
// e is the least with round(max / 2^(e - 133)) <= 127, so the largest value of a
// block is at least 63.75 steps and a value is off by at most half a step, 1 / 127.5
// of the block's largest (but for blocks below 2^-127, whose step stays 2^-133, and
// the last half step below 2^128, which keeps 127 steps). Multiplying by a
// power of two is exact, so the only rounding is the one to whole numbers
// (nearest, ties to even), and a value read back has seven significant bits:
// it is a bf16 number, whatever the block. A block that holds an infinity or
// a NaN reads back as NaN.
#pragma once

#include "common.cuh"

namespace tnops {
namespace {

constexpr int kInt8Block = 32;

// Exponent byte of a block from its largest magnitude: with a step that makes it
// 64 to 128 steps, 127.5 or more (a mantissa of at least 127.5 / 64) would round
// to 128. Adding 2^16 to the fp32 bits carries into the exponent from there on.
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
// q as a two's complement byte. x / step + 1.5 2^23 is a whole number whose
// last byte is q (one FMA, where a conversion takes the special-function
// unit). Only fp32 values above 127.5 2^121 can reach 128 (e stops at 254):
// they keep 127.
__device__ __forceinline__ uint32_t int8Quantize(float x, Int8Inverse inv) {
  const float y = fminf(fmaxf(x * inv.a * inv.b, -127.f), 127.f);
  return __float_as_uint(y + 12582912.f) & 0xffu;
}
// Four values to four bytes, for an exponent in [6, 254): one factor, and
// nothing to clamp.
__device__ __forceinline__ bool int8Plain(uint32_t e) { return e - 6u < 248u; }
__device__ __forceinline__ uint32_t int8Quantize4(float a, float b, float c, float d, float inv) {
  const uint32_t x = __float_as_uint(fmaf(a, inv, 12582912.f)),
                 y = __float_as_uint(fmaf(b, inv, 12582912.f)),
                 z = __float_as_uint(fmaf(c, inv, 12582912.f)),
                 w = __float_as_uint(fmaf(d, inv, 12582912.f));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}
__device__ __forceinline__ float int8Step(uint32_t e) {
  if (e == 255u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(e >= 7u ? (e - 6u) << 23 : 1u << (e + 16u));
}
// Four bytes to four values: q + 128 is put in the last byte of 2^23, from
// which 2^23 + 128 is taken; both steps are exact.
__device__ __forceinline__ float4 int8x4(uint32_t q, float step) {
  const uint32_t u = q ^ 0x80808080u;
  auto value = [&](uint32_t bytes) {
    return (__uint_as_float(__byte_perm(u, 0x4b000000u, bytes)) - 8388736.f) * step;
  };
  return make_float4(value(0x7650), value(0x7651), value(0x7652), value(0x7653));
}

}  // namespace
}  // namespace tnops
