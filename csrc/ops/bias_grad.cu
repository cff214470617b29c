// bias_grad.cu - bias gradients of the GPT-2 linear layers, optionally fused
// with the tanh-GELU backward that precedes them.
//
//   tnops_bias_grad:     db[n] = sum_m g[m, n]                   (g bf16, db fp32)
//   tnops_gelu_bwd_bias: gp[m, n] = bf16(gy[m, n] * gelu'(pre[m, n]))
//                        db[n]    = sum_m gp[m, n]
//   tnops_gelu_bwd_bias_int8: the same with pre kept in 8 bits
//                        (int8_blocks.cuh), read back as it is used.
//
// Column sums of an [M, N] row-major bf16 matrix, deterministic: pass 1
// tiles the matrix into (256-column, rowsPer-row) blocks; each warp of a CTA
// owns 256 columns (8 per lane, one 16-byte load per row) and every 8th row
// of the block, 4 rows in flight; the 8 warp sums are added in warp order
// into one fp32 partial per block (the result, where one block is all). Pass 2
// adds the partials of a column in block order (colReduce, common.cuh). The
// summation order depends only on (M, N), never on scheduling. Rounding of the
// GELU gradient to bf16 happens before it is summed, as when the gradient
// tensor is materialised and then reduced; with an 8-bit pre the sum is of the
// fp32 products.
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"
#include "int8_blocks.cuh"
#include "packed_f32.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

constexpr int kCols = 256;  // columns per CTA (8 per lane x 32 lanes)
constexpr int kWarps = 8;
constexpr int kUnroll = 4;  // rows in flight per warp

__device__ __forceinline__ void bf16x8ToF(uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Derivative of the tanh approximation of GELU, 0.5 x (1 + tanh(u)) with
// u = k0 (x + k1 x^3), from the product rule:
//   0.5 (1 + t) + 0.5 x (1 - t^2) u',  t = tanh(u),  u' = k0 + 3 k0 k1 x^2.
// With e = e^(-2u) and r = 1 / (1 + e): 0.5 (1 + t) = r and
// 1 - t^2 = 4 r (1 - r) = 4 r (e r), so the derivative is
// r + 2 x r (e r) u': one ex2 and one fast division, and 1 - t^2 comes from
// e r directly, never from 1 - t*t (which cancels where |t| is near 1).
__device__ __forceinline__ float ex2Approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float geluTanhGrad(float x) {
  const float k0 = 0.7978845608028654f;  // sqrt(2 / pi)
  const float k0k1 = 0.7978845608028654f * 0.044715f;
  const float m2log2e = -2.0f * 1.4426950408889634f;
  const float x2 = x * x;
  // |u| <= 40 keeps e and r finite (e^80 < FLT_MAX); the derivative is 0 or
  // 1 to float precision well before that.
  const float u = fminf(fmaxf(x * fmaf(k0k1, x2, k0), -40.0f), 40.0f);
  const float e = ex2Approx(u * m2log2e);
  const float r = __fdividef(1.0f, 1.0f + e);
  const float du = fmaf(3.0f * k0k1, x2, k0);
  return fmaf(2.0f * x * r * (e * r), du, r);
}

// max(lo, min(x, hi)), NaN for NaN.
__device__ __forceinline__ float within(float x, float lo, float hi) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(hi));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(lo));
  return x;
}
// The same derivative of two numbers at once. x is held within +-9.5, where the
// derivative is 0 or 1 to 1e-29 and nothing passes the fp32 range (further out
// e^(-2u) would, then x^2).
__device__ __forceinline__ uint64_t geluTanhGrad2(uint64_t in) {
  const float k0 = 0.7978845608028654f, k0k1 = 0.7978845608028654f * 0.044715f;
  const float m2log2e = -2.0f * 1.4426950408889634f;
  float a, b;
  unpack2(in, a, b);
  const uint64_t x = pack2(within(a, -9.5f, 9.5f), within(b, -9.5f, 9.5f));
  const uint64_t x2 = mul2(x, x);
  const uint64_t du = fma2(pack2(3.0f * k0k1, 3.0f * k0k1), x2, pack2(k0, k0));
  unpack2(mul2(mul2(x, fma2(pack2(k0k1, k0k1), x2, pack2(k0, k0))), pack2(m2log2e, m2log2e)), a,
          b);
  const uint64_t e = pack2(ex2Approx(a), ex2Approx(b));
  unpack2(add2(e, pack2(1.0f, 1.0f)), a, b);
  float ra, rb;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ra) : "f"(a));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rb) : "f"(b));
  const uint64_t r = pack2(ra, rb);
  const uint64_t t = mul2(mul2(x, r), mul2(e, r));
  return fma2(add2(t, t), du, r);
}
// Four 8-bit values as two pairs.
__device__ __forceinline__ void int8x4Pairs(uint32_t q, uint64_t step, uint64_t& lo,
                                            uint64_t& hi) {
  const uint32_t u = q ^ 0x80808080u;
  const uint64_t off = pack2(-8388736.f, -8388736.f);
  auto at = [&](uint32_t bytes) { return __uint_as_float(__byte_perm(u, 0x4b000000u, bytes)); };
  lo = mul2(add2(pack2(at(0x7650), at(0x7651)), off), step);
  hi = mul2(add2(pack2(at(0x7652), at(0x7653)), off), step);
}

// What the GELU gradient reads pre from: nothing (no GELU), bf16, or 8-bit
// blocks (whose exponents are `preExp`).
enum class Pre { kNone, kBf16, kInt8 };

// T: what the sums are written as (fp32 partial sums, or the result itself
// where one block of rows is all); null: no sums.
template <Pre PRE, class T>
__global__ void __launch_bounds__(kWarps * 32)
    colsumPartial(const uint16_t* __restrict__ gy, const void* __restrict__ pre,
                  const uint8_t* __restrict__ preExp, uint16_t* __restrict__ gout,
                  T* __restrict__ partial, int M, int N, int rowsPer) {
  const int blocks = (N + kInt8Block - 1) / kInt8Block;
  __shared__ float sAcc[kWarps][kCols];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col0 = blockIdx.x * kCols + lane * 8;
  const int r0 = blockIdx.y * rowsPer;
  const int r1 = min(M, r0 + rowsPer);
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  if (col0 < N) {
    for (int rb = r0 + w; rb < r1; rb += kWarps * kUnroll) {
      uint4 g[kUnroll], p[kUnroll];  // 8-bit pre: eight values and the exponent
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int r = rb + u * kWarps;
        if (r < r1) {
          const size_t off = (size_t)r * N + col0;
          g[u] = __ldcs(reinterpret_cast<const uint4*>(gy + off));
          if (PRE == Pre::kBf16)
            p[u] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(pre) + off));
          if (PRE == Pre::kInt8) {
            const uint2 q =
                __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pre) + off));
            p[u] = make_uint4(q.x, q.y, preExp[(size_t)r * blocks + col0 / kInt8Block], 0u);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int r = rb + u * kWarps;
        if (r >= r1) continue;
        float f[8];
        bf16x8ToF(g[u], f);
        if (PRE == Pre::kInt8) {
          const float s1 = int8Step(p[u].z);
          const uint64_t step = pack2(s1, s1);
          uint64_t x[4];
          int8x4Pairs(p[u].x, step, x[0], x[1]);
          int8x4Pairs(p[u].y, step, x[2], x[3]);
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a, b;
            unpack2(mul2(pack2(f[2 * i], f[2 * i + 1]), geluTanhGrad2(x[i])), a, b);
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            o[i] = *reinterpret_cast<const uint32_t*>(&h);
            f[2 * i] = a;  // the bias gradient's sum is of the unrounded ones
            f[2 * i + 1] = b;
          }
          *reinterpret_cast<uint4*>(gout + (size_t)r * N + col0) =
              make_uint4(o[0], o[1], o[2], o[3]);
        } else if (PRE == Pre::kBf16) {
          float x[8];
          bf16x8ToF(p[u], x);
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t lo = f2bf(f[2 * i] * geluTanhGrad(x[2 * i]));
            const uint16_t hi = f2bf(f[2 * i + 1] * geluTanhGrad(x[2 * i + 1]));
            o[i] = (uint32_t)lo | ((uint32_t)hi << 16);
            f[2 * i] = bf2f(lo);
            f[2 * i + 1] = bf2f(hi);
          }
          *reinterpret_cast<uint4*>(gout + (size_t)r * N + col0) =
              make_uint4(o[0], o[1], o[2], o[3]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += f[e];
      }
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sAcc[w][lane * 8 + e] = acc[e];
  __syncthreads();
  const int c = blockIdx.x * kCols + threadIdx.x;
  if (c < N) {
    float s = sAcc[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) s += sAcc[k][threadIdx.x];
    putSum(partial + (size_t)blockIdx.y * N + c, s);
  }
}

}  // namespace
}  // namespace tnops

using namespace tnops;

// Row blocks: enough CTAs for ~8 per SM, at least 32 rows each.
extern "C" int tnops_colsum_parts(int M, int N) {
  const int colBlocks = (N + kCols - 1) / kCols;
  int parts = (kSMs * 8 + colBlocks - 1) / colBlocks;
  const int maxParts = M / 32 > 0 ? M / 32 : 1;
  return parts < 1 ? 1 : parts > maxParts ? maxParts : parts;
}

template <class T>
static int launchColsum(Pre kind, const uint16_t* gy, const void* pre, const uint8_t* preExp,
                        uint16_t* gout, T* db, float* partial, int M, int N,
                        cudaStream_t stream) {
  if (M <= 0 || N <= 0 || N % 8 != 0 || (db == nullptr && gout == nullptr)) return 1;
  // 16-byte pieces of every row (8-byte ones of an 8-bit pre): N % 8 == 0
  // keeps the rows on the boundary when the base pointers are.
  const uintptr_t preMask = kind == Pre::kInt8 ? 7 : 15;
  if (((reinterpret_cast<uintptr_t>(gy) | reinterpret_cast<uintptr_t>(gout)) & 15) ||
      (reinterpret_cast<uintptr_t>(pre) & preMask))
    return 1;
  const int parts = tnops_colsum_parts(M, N);
  const int rowsPer = (M + parts - 1) / parts;
  const dim3 grid((unsigned)((N + kCols - 1) / kCols), (unsigned)parts);
  auto run = [&](auto* sums) {
    using S = std::remove_pointer_t<decltype(sums)>;
    auto kernel = kind == Pre::kNone    ? colsumPartial<Pre::kNone, S>
                  : kind == Pre::kBf16 ? colsumPartial<Pre::kBf16, S>
                                       : colsumPartial<Pre::kInt8, S>;
    kernel<<<grid, kWarps * 32, 0, stream>>>(gy, pre, preExp, gout, sums, M, N, rowsPer);
  };
  if (parts == 1 || db == nullptr) {
    run(db);
    return launched(cudaGetLastError()) == 0 ? 0 : 2;
  }
  if (partial == nullptr) return 1;
  run(partial);
  colReduce<T><<<(N + 31) / 32, kColReduceWarps * 32, 0, stream>>>(partial, parts, N, N, N, db,
                                                                   static_cast<T*>(nullptr));
  gLaunches.fetch_add(2, std::memory_order_relaxed);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

// partial: tnops_colsum_parts(M, N) * N floats of scratch.
extern "C" int tnops_bias_grad(const uint16_t* g, float* db, float* partial, int M, int N,
                               cudaStream_t stream) {
  return launchColsum(Pre::kNone, g, nullptr, nullptr, nullptr, db, partial, M, N, stream);
}

extern "C" int tnops_gelu_bwd_bias(const uint16_t* gy, const uint16_t* pre, uint16_t* gpre,
                                   float* db, float* partial, int M, int N, cudaStream_t stream) {
  return launchColsum(Pre::kBf16, gy, pre, nullptr, gpre, db, partial, M, N, stream);
}

extern "C" int tnops_bias_grad_bf16(const uint16_t* g, uint16_t* db, float* partial, int M, int N,
                                    cudaStream_t stream) {
  return launchColsum(Pre::kNone, g, nullptr, nullptr, nullptr, db, partial, M, N, stream);
}

extern "C" int tnops_gelu_bwd_bias_int8(const uint16_t* gy, const uint8_t* pre_q,
                                        const uint8_t* pre_e, uint16_t* gpre, void* db,
                                        int db_f32, float* partial, int M, int N,
                                        cudaStream_t stream) {
  return db_f32 ? launchColsum(Pre::kInt8, gy, pre_q, pre_e, gpre, static_cast<float*>(db),
                               partial, M, N, stream)
                : launchColsum(Pre::kInt8, gy, pre_q, pre_e, gpre, static_cast<uint16_t*>(db),
                               partial, M, N, stream);
}
