// act_int8.cu - activations to 8 bits as they are kept for the backward pass,
// and back (the form: int8_blocks.cuh). Bound by memory: 2 or 4 bytes read and
// 1 + 1/32 written per value, or the reverse.
#include "int8_blocks.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float loadAs(const uint16_t* p) { return bf2f(*p); }
__device__ __forceinline__ float loadAs(const float* p) { return *p; }
__device__ __forceinline__ void storeAs(uint16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void storeAs(float* p, float v) { *p = v; }

// fmaxf drops a NaN, so a block's NaNs are carried as infinity.
__device__ __forceinline__ float magnitude(float v) {
  return __uint_as_float(min(__float_as_uint(fabsf(v)), 0x7f800000u));
}

// One warp per block of 32 neighbours, one value per lane.
template <class T>
__global__ void __launch_bounds__(kThreads)
    quantizeInt8(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ e,
                 int64_t rows, int cols, int blocks) {
  const int lane = threadIdx.x & 31;
  const int64_t n = rows * blocks;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b < n;
       b += warps) {
    const int64_t row = b / blocks;
    const int c = (int)(b % blocks) * kInt8Block + lane;
    const float v = c < cols ? loadAs(x + row * cols + c) : 0.f;
    const uint32_t ex = int8Exponent(warpMax(magnitude(v)));
    if (c < cols) q[row * cols + c] = (uint8_t)int8Quantize(v, int8Inverse(ex));
    if (lane == 0) e[b] = (uint8_t)ex;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    dequantizeInt8(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                   T* __restrict__ x, int64_t rows, int cols, int blocks) {
  const int lane = threadIdx.x & 31;
  const int64_t n = rows * blocks;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b < n;
       b += warps) {
    const int64_t row = b / blocks;
    const int c = (int)(b % blocks) * kInt8Block + lane;
    if (c < cols) storeAs(x + row * cols + c, (float)(int8_t)q[row * cols + c] * int8Step(e[b]));
  }
}

unsigned gridFor(int64_t blocks) {
  const int64_t ctas = (blocks + kThreads / 32 - 1) / (kThreads / 32);
  return (unsigned)(ctas < kSMs * 8 ? ctas : kSMs * 8);
}

}  // namespace
}  // namespace tnops

using namespace tnops;

extern "C" int tnops_quantize_int8(const void* x, int x_f32, uint8_t* q, uint8_t* e, int64_t rows,
                                   int cols, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 1;
  const int blocks = (cols + kInt8Block - 1) / kInt8Block;
  if (x_f32)
    quantizeInt8<<<gridFor(rows * blocks), kThreads, 0, stream>>>(static_cast<const float*>(x), q,
                                                                 e, rows, cols, blocks);
  else
    quantizeInt8<<<gridFor(rows * blocks), kThreads, 0, stream>>>(
        static_cast<const uint16_t*>(x), q, e, rows, cols, blocks);
  return launched(cudaGetLastError());
}

extern "C" int tnops_dequantize_int8(const uint8_t* q, const uint8_t* e, void* x, int x_f32,
                                     int64_t rows, int cols, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 1;
  const int blocks = (cols + kInt8Block - 1) / kInt8Block;
  if (x_f32)
    dequantizeInt8<<<gridFor(rows * blocks), kThreads, 0, stream>>>(q, e, static_cast<float*>(x),
                                                                   rows, cols, blocks);
  else
    dequantizeInt8<<<gridFor(rows * blocks), kThreads, 0, stream>>>(
        q, e, static_cast<uint16_t*>(x), rows, cols, blocks);
  return launched(cudaGetLastError());
}
