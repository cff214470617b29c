// act_int8.cu - activations to 8 bits as they are kept for the backward pass,
// and back (the form: int8_blocks.cuh). Bound by memory: 2 or 4 bytes read and
// 1 + 1/32 written per value, or the reverse.
//
// bf16 rows of a multiple of 8 values take 16-byte pieces: four neighbouring
// lanes hold a block, each thread several pieces in flight. Other rows and
// fp32 take one warp per block, one value per lane.
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

constexpr int kPieces = 4;  // 16-byte pieces in flight per thread

// Piece s of `slots` = rows * blocks * 4 covers values 8 (s mod 4 blocks) ..
// + 7 of row s / (4 blocks); those past the row's end are skipped.
struct Piece {
  int64_t at;  // first value, or -1
};
__device__ __forceinline__ Piece pieceAt(uint32_t s, uint32_t slots, uint32_t perRow, int cols) {
  if (s >= slots) return {-1};
  const uint32_t row = s / perRow, c = (s - row * perRow) * 8;
  return {c < (uint32_t)cols ? (int64_t)row * cols + c : -1};
}

__global__ void __launch_bounds__(kThreads)
    quantizePieces(const uint16_t* __restrict__ x, uint8_t* __restrict__ q,
                   uint8_t* __restrict__ e, uint32_t slots, uint32_t perRow, int cols) {
  const uint32_t s0 = blockIdx.x * (kThreads * kPieces) + threadIdx.x;
  Piece p[kPieces];
  uint4 u[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    p[i] = pieceAt(s0 + i * kThreads, slots, perRow, cols);
    u[i] = p[i].at >= 0 ? __ldcs(reinterpret_cast<const uint4*>(x + p[i].at))
                        : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
    // bf16 magnitudes order like their bits, NaNs above infinity.
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = __vmaxu2(top, w[k] & 0x7fff7fffu);
    top = max(top >> 16, top & 0xffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t ex = int8Exponent(__uint_as_float(top << 16));
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(w[k] << 16);
      v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
    uint32_t o[2];
    if (int8Plain(ex)) {
      const float inv = int8Inverse(ex).a;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        o[k] = int8Quantize4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3], inv);
    } else {
      const Int8Inverse inv = int8Inverse(ex);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        o[k] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[k] |= int8Quantize(v[4 * k + j], inv) << (8 * j);
      }
    }
    if (p[i].at >= 0) *reinterpret_cast<uint2*>(q + p[i].at) = make_uint2(o[0], o[1]);
    const uint32_t s = s0 + i * kThreads;
    if ((s & 3) == 0 && s < slots) e[s >> 2] = (uint8_t)ex;
  }
}

__global__ void __launch_bounds__(kThreads)
    dequantizePieces(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                     uint16_t* __restrict__ x, uint32_t slots, uint32_t perRow, int cols) {
  const uint32_t s0 = blockIdx.x * (kThreads * kPieces) + threadIdx.x;
  Piece p[kPieces];
  uint2 u[kPieces];
  uint32_t ex[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    p[i] = pieceAt(s0 + i * kThreads, slots, perRow, cols);
    u[i] = make_uint2(0u, 0u);
    ex[i] = 0u;
    if (p[i].at < 0) continue;
    u[i] = __ldcs(reinterpret_cast<const uint2*>(q + p[i].at));
    ex[i] = __ldg(e + ((s0 + i * kThreads) >> 2));
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    if (p[i].at < 0) continue;
    const float step = int8Step(ex[i]);
    const uint2 a = tobf4(int8x4(u[i].x, step)), b = tobf4(int8x4(u[i].y, step));
    *reinterpret_cast<uint4*>(x + p[i].at) = make_uint4(a.x, a.y, b.x, b.y);
  }
}

// Whether the piece kernels take these rows, and their piece counts.
struct PieceGrid {
  bool fits;
  uint32_t slots, perRow;
  unsigned ctas;
};
PieceGrid pieceGrid(const void* x, const void* q, int64_t rows, int cols, int blocks) {
  const int64_t perRow = 4 * (int64_t)blocks, slots = rows * perRow;
  PieceGrid g{cols % 8 == 0 && slots < (1ll << 31) && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                  (reinterpret_cast<uintptr_t>(q) & 7) == 0,
              (uint32_t)slots, (uint32_t)perRow, 0};
  g.ctas = (unsigned)((slots + kThreads * kPieces - 1) / (kThreads * kPieces));
  return g;
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
  const PieceGrid g = pieceGrid(x, q, rows, cols, blocks);
  if (!x_f32 && g.fits)
    quantizePieces<<<g.ctas, kThreads, 0, stream>>>(static_cast<const uint16_t*>(x), q, e, g.slots,
                                                    g.perRow, cols);
  else if (x_f32)
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
  const PieceGrid g = pieceGrid(x, q, rows, cols, blocks);
  if (!x_f32 && g.fits)
    dequantizePieces<<<g.ctas, kThreads, 0, stream>>>(q, e, static_cast<uint16_t*>(x), g.slots,
                                                      g.perRow, cols);
  else if (x_f32)
    dequantizeInt8<<<gridFor(rows * blocks), kThreads, 0, stream>>>(q, e, static_cast<float*>(x),
                                                                   rows, cols, blocks);
  else
    dequantizeInt8<<<gridFor(rows * blocks), kThreads, 0, stream>>>(
        q, e, static_cast<uint16_t*>(x), rows, cols, blocks);
  return launched(cudaGetLastError());
}
