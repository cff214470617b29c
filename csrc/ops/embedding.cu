// embedding.cu - token and position embedding, and the gradient of a table by
// its tokens.
//
//   y[r]  = scale w[token[r]] + p[position[r]]
//   dw[v] = scale sum over r with token[r] = v of g[r]   (likewise dp)
//
// An index outside its table contributes nothing: zero to y, and no gradient.
// Sums are fp32 in row order, whatever the launch, and are rounded once to the
// table's type.
#include "common.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float loadAs(const uint16_t* p) { return bf2f(*p); }
__device__ __forceinline__ float loadAs(const float* p) { return *p; }
__device__ __forceinline__ void storeAs(uint16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void storeAs(float* p, float v) { *p = v; }

// One CTA per row.
template <class W, class Y>
__global__ void __launch_bounds__(kThreads)
    embeddingFwd(const int64_t* __restrict__ token, const int64_t* __restrict__ position,
                 const W* __restrict__ w, const W* __restrict__ p, Y* __restrict__ y, int seq,
                 int vocab, int context, int cols, float scale) {
  const int64_t r = blockIdx.x;
  const int64_t t = token[r], at = position ? position[r] : r % seq;
  const bool hasW = t >= 0 && t < vocab, hasP = p != nullptr && at >= 0 && at < context;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float a = hasW ? loadAs(w + t * cols + c) * scale : 0.f;
    storeAs(y + r * cols + c, hasP ? a + loadAs(p + at * cols + c) : a);
  }
}

// One CTA per 32 table rows and 256 columns: it looks through all tokens in
// order, lists those of its rows, and adds their gradients row by row.
constexpr int kRows = 32;
template <class G, class W>
__global__ void __launch_bounds__(kThreads)
    embeddingGrad(const G* __restrict__ g, const int64_t* __restrict__ token,
                  W* __restrict__ dw, int64_t rows, int seq, int vocab, int cols, float scale) {
  __shared__ float acc[kRows][kThreads];
  __shared__ int sRow[kThreads], sSlot[kThreads], sBase[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int v0 = blockIdx.x * kRows;
  const int c = blockIdx.y * kThreads + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kRows; ++i) acc[i][threadIdx.x] = 0.f;
  for (int64_t r0 = 0; r0 < rows; r0 += kThreads) {
    const int64_t r = r0 + threadIdx.x;
    const int64_t t = r >= rows ? -1 : token ? token[r] : r % seq;
    const bool mine = t >= v0 && t < v0 + kRows && t < vocab;
    const uint32_t votes = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) sBase[warp] = __popc(votes);
    __syncthreads();
    int before = 0, total = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
      before += i < warp ? sBase[i] : 0;
      total += sBase[i];
    }
    if (mine) {
      const int at = before + __popc(votes & ((1u << lane) - 1u));
      sRow[at] = threadIdx.x;
      sSlot[at] = (int)(t - v0);
    }
    __syncthreads();
    if (c < cols)
      for (int i = 0; i < total; ++i)
        acc[sSlot[i]][threadIdx.x] += loadAs(g + (r0 + sRow[i]) * cols + c);
    __syncthreads();
  }
  if (c < cols)
    for (int i = 0; i < kRows && v0 + i < vocab; ++i)
      storeAs(dw + (int64_t)(v0 + i) * cols + c, scale * acc[i][threadIdx.x]);
}

template <class W, class Y>
int fwd(const int64_t* token, const int64_t* position, const void* w, const void* p, void* y,
        int64_t rows, int seq, int vocab, int context, int cols, float scale,
        cudaStream_t stream) {
  embeddingFwd<<<(unsigned)rows, kThreads, 0, stream>>>(
      token, position, static_cast<const W*>(w), static_cast<const W*>(p), static_cast<Y*>(y), seq,
      vocab, context, cols, scale);
  return launched(cudaGetLastError());
}

template <class G, class W>
int grad(const void* g, const int64_t* token, void* dw, int64_t rows, int seq, int vocab, int cols,
         float scale, cudaStream_t stream) {
  const dim3 grid((unsigned)((vocab + kRows - 1) / kRows),
                  (unsigned)((cols + kThreads - 1) / kThreads));
  embeddingGrad<<<grid, kThreads, 0, stream>>>(static_cast<const G*>(g), token,
                                               static_cast<W*>(dw), rows, seq, vocab, cols, scale);
  return launched(cudaGetLastError());
}

}  // namespace
}  // namespace tnops

using namespace tnops;

extern "C" int tnops_embedding_fwd(const int64_t* token, const int64_t* position, const void* w,
                                   const void* p, int w_f32, void* y, int y_f32, int64_t rows,
                                   int seq, int vocab, int context, int cols, float scale,
                                   cudaStream_t stream) {
  if (rows <= 0 || rows > INT32_MAX || seq <= 0 || vocab <= 0 || cols <= 0 || (p && context <= 0))
    return 1;
  if (w_f32)
    return y_f32 ? fwd<float, float>(token, position, w, p, y, rows, seq, vocab, context, cols,
                                     scale, stream)
                 : fwd<float, uint16_t>(token, position, w, p, y, rows, seq, vocab, context, cols,
                                        scale, stream);
  return y_f32 ? fwd<uint16_t, float>(token, position, w, p, y, rows, seq, vocab, context, cols,
                                      scale, stream)
               : fwd<uint16_t, uint16_t>(token, position, w, p, y, rows, seq, vocab, context,
                                         cols, scale, stream);
}

extern "C" int tnops_embedding_grad(const void* g, int g_f32, const int64_t* token, int seq,
                                    void* dw, int dw_f32, int64_t rows, int vocab, int cols,
                                    float scale, cudaStream_t stream) {
  if (rows <= 0 || rows > INT32_MAX || (!token && seq <= 0) || vocab <= 0 || cols <= 0) return 1;
  if (g_f32)
    return dw_f32 ? grad<float, float>(g, token, dw, rows, seq, vocab, cols, scale, stream)
                  : grad<float, uint16_t>(g, token, dw, rows, seq, vocab, cols, scale, stream);
  return dw_f32 ? grad<uint16_t, float>(g, token, dw, rows, seq, vocab, cols, scale, stream)
                : grad<uint16_t, uint16_t>(g, token, dw, rows, seq, vocab, cols, scale, stream);
}
