// linear_ce.cu - a linear layer over a large vocabulary and its softmax
// cross-entropy, without the [rows, classes] logits in memory.
//
//   l[r, v] = sum_c x[r, c] w[v, c]
//   lse[r]  = log sum_v exp(l[r, v]),   loss[r] = lse[r] - l[r, target[r]]
//   d[r, v] = k[r] (exp(l[r, v] - lse[r]) - [v = target[r]])
//   dx = d w,   dw = d^T x
//
// with k[r] the gradient that arrives at loss[r] (0 for a row whose target is
// no class). The forward pass is one GEMM whose epilogue keeps, per row and
// 128 columns, the largest logit and the sum of exponentials below it (fp32,
// from the fp32 accumulators: no logit is rounded), and a second kernel joins
// them. The backward pass goes over the vocabulary in pieces: a GEMM forms the
// piece's logits again and writes d for it (bf16, the operand type of the two
// products that follow; a factor that all rows share is left to the products'
// fp32 results: rounded into every d it would scale the whole gradient by up to
// 2^-8), and one launch of linear_grads.cu forms this piece's
// rows of dw and adds its share to dx (fp32 between pieces). Beyond its inputs
// and outputs the backward pass holds one piece of d and, with more than one
// piece, dx in fp32.
// 8 rows classes width operations, 2 of them for the logits formed twice.
#include "linear_grads.h"
#include "panel_gemm.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// v[at], kept in registers (a loop of selects becomes an array in memory).
__device__ __forceinline__ float valueAt(const float (&v)[32], int at) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.s32 p, %1, %2;\n\t"
        "@p mov.f32 %0, %3;\n\t}"
        : "+f"(t)
        : "r"(at), "r"(i), "f"(v[i]));
  return t;
}

// The bf16 number `bits` in place of number `at` of 16 pairs, likewise.
__device__ __forceinline__ void putBf16(uint32_t (&w)[16], int at, uint32_t bits) {
  const uint32_t order = (at & 1) ? 0x5410u : 0x3254u;  // bytes of (pair, bits)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t with = __byte_perm(w[i], bits, order);
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.s32 p, %1, %2;\n\t"
        "@p mov.b32 %0, %3;\n\t}"
        : "+r"(w[i])
        : "r"(at >> 1), "r"(i), "r"(with));
  }
}

// Running maximum and sum of exponentials of one row over 128 columns.
struct StatsEpi {
  const int64_t* target;
  float2* partial;  // [2 * tilesN][rows]: (maximum, sum of exp(l - maximum))
  float* logitOfTarget;
  int rows, classes;

  struct State {
    float m, s;
    int64_t target;
  };
  __device__ __forceinline__ State begin(int row) const {
    return {-INFINITY, 0.f, row < rows ? target[row] : -1};
  }
  // 32 logits: their maximum, then its difference to two of them and that times
  // log2 e in one packed instruction each, one ex2 for each and one packed
  // addition for two. The difference comes first: it is exact where it counts,
  // the largest logit adds exactly 1 and an unchanged maximum leaves the sum as
  // it is, so that lse is never below a logit. (One FMA with -maximum log2 e
  // scales every term by that product's rounding, up to 2^-14 of them at logits of 1000.)
  __device__ __forceinline__ int ahead(int) const { return 0; }
  __device__ __forceinline__ void chunk(State& st, const float (&in)[32], int, int row,
                                        int col0) const {
    if (col0 >= classes) return;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = in[i];
    if (col0 + 32 > classes) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = col0 + i < classes ? in[i] : -INFINITY;
    }
    const int64_t at = st.target - col0;
    if (at >= 0 && at < 32 && st.target < classes)
      logitOfTarget[row] = valueAt(v, (int)at);
    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], v[i]);
    const float m = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), st.m);
    // fmaxf passes over NaNs: with none but those and -inf so far the maximum is
    // -inf, and the sum is taken all the same, from 0, so that a NaN stays in it.
    const float nm = m == -INFINITY ? 0.f : -m;
    const uint64_t scale = pack2(kLog2e, kLog2e), shift = pack2(nm, nm);
    uint64_t s[4] = {pack2(st.s * ex2Approx((st.m + nm) * kLog2e), 0.f), 0ull, 0ull, 0ull};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      unpack2(mul2(add2(pack2(v[2 * i], v[2 * i + 1]), shift), scale), a, b);
      s[i & 3] = add2(s[i & 3], pack2(ex2Approx(a), ex2Approx(b)));
    }
    float a, b;
    unpack2(add2(add2(s[0], s[1]), add2(s[2], s[3])), a, b);
    st.m = m;
    st.s = a + b;
  }
  __device__ __forceinline__ void end(const State& st, int row, int part) const {
    if (row < rows) partial[(size_t)part * rows + row] = make_float2(st.m, st.s);
  }
};

// d for one piece of the vocabulary, from lse of the whole row.
struct SoftmaxGradEpi {
  uint16_t* d;  // [rows, ld]
  const int64_t* target;
  const float* lse;
  const float* grad;  // gradient of each row's loss, or null for 1
  int ld, rows, classes, first, width;

  // |k| exp(l - lse) = 2^(l log2e + nb) with nb = log2 |k| - lse log2e: the
  // factor costs nothing per logit; k's sign goes on the packed results. The
  // rounding of nb scales a row's d by up to 2^-14 at logits of 1000, less than
  // bf16's 2^-8, but p - 1 of a sure row would be all error: the target's own
  // takes the difference first.
  struct State {
    float nb, lse, k;
    int at;               // the target's column in this piece (any other value: none)
    uint32_t keep, sign;  // masks of a pair of bf16: all or nothing, k's sign
  };
  __device__ __forceinline__ State begin(int row) const {
    State st{0.f, 0.f, 0.f, -1, 0u, 0u};
    if (row < rows) {
      const int64_t t = target[row];
      if (t >= 0 && t < classes) {
        st.k = grad != nullptr ? grad[row] : 1.f;
        st.lse = lse[row];
        st.nb = -st.lse * kLog2e;
        if (grad != nullptr) st.nb += log2f(fabsf(st.k));
        st.at = (int)(t - first);
        st.keep = 0xffffffffu;
        st.sign = st.k < 0.f ? 0x80008000u : 0u;
      }
    }
    return st;
  }
  __device__ __forceinline__ int ahead(int) const { return 0; }
  __device__ __forceinline__ void chunk(State& st, const float (&v)[32], int, int row,
                                        int col0) const {
    if (row >= rows || col0 >= width) return;
    const uint64_t scale = pack2(kLog2e, kLog2e), shift = pack2(st.nb, st.nb);
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      unpack2(fma2(pack2(v[2 * i], v[2 * i + 1]), scale, shift), a, b);
      // A row that does not count gives zeros whatever its logits are.
      w[i] = (packBf16(ex2Approx(a), ex2Approx(b)) & st.keep) ^ st.sign;
    }
    const int at = st.at - col0;
    if (at >= 0 && at < 32) {
      // The target's own: k (p - 1), rounded once.
      const float l = valueAt(v, at);
      const float d = st.k * (ex2Approx((l - st.lse) * kLog2e) - 1.f);
      putBf16(w, at, f2bf(d));
    }
    // Whole: d's rows are `ld` apart, a multiple of 32 at or past the width.
    storeRow32(d + (size_t)row * ld + col0, w, true, 4);
  }
  __device__ __forceinline__ void end(const State&, int, int) const {}
};

// (maximum, sum) of two sets; -inf and 0 stand for an empty one.
__device__ __forceinline__ float2 joinSums(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, a.y + b.y);
  return make_float2(m, a.y * ex2Approx((a.x - m) * kLog2e) + b.y * ex2Approx((b.x - m) * kLog2e));
}

// Joins a row's partial statistics: eight rows per CTA, the parts dealt to 32
// threads of each row, four loads in flight; then the threads' sums in a fixed
// tree. loss comes in with the targets' logits.
constexpr int kJoinRows = 8, kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads)
    joinStats(const float2* __restrict__ partial, const int64_t* __restrict__ target,
              float* __restrict__ lse, float* __restrict__ loss, int parts, int rows,
              int classes) {
  __shared__ float2 s[kJoinThreads / 32][kJoinRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * kJoinRows + (lane & (kJoinRows - 1));
  constexpr int U = 4, kStep = kJoinThreads / kJoinRows;
  float2 st = make_float2(-INFINITY, 0.f);
  if (row < rows)
    for (int p = threadIdx.x / kJoinRows; p < parts; p += U * kStep) {
      float2 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = p + u * kStep < parts ? partial[(size_t)(p + u * kStep) * rows + row]
                                     : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) st = joinSums(st, v[u]);
    }
#pragma unroll
  for (int d = kJoinRows; d < 32; d *= 2)
    st = joinSums(st, make_float2(__shfl_xor_sync(0xffffffffu, st.x, d),
                                  __shfl_xor_sync(0xffffffffu, st.y, d)));
  if (lane < kJoinRows) s[warp][lane] = st;
  __syncthreads();
  if (threadIdx.x < kJoinRows && row < rows) {
#pragma unroll
    for (int w = 1; w < kJoinThreads / 32; ++w) st = joinSums(st, s[w][lane]);
    const float l = st.x + logf(st.y);
    const int64_t t = target[row];
    lse[row] = l;
    loss[row] = t >= 0 && t < classes ? l - loss[row] : 0.f;
  }
}

// out = the sum of the losses, or their mean over the rows that count;
// share = 1 / the number of rows that count (at least one). One CTA, fixed
// order.
constexpr int kMeanThreads = 1024;
__global__ void __launch_bounds__(kMeanThreads)
    meanLoss(const float* __restrict__ loss, const int64_t* __restrict__ target, int rows,
             int classes, int mean, float* __restrict__ out, float* __restrict__ share) {
  __shared__ float sSum[32];
  __shared__ int sCount[32];
  float sum = 0.f;
  int count = 0;
  for (int r = threadIdx.x; r < rows; r += kMeanThreads) {
    sum += loss[r];
    const int64_t t = target[r];
    count += t >= 0 && t < classes;
  }
  sum = warpSum(sum);
  count = __reduce_add_sync(0xffffffffu, count);
  if ((threadIdx.x & 31) == 0) {
    sSum[threadIdx.x >> 5] = sum;
    sCount[threadIdx.x >> 5] = count;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = warpSum(sSum[threadIdx.x]);
    count = __reduce_add_sync(0xffffffffu, sCount[threadIdx.x]);
    if (threadIdx.x == 0) {
      const float s = 1.0f / (float)(count > 0 ? count : 1);
      *out = mean ? sum * s : sum;
      *share = s;
    }
  }
}

__global__ void f32ToBf16(const float* __restrict__ in, uint16_t* __restrict__ out, size_t n4) {
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += stride)
    reinterpret_cast<uint2*>(out)[i] = tobf4(reinterpret_cast<const float4*>(in)[i]);
}

int tilesOf(int n) { return (n + 255) / 256; }

}  // namespace

unsigned linearCeStatus(int reset) { return readStatus(reset); }

}  // namespace tnops

using namespace tnops;

extern "C" int tnops_linear_ce_parts(int classes) { return 2 * tilesOf(classes); }

extern "C" int tnops_linear_ce_fwd(const void* x, const void* w, const int64_t* target,
                                   float* loss, float* lse, float* partial, int rows, int width,
                                   int classes, cudaStream_t stream) {
  if (rows <= 0 || classes <= 0 || width <= 0 || width % 8 != 0 || !aligned16(x) ||
      !aligned16(w))
    return 1;
  PanelGemmArgs<StatsEpi> args{};
  args.epi = {target, reinterpret_cast<float2*>(partial), loss, rows, classes};
  if (int rc = launchPanelGemm(args, x, w, rows, classes, width, stream)) return rc;
  joinStats<<<(rows + kJoinRows - 1) / kJoinRows, kJoinThreads, 0, stream>>>(
      args.epi.partial, target, lse, loss, tnops_linear_ce_parts(classes), rows, classes);
  return launched(cudaGetLastError());
}

extern "C" int tnops_linear_ce_mean(const float* loss, const int64_t* target, float* out,
                                    float* share, int rows, int classes, int mean,
                                    cudaStream_t stream) {
  if (rows <= 0) return 1;
  meanLoss<<<1, kMeanThreads, 0, stream>>>(loss, target, rows, classes, mean, out, share);
  return launched(cudaGetLastError());
}

// Classes per piece: whole 256-wide tiles, spread evenly over the least number
// of pieces whose d fits the budget, or over up to five more where their
// products leave fewer SM pairs idle (16384 rows of 50257 classes and 512 MiB:
// six pieces instead of four, a tenth less). A piece costs about 20 K blocks
// of launches besides.
extern "C" int tnops_linear_ce_piece(int rows, int width, int classes, int64_t budget) {
  if (rows <= 0 || width <= 0 || classes <= 0) return 0;
  const int64_t tiles = ((int64_t)classes + 255) / 256;
  int64_t most = budget / ((int64_t)rows * 512);
  if (most < 1) most = 1;
  const int64_t least = (tiles + most - 1) / most;
  int64_t best = 0, bestCost = 0;
  for (int64_t n = least; n <= tiles && n < least + 6; ++n) {
    const int64_t piece = (tiles + n - 1) / n * 256;
    const int whole = (int)(classes / piece), last = (int)(classes - whole * piece);
    int64_t cost = 20 * (whole + (last > 0));
    if (whole > 0) cost += whole * (int64_t)linearGradsCost(rows, (int)piece, width);
    if (last > 0) cost += linearGradsCost(rows, last, width);
    if (best == 0 || cost < bestCost) {
      best = piece;
      bestCost = cost;
    }
  }
  return (int)best;
}

// Rows of padding after the classes that the last piece's product writes; more
// of them are left to a memset.
static int paddedRows(int classes, int vocab) {
  return vocab - classes < 256 ? vocab - classes : 0;
}

extern "C" size_t tnops_linear_ce_scratch(int rows, int width, int classes, int vocab, int piece,
                                          int want_dx, int want_dw) {
  if (rows <= 0 || width <= 0 || classes <= 0 || vocab < classes || piece <= 0) return 0;
  const int last = (classes - 1) % piece + 1;
  const size_t a = last == classes ? 0
                                   : linearGradsScratch(rows, piece, 0, width, want_dx, want_dw),
               b = linearGradsScratch(rows, last, paddedRows(classes, vocab), width, want_dx,
                                      want_dw);
  return a > b ? a : b;
}

extern "C" int tnops_linear_ce_bwd(const void* x, const void* w, const int64_t* target,
                                   const float* lse, const float* grad, int grad_step,
                                   const float* share, void* d, int piece, float* dx_f32,
                                   void* scratch, size_t scratch_bytes, void* dx, void* dw,
                                   int dw_f32, int rows, int width, int classes, int vocab,
                                   cudaStream_t stream) {
  if (rows <= 0 || classes <= 0 || vocab < classes || width <= 0 || width % 8 != 0 ||
      piece <= 0 || piece % 32 != 0 || (grad_step != 0 && grad_step != 1) || !aligned16(x) ||
      !aligned16(w) || (reinterpret_cast<uintptr_t>(d) & 31) ||
      (dx && !aligned16(dx)) || (dw && !aligned16(dw)))
    return 1;
  const bool whole = classes <= piece;
  if (!aligned16(scratch)) return 1;
  if (dx && !whole && (dx_f32 == nullptr || !aligned16(dx_f32))) return 1;
  const size_t dwSize = dw_f32 ? 4 : 2;
  const int padded = paddedRows(classes, vocab);
  if (dw && vocab > classes + padded) {
    const cudaError_t e = cudaMemsetAsync(static_cast<char*>(dw) + dwSize * width * (size_t)classes,
                                          0, dwSize * width * (size_t)(vocab - classes), stream);
    if (e != cudaSuccess) return (int)e;
  }
  for (int first = 0; first < classes; first += piece) {
    const int n = classes - first < piece ? classes - first : piece;
    const void* wPiece = static_cast<const uint16_t*>(w) + (size_t)first * width;
    PanelGemmArgs<SoftmaxGradEpi> args{};
    SoftmaxGradEpi& e = args.epi;
    e.d = static_cast<uint16_t*>(d);
    e.ld = piece;
    e.target = target;
    e.lse = lse;
    e.grad = grad_step ? grad : nullptr;
    e.rows = rows;
    e.classes = classes;
    e.first = first;
    e.width = n;
    if (int rc = launchPanelGemm(args, x, wPiece, rows, n, width, stream)) return rc;
    LinearGrads g{};
    g.scale[0] = grad_step ? nullptr : grad;
    g.scale[1] = share;
    g.scratch = scratch;
    g.scratchBytes = scratch_bytes;
    g.g = d;
    g.ldg = piece;
    g.w = wPiece;
    g.x = x;
    g.dx = whole ? dx : dx_f32;
    g.dxStore = !dx ? kStoreNone : whole ? kStoreBf16 : first == 0 ? kStoreF32 : kAddF32;
    g.dw = dw ? static_cast<char*>(dw) + dwSize * width * (size_t)first : nullptr;
    g.dwStore = !dw ? kStoreNone : dw_f32 ? kStoreF32 : kStoreBf16;
    g.rows = rows;
    g.outs = n;
    g.ins = width;
    g.padded = first + n == classes ? padded : 0;
    if (int rc = linearGrads(g, stream)) return rc;
  }
  if (dx && !whole) {
    const size_t n4 = (size_t)rows * width / 4;
    const size_t blocks = (n4 + 255) / 256;
    f32ToBf16<<<(unsigned)(blocks < kSMs * 8 ? blocks : kSMs * 8), 256, 0, stream>>>(
        dx_f32, static_cast<uint16_t*>(dx), n4);
    return launched(cudaGetLastError());
  }
  return 0;
}
