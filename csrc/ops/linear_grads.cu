// linear_grads.cu - both products of a linear layer's backward pass in one
// launch of the CTA-pair pipeline (pair_gemm.cuh):
//
//   dX[r, k] = sum_n G[r, n] W[n, k]      A = G (K-major),  B = W (MN-major)
//   dW[n, k] = sum_r G[r, n] X[r, k]      A = G (MN-major), B = X (MN-major)
//
// G, W and X are read as they lie. 4 rows outs ins operations; each operand
// is read once per 256 or 512 rows or columns of the other side, from L2 when
// the neighbouring pairs work on the same rows. A layer's dW has few tiles with
// long sums (15 of 128 K blocks for 8192 rows of a 768 -> 2304 layer, next to
// 48 of 36 for dX, on 74 pairs): the schedule (pair_schedule.h) lets the pairs
// without a long tile begin with the short ones, and where that still leaves
// pairs idle it cuts the long sums, whose parts a second kernel adds.
#include "linear_grads.h"

#include "pair_gemm.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

struct JoinArgs {
  const float* partial;  // [split * tiles][512][256]
  void* out;
  int tiles, tilesN, split, rows, cols, mode;
};

// Adds the parts of a cut tile (blockIdx.x) in the order of the sum and writes
// 16 of its rows (blockIdx.y). Bound by memory, L2 for the most part.
constexpr int kJoinThreads = 256, kJoinRows = 16;
__global__ void __launch_bounds__(kJoinThreads)
    joinCutTiles(const __grid_constant__ JoinArgs a) {
  const int tile = (int)blockIdx.x;
  const int col = (threadIdx.x & 63) * 4, outCol = tile % a.tilesN * 256 + col;
  const int r0 = blockIdx.y * kJoinRows + (threadIdx.x >> 6);
  if (outCol >= a.cols) return;  // cols % 8 == 0: a thread's four are in or out
  float4 acc[kJoinRows / 4] = {};
  for (int p = 0; p < a.split; ++p) {
    const float* part = a.partial + ((size_t)p * a.tiles + tile) * (kPairBM * 256);
#pragma unroll
    for (int i = 0; i < kJoinRows / 4; ++i) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(part + (r0 + 4 * i) * 256 + col));
      acc[i].x += v.x; acc[i].y += v.y; acc[i].z += v.z; acc[i].w += v.w;
    }
  }
#pragma unroll
  for (int i = 0; i < kJoinRows / 4; ++i) {
    const int row = tile / a.tilesN * kPairBM + r0 + 4 * i;
    if (row >= a.rows) continue;
    const size_t at = (size_t)row * a.cols + outCol;
    if (a.mode == kStoreBf16) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = tobf4(acc[i]);
    } else {
      float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
      if (a.mode == kAddF32) {
        const float4 o = *out;
        acc[i].x += o.x; acc[i].y += o.y; acc[i].z += o.z; acc[i].w += o.w;
      }
      *out = acc[i];
    }
  }
}

// Tile counts and sums of the launch: the product with the longer sum first.
// kinds[i]: whether product i is dX.
int shapes(int rows, int outs, int padded, int ins, bool wantDx, bool wantDw, GemmProblem* prob,
           bool* isDx) {
  int n = 0;
  auto add = [&](bool dx) {
    GemmProblem& p = prob[n];
    p.real = dx ? rows : outs;
    p.rows = dx ? rows : outs + padded;
    p.tilesM = (p.rows + kPairBM - 1) / kPairBM;
    p.tilesN = (ins + 255) / 256;
    p.kBlocks = ((dx ? outs : rows) + kBK - 1) / kBK;
    p.aMn = dx ? 0 : 1;
    isDx[n++] = dx;
  };
  const bool dxFirst = outs >= rows;
  if (wantDx && dxFirst) add(true);
  if (wantDw) add(false);
  if (wantDx && !dxFirst) add(true);
  return n;
}

size_t scratchFor(const PairSchedule& s) {
  return (size_t)s.slots() * kPairBM * 256 * sizeof(float);
}

}  // namespace

int linearGrads(const LinearGrads& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.outs <= 0 || a.ins <= 0 || a.padded < 0 || a.ldg < a.outs) return 1;
  if (a.ldg % 8 != 0 || a.ins % 8 != 0) return 1;  // 16-byte rows (TMA)
  if (!aligned16(a.g) || (a.dxStore && (!aligned16(a.w) || !aligned16(a.dx))) ||
      (a.dwStore && (!aligned16(a.x) || !aligned16(a.dw))) || !aligned16(a.scratch))
    return 1;
  PairGemmArgs args{};
  bool isDx[2] = {};
  args.scale[0] = a.scale[0];
  args.scale[1] = a.scale[1];
  args.problems = shapes(a.rows, a.outs, a.padded, a.ins, a.dxStore != kStoreNone,
                         a.dwStore != kStoreNone, args.prob, isDx);
  if (args.problems == 0) return 0;
  planGemm(&args);
  const PairSchedule& plan = args.schedule;
  if (scratchFor(plan) > a.scratchBytes || (plan.slots() > 0 && a.scratch == nullptr)) return 1;
  JoinArgs join[2] = {};
  for (int i = 0; i < args.problems; ++i) {
    GemmProblem& p = args.prob[i];
    const int m = p.rows, sum = isDx[i] ? a.outs : a.rows;
    const int mode = isDx[i] ? a.dxStore : a.dwStore;
    void* out = isDx[i] ? a.dx : a.dw;
    args.cols[i] = a.ins;
    args.mode[i] = mode;
    join[i] = {static_cast<const float*>(a.scratch) + (size_t)plan.slotBase(i) * kPairBM * 256,
               out, plan.tiles[i], p.tilesN, plan.split[i], m, a.ins, mode};
    if (!operandMap(&p.mapA, a.g, a.rows, a.outs, a.ldg, !isDx[i]) ||
        !operandMap(&p.mapB, isDx[i] ? a.w : a.x, sum, a.ins, a.ins, true) ||
        !(mode == kStoreBf16 ? bf16OutMap(&args.mapOut[i], out, m, a.ins, a.ins)
                             : f32OutMap(&args.mapOut[i], out, m, a.ins, a.ins)))
      return 4;
  }
  if (plan.slots() > 0 &&
      !f32OutMap(&args.mapPartial, a.scratch, (int64_t)plan.slots() * kPairBM, 256, 256))
    return 4;
  if (int rc = launchPairGemm(args, stream)) return rc;
  for (int i = 0; i < args.problems; ++i) {
    if (plan.split[i] == 1) continue;
    joinCutTiles<<<dim3((unsigned)plan.tiles[i], kPairBM / kJoinRows), kJoinThreads, 0, stream>>>(
        join[i]);
    if (int rc = launched(cudaGetLastError())) return rc;
  }
  return 0;
}

size_t linearGradsScratch(int rows, int outs, int padded, int ins, bool wantDx, bool wantDw) {
  if (rows <= 0 || outs <= 0 || padded < 0 || ins <= 0) return 0;
  PairGemmArgs args{};
  bool isDx[2];
  args.problems = shapes(rows, outs, padded, ins, wantDx, wantDw, args.prob, isDx);
  if (args.problems == 0) return 0;
  planGemm(&args);
  return scratchFor(args.schedule);
}

int linearGradsCost(int rows, int outs, int ins) {
  PairGemmArgs args{};
  bool isDx[2];
  args.problems = shapes(rows, outs, 0, ins, true, true, args.prob, isDx);
  planGemm(&args);
  return planRounds(&args.schedule) + args.schedule.slots() / 2;
}

unsigned linearGradsStatus(int reset) { return readStatus(reset); }

}  // namespace tnops

using namespace tnops;

extern "C" size_t tnops_linear_grads_scratch(int rows, int outs, int ins, int want_dx,
                                             int want_dw) {
  return linearGradsScratch(rows, outs, 0, ins, want_dx != 0, want_dw != 0);
}

extern "C" int tnops_linear_grads(const void* g, int64_t ldg, const void* w, const void* x,
                                  void* dx, void* dw, int dw_f32, int rows, int outs, int ins,
                                  void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  if (g == nullptr || (dx && !w) || (dw && !x)) return 1;
  LinearGrads a{g, ldg, w, x, dx, dw, scratch, scratch_bytes, dx ? kStoreBf16 : kStoreNone,
                dw ? (dw_f32 ? kStoreF32 : kStoreBf16) : kStoreNone, rows, outs, ins, 0,
                {nullptr, nullptr}};
  return linearGrads(a, stream);
}
