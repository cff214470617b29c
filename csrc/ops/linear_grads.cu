// linear_grads.cu - both products of a linear layer's backward pass in one
// launch of the CTA-pair pipeline (pair_gemm.cuh):
//
//   dX[r, k] = sum_n G[r, n] W[n, k]      A = G (K-major),  B = W (MN-major)
//   dW[n, k] = sum_r G[r, n] X[r, k]      A = G (MN-major), B = X (MN-major)
//
// G, W and X are read as they lie. 4 rows outs ins operations; each operand
// is read once per 256 rows or columns of the other side, from L2 when the
// neighbouring pairs work on the same rows. The tiles with the longer sum go
// first, so that the short ones fill the last wave.
#include "linear_grads.h"
#include "pair_gemm.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

struct StoreEpi {
  CUtensorMap mapOut[2];
  int rows[2], cols[2], mode[2];

  struct State {};
  __device__ __forceinline__ State begin(int, int) const { return {}; }
  __device__ __forceinline__ void chunk(State&, const float (&v)[32], int which, int lane,
                                        int row0, int col0, uint32_t buf) const {
    const bool inside = row0 < rows[which] && col0 < cols[which];
    if (mode[which] == kStoreBf16)
      storeBf16(v, lane, buf, &mapOut[which], row0, col0, inside);
    else
      storeF32(v, lane, buf, &mapOut[which], row0, col0, inside, mode[which] == kAddF32);
  }
  __device__ __forceinline__ void end(const State&, int, int) const {}
};

int tilesOf(int n) { return (n + 255) / 256; }

}  // namespace

int linearGrads(const LinearGrads& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.outs <= 0 || a.ins <= 0 || a.ldg < a.outs) return 1;
  if (a.ldg % 8 != 0 || a.ins % 8 != 0) return 1;  // 16-byte rows (TMA)
  if (!aligned16(a.g) || (a.dxStore && (!aligned16(a.w) || !aligned16(a.dx))) ||
      (a.dwStore && (!aligned16(a.x) || !aligned16(a.dw))))
    return 1;
  PairGemmArgs<StoreEpi> args{};
  auto add = [&](bool isDx) {
    const int i = args.problems++;
    GemmProblem& p = args.prob[i];
    const int m = isDx ? a.rows : a.outs, sum = isDx ? a.outs : a.rows;
    p.tilesM = tilesOf(m);
    p.tilesN = tilesOf(a.ins);
    p.kBlocks = (sum + kBK - 1) / kBK;
    p.aMn = isDx ? 0 : 1;
    p.bMn = 1;
    const int mode = isDx ? a.dxStore : a.dwStore;
    args.epi.rows[i] = m;
    args.epi.cols[i] = a.ins;
    args.epi.mode[i] = mode;
    void* out = isDx ? a.dx : a.dw;
    return operandMap(&p.mapA, a.g, a.rows, a.outs, a.ldg, !isDx) &&
           operandMap(&p.mapB, isDx ? a.w : a.x, sum, a.ins, a.ins, true) &&
           (mode == kStoreBf16 ? bf16OutMap(&args.epi.mapOut[i], out, m, a.ins, a.ins)
                               : f32OutMap(&args.epi.mapOut[i], out, m, a.ins, a.ins));
  };
  const bool dxFirst = a.outs >= a.rows;
  bool ok = true;
  if (a.dxStore && dxFirst) ok = ok && add(true);
  if (a.dwStore) ok = ok && add(false);
  if (a.dxStore && !dxFirst) ok = ok && add(true);
  if (!ok) return 4;
  if (args.problems == 0) return 0;
  return launchPairGemm(args, stream);
}

unsigned linearGradsStatus(int reset) { return readStatus(reset); }

}  // namespace tnops

using namespace tnops;

extern "C" int tnops_linear_grads(const void* g, int64_t ldg, const void* w, const void* x,
                                  void* dx, void* dw, int dw_f32, int rows, int outs, int ins,
                                  cudaStream_t stream) {
  if (g == nullptr || (dx && !w) || (dw && !x)) return 1;
  LinearGrads a{g, ldg, w, x, dx, dw, dx ? kStoreBf16 : kStoreNone,
                dw ? (dw_f32 ? kStoreF32 : kStoreBf16) : kStoreNone, rows, outs, ins};
  return linearGrads(a, stream);
}
