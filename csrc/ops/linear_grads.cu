// linear_grads.cu - both products of a linear layer's backward pass in one
// launch of the CTA-pair pipeline (pair_gemm.cuh):
//
//   dX[r, k] = sum_n G[r, n] W[n, k]      A = G (K-major),  B = W (MN-major)
//   dW[n, k] = sum_r G[r, n] X[r, k]      A = G (MN-major), B = X (MN-major)
//
// G, W and X are read as they lie. 4 rows outs ins operations; each operand
// is read once per 256 rows or columns of the other side, from L2 when the
// neighbouring pairs work on the same rows. A layer's dW has few tiles with
// long sums (27 of 128 K blocks for 8192 rows of a 768 -> 2304 layer, next to
// 96 of 36 for dX, on 74 pairs), so the tiles that fill no whole round are cut
// along the sum (pair_schedule.h) and joined by a second kernel.
#include "linear_grads.h"
#include "pair_gemm.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

struct StoreEpi {
  static constexpr bool kCuts = true;
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

struct JoinArgs {
  PairSchedule schedule;
  const float* partial;  // [2 * pairs][256][256]
  void* out[2];
  int rows[2], cols[2], tilesN[2], mode[2];
};

// Adds the parts of a cut tile in pair order and writes 8 of its rows
// (blockIdx.y): one CTA per pair whose part is a tile's first. Bound by memory
// (L2 for the most part): at most 2 * 74 parts of 256 KiB.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads)
    joinCutTiles(const __grid_constant__ JoinArgs a) {
  CutTile c;
  if (!cutTileOf(a.schedule, (int)blockIdx.x, &c)) return;
  const int tileM = c.tile / a.tilesN[c.which], tileN = c.tile % a.tilesN[c.which];
  const int rows = a.rows[c.which], cols = a.cols[c.which], mode = a.mode[c.which];
  const int col = (threadIdx.x & 63) * 4, outCol = tileN * 256 + col;
  float4 acc[2] = {};
  for (int q = (int)blockIdx.x; q < a.schedule.pairs && a.schedule.restStart(q) < c.end; ++q) {
    const int slot = cutSlot(a.schedule, c, q);
    if (slot < 0) continue;
    const float* part = a.partial + (size_t)(2 * q + slot) * 65536;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = blockIdx.y * 8 + (threadIdx.x >> 6) + 4 * i;
      const float4 v = __ldcs(reinterpret_cast<const float4*>(part + r * 256 + col));
      acc[i].x += v.x; acc[i].y += v.y; acc[i].z += v.z; acc[i].w += v.w;
    }
  }
  if (outCol >= cols) return;  // cols % 8 == 0: a thread's four are in or out
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = tileM * 256 + blockIdx.y * 8 + (threadIdx.x >> 6) + 4 * i;
    if (row >= rows) continue;
    const size_t at = (size_t)row * cols + outCol;
    if (mode == kStoreBf16) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out[c.which]) + at) = tobf4(acc[i]);
    } else {
      float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.out[c.which]) + at);
      if (mode == kAddF32) {
        const float4 o = *out;
        acc[i].x += o.x; acc[i].y += o.y; acc[i].z += o.z; acc[i].w += o.w;
      }
      *out = acc[i];
    }
  }
}

}  // namespace

int linearGrads(const LinearGrads& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.outs <= 0 || a.ins <= 0 || a.ldg < a.outs) return 1;
  if (a.ldg % 8 != 0 || a.ins % 8 != 0) return 1;  // 16-byte rows (TMA)
  if (!aligned16(a.g) || (a.dxStore && (!aligned16(a.w) || !aligned16(a.dx))) ||
      (a.dwStore && (!aligned16(a.x) || !aligned16(a.dw))) || a.scratch == nullptr ||
      !aligned16(a.scratch))
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
  const int sms = smPairs(), pairs = sms < kSMs / 2 ? sms : kSMs / 2;
  planGemm(&args, pairs, true);
  if (!f32OutMap(&args.mapPartial, a.scratch, (int64_t)2 * pairs * kPairBM, 256, 256)) return 4;
  if (int rc = launchPairGemm(args, stream)) return rc;
  if (args.schedule.restBlocks() == 0) return 0;
  JoinArgs join{};
  join.schedule = args.schedule;
  join.partial = static_cast<const float*>(a.scratch);
  for (int i = 0; i < args.problems; ++i) {
    join.out[i] = args.prob[i].aMn ? a.dw : a.dx;
    join.rows[i] = args.epi.rows[i];
    join.cols[i] = args.epi.cols[i];
    join.tilesN[i] = args.prob[i].tilesN;
    join.mode[i] = args.epi.mode[i];
  }
  joinCutTiles<<<dim3((unsigned)pairs, 32), kJoinThreads, 0, stream>>>(join);
  return launched(cudaGetLastError());
}

unsigned linearGradsStatus(int reset) { return readStatus(reset); }

}  // namespace tnops

using namespace tnops;

extern "C" size_t tnops_linear_grads_scratch(void) {
  return (size_t)kSMs * 256 * 256 * sizeof(float);  // two slots for each of kSMs / 2 pairs
}

extern "C" int tnops_linear_grads(const void* g, int64_t ldg, const void* w, const void* x,
                                  void* dx, void* dw, int dw_f32, int rows, int outs, int ins,
                                  void* scratch, cudaStream_t stream) {
  if (g == nullptr || (dx && !w) || (dw && !x)) return 1;
  LinearGrads a{g, ldg, w, x, dx, dw, scratch, dx ? kStoreBf16 : kStoreNone,
                dw ? (dw_f32 ? kStoreF32 : kStoreBf16) : kStoreNone, rows, outs, ins};
  return linearGrads(a, stream);
}
