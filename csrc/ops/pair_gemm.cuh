// pair_gemm.cuh - the matrix products behind the backward passes of the
// training operators: one persistent CTA-pair pipeline (tcgen05 cta_group::2,
// fp32 accumulators in TMEM).
//
//   D[m, n] = sum_k A(m, k) B(n, k)
//
// A may be K-major or MN-major, B is MN-major (pair_parts.cuh): the products of
// a backward pass (dX = G W, dW = G^T X) read G, W and X as they lie, without a
// transposed copy.
//
// The pipeline is that of the GEMM with the bias epilogue (gemm_tcgen05.cu)
// with tiles of 512 x 256: each CTA of a pair stages, per 64-wide K block, 128
// rows of A for each 256-row half of the tile and 128 rows of B (48 KiB, four
// stages), the even CTA issues the MMAs, and the two halves' accumulators fill
// the 512 TMEM columns. An SM then loads 48 bytes per clock of MMA where a
// 256 x 256 tile takes 64, more than L2 delivers to all SMs at once (8192^3 of
// zeros, so that power does not limit: 1810 TFLOP/s against 1430). With no
// accumulator to spare, an epilogue warp reads all that it has of a half into
// registers and hands the accumulator back before it stores any of it.
// A launch may hold two products (`GemmProblem`), so that dX and dW of a layer
// fill the GPU together; who computes what is pair_schedule.h's. Every wait is
// bounded as there; the first failure is kept in the file's status word.
#pragma once

#include "linear_grads.h"
#include "pair_parts.cuh"
#include "pair_schedule.h"

namespace tnops {
namespace {

constexpr int kPairBM = 512;
constexpr int kPairStages = 4;
constexpr uint32_t kPairStage = 3 * kHalf;  // two halves of A, one of B
constexpr uint32_t kPairSmemBytes = kPairStages * kPairStage + kEpiBytes + 1024;

// One product of a launch. The tensor maps' boxes are {64 k, 128 rows} for a
// K-major A and {64 m, 64 k} for an MN-major operand; out-of-range rows and
// columns read zero, so K, M and N need no padding.
struct alignas(64) GemmProblem {
  CUtensorMap mapA, mapB;
  int tilesM, tilesN, kBlocks;
  int rows;  // m
  int real;  // rows of A; results of those behind are zero, whatever B holds
  int aMn;
};

struct alignas(64) PairGemmArgs {
  GemmProblem prob[2];
  CUtensorMap mapOut[2];
  CUtensorMap mapPartial;  // [512 slots, 256] fp32: parts of cut tiles
  int problems;
  int cols[2];             // n
  int mode[2];             // GradStore
  const float* scale[2];   // factors of every result (null: none)
  PairSchedule schedule;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    pairGemmKernel(const __grid_constant__ PairGemmArgs args) {
  __shared__ __align__(8) uint64_t sFull[kPairStages];
  __shared__ __align__(8) uint64_t sEmpty[kPairStages];
  __shared__ __align__(8) uint64_t sAccFull[2];
  __shared__ __align__(8) uint64_t sAccEmpty[2];
  __shared__ __align__(8) uint64_t sDone;
  __shared__ uint32_t sTmem;
  __shared__ int sAbort;
  extern __shared__ uint8_t dsmem[];
  const uint32_t base = (smemAddr(dsmem) + 1023u) & ~1023u;
  const uint32_t epi0 = base + kPairStages * kPairStage;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = clusterRank();
  const int pair = (int)(blockIdx.x >> 1);
  const PairSchedule& schedule = args.schedule;
  volatile int* abort = &sAbort;

  if (threadIdx.x == 0) {
    sAbort = 0;
    for (int s = 0; s < kPairStages; ++s) {
      mbarInit(&sFull[s], 1);
      mbarInit(&sEmpty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbarInit(&sAccFull[b], 1);
      mbarInit(&sAccEmpty[b], 2 * kEpiWarps);
    }
    mbarInit(&sDone, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smemAddr(&sTmem)),
                 "r"(2 * kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fenceBeforeSync();
  __syncthreads();
  clusterSync();  // barriers initialised and TMEM allocated in both CTAs
  fenceAfterSync();
  const uint32_t tmem = sTmem;

  if (warp == 0 && lane == 0) {
    // Producer (both CTAs): this CTA's halves of A and B.
    uint32_t g = 0;
    PairWalk walk;
    PairWork w;
    walk.init(schedule, pair);
    while (!*abort && walk.next(schedule, &w)) {
      const GemmProblem& p = args.prob[w.which];
      const int m0 = (w.tile / p.tilesN) * kPairBM + (int)rank * 128;
      const bool both = (w.tile / p.tilesN) * kPairBM + 256 < p.rows;  // the second half has rows
      const int n0 = (w.tile % p.tilesN) * 256 + (int)rank * 128;
      const int aMn = p.aMn;
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++g) {
        const uint32_t s = g % kPairStages, round = g / kPairStages;
        if (!mbarWait(&sEmpty[s], (round & 1u) ^ 1u, abort, 1)) break;
        if (rank == 0) mbarExpectTx(&sFull[s], (both ? 6 : 4) * kHalf);  // both CTAs' loads
        const uint32_t bar = inLeader(&sFull[s]), at = base + s * kPairStage;
        loadHalf(at, &p.mapA, aMn, m0, kb * kBK, bar);
        loadHalf(at + 2 * kHalf, &p.mapB, 1, n0, kb * kBK, bar);
        if (both) loadHalf(at + kHalf, &p.mapA, aMn, m0 + 256, kb * kBK, bar);
      }
    }
    if (*abort) {
      if (rank == 0) {
        for (uint32_t q = g > (uint32_t)kPairStages ? g - kPairStages : 0; q < g; ++q)
          mbarWait(&sFull[q % kPairStages], (q / kPairStages) & 1u, abort, 4, true);
      } else {
        // This CTA's loads complete on the even CTA's barriers: let them land.
        const uint64_t t0 = globalTimer();
        while (globalTimer() - t0 < 200000ull) {
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // MMA issuer (even CTA only).
    const bool elected = electOne();
    uint32_t g = 0, local = 0;
    PairWalk walk;
    PairWork w;
    walk.init(schedule, pair);
    bool ok = true;
    for (; ok && walk.next(schedule, &w); ++local) {
      const GemmProblem& p = args.prob[w.which];
      const uint64_t descA = pairDescBase(p.aMn), descB = pairDescBase(1);
      const uint32_t stepA = p.aMn ? 2048 : 32, stepB = 2048;
      const uint32_t instr = pairInstrDesc(p.aMn, 1);
      const int halves = (w.tile / p.tilesN) * kPairBM + 256 < p.rows ? 2 : 1;
      const uint32_t fresh = (local & 1u) ^ 1u;  // phase of an accumulator handed back
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++g) {
        const uint32_t s = g % kPairStages;
        if (!(ok = warpWait(&sFull[s], (g / kPairStages) & 1u, abort, 2))) break;
        fenceAfterSync();
        const uint32_t at = base + s * kPairStage;
        for (int h = 0; h < 2; ++h) {
          // Both accumulators are waited for even where the second half has no
          // rows: its commit below must not come before the epilogue has seen
          // the one before, or a phase of the barrier passes unseen.
          if (kb == w.kb0) {
            if (!(ok = warpWait(&sAccEmpty[h], fresh, abort, 2))) break;
            fenceAfterSync();
          }
          if (h < halves && elected) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              pairMma(tmem + h * kTmemCols, pairDesc(descA, at + h * kHalf + k * stepA),
                      pairDesc(descB, at + 2 * kHalf + k * stepB), instr,
                      kb != w.kb0 || k != 0 ? 1u : 0u);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elected) commitPair(&sEmpty[s]);
        __syncwarp();
      }
      if (!ok) break;
      if (elected) {
        commitPair(&sAccFull[0]);
        commitPair(&sAccFull[1]);
      }
      __syncwarp();
    }
    if (elected) commitPairLocal(&sDone);
    __syncwarp();
    if (*abort) mbarWait(&sDone, 0, abort, 5, true);
  } else if (warp >= 2) {
    // Epilogue (both CTAs): this CTA's 128 rows of each half of the tile; TMEM
    // lane quarter warp % 4, column half (warp - 2) / 4.
    const int quarter = warp & 3, side = (warp - 2) >> 2;
    const uint32_t buf = epi0 + (uint32_t)(warp - 2) * kEpiBuf;
    uint32_t local = 0;
    PairWalk walk;
    PairWork w;
    walk.init(schedule, pair);
    bool ok = true;
    const float scale = (args.scale[0] ? *args.scale[0] : 1.f) *
                        (args.scale[1] ? *args.scale[1] : 1.f);
    for (; ok && walk.next(schedule, &w); ++local) {
      const GemmProblem& p = args.prob[w.which];
      const int tileN = w.tile % p.tilesN;
      for (int h = 0; h < 2; ++h) {
        const int inTile = h * 256 + (int)rank * 128 + quarter * 32;
        const int row0 = (w.tile / p.tilesN) * kPairBM + inTile;
        if (!(ok = warpWait(&sAccFull[h], local & 1u, abort, 3))) break;
        fenceAfterSync();
        const uint32_t acc = tmem + h * kTmemCols + ((uint32_t)(quarter * 32) << 16);
        const bool any = row0 < p.rows;  // the same for the whole warp
        // All of the warp's 32 x 128 first: the accumulator goes back before
        // anything is stored.
        uint32_t r[4][32];
        if (any) {
#pragma unroll
          for (int i = 0; i < 4; ++i) tmemIssue32(acc + (uint32_t)(side * 128 + 32 * i), r[i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) tmemWait(r[i]);
          if (row0 + 32 > p.real && row0 + lane >= p.real) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int k = 0; k < 32; ++k) r[i][k] = 0u;
          }
        }
        fenceBeforeSync();
        __syncwarp();
        if (lane == 0) arriveInLeader(&sAccEmpty[h]);
        if (!any) continue;
        const int mode = args.mode[w.which], cols = args.cols[w.which];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(r[i][k]) * scale;
          const int c = side * 128 + 32 * i, col0 = tileN * 256 + c;
          if (w.slot >= 0)
            storeF32(v, lane, buf, &args.mapPartial, w.slot * kPairBM + inTile, c, true, false);
          else if (mode == kStoreBf16)
            storeBf16(v, lane, buf, &args.mapOut[w.which], row0, col0, col0 < cols);
          else
            storeF32(v, lane, buf, &args.mapOut[w.which], row0, col0, col0 < cols,
                     mode == kAddF32);
        }
      }
    }
    epilogueDrain(lane);
  }
  fenceBeforeSync();
  __syncthreads();
  clusterSync();  // neither CTA leaves while the pair's MMAs or arrivals can reach it
  if (warp == 1) {
    fenceAfterSync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(2 * kTmemCols)
                 : "memory");
  }
}

// -- host side -------------------------------------------------------------------

// Plans the launch for kSMs / 2 pairs. Product 0 must be the one with the
// longer sum.
inline void planGemm(PairGemmArgs* args) {
  PairSchedule& s = args->schedule;
  s = {};
  s.pairs = kSMs / 2;
  for (int i = 0; i < 2; ++i) {
    s.k[i] = 1;
    if (i >= args->problems) continue;
    s.tiles[i] = args->prob[i].tilesM * args->prob[i].tilesN;
    s.k[i] = args->prob[i].kBlocks;
  }
  planPairs(&s, true);
}

// Launches the products of `args`, whose schedule is planned. Returns 0, or a
// non-zero code without a launch.
inline int launchPairGemm(const PairGemmArgs& args, cudaStream_t stream) {
  // Opt in to the shared memory once per device (bit d of `done`).
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 3;
  const uint64_t bit = 1ull << dev;
  if (!(done.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(pairGemmKernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kPairSmemBytes) != cudaSuccess)
      return 3;
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  const PairSchedule& s = args.schedule;
  // In a first round, pairs past the last unit have nothing to do.
  const int units = s.units(0) + s.units(1), pairs = units < s.pairs ? units : s.pairs;
  pairGemmKernel<<<2u * (unsigned)pairs, kThreads, kPairSmemBytes, stream>>>(args);
  return launched(cudaGetLastError());
}

}  // namespace
}  // namespace tnops
