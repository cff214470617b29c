// pair_gemm.cuh - the matrix products behind the training operators: one
// persistent CTA-pair pipeline (tcgen05 cta_group::2, 256 x 256 tiles, fp32
// accumulators in TMEM) whose operands may lie either way round in memory and
// whose epilogue is the caller's.
//
//   D[m, n] = sum_k A(m, k) B(n, k)
//
// An operand is "K-major" when k is contiguous in memory ([m, k] rows) and
// "MN-major" when m (or n) is contiguous ([k, m] rows): with both, the
// products of a backward pass (dX = G W, dW = G^T X) read G, W and X as they
// lie, without a transposed copy. In shared memory, with the 128-byte swizzle:
//   K-major   128 rows of 64 k (128 bytes), 8-row atoms of 1024 bytes; the
//             descriptor's stride is the 1024 bytes from 8 rows to the next 8,
//             and a K = 16 slice starts 32 bytes after the one before it;
//   MN-major  two chunks of 64 m, each 64 rows (one per k) of 128 bytes; the
//             leading offset is the 8192 bytes from one chunk to the next, the
//             stride the 1024 bytes from 8 k to the next 8, and a K = 16
//             slice starts 2048 bytes after the one before it.
// The pipeline is that of the GEMM with the bias epilogue (gemm_tcgen05.cu):
// each CTA of a pair stages 128 rows of A and of B per 64-wide K block in a
// six-stage ring, the even CTA issues the MMAs, two accumulators of 256 TMEM
// columns let the epilogue of a tile run under the next tile's main loop.
// A launch may hold two products (`GemmProblem`), so that dX and dW of a layer
// fill the GPU together; who computes what is pair_schedule.h's. Every wait is
// bounded as there; the first failure is kept in the file's status word.
#pragma once

#include "pair_schedule.h"
#include "tcgen05.cuh"

namespace tnops {
namespace {

constexpr int kPairBM = 256;
constexpr int kPairStages = 6;
constexpr uint32_t kPairSmemBytes = kPairStages * 2 * kHalf + kEpiBytes + 1024;

// One product of a launch. The tensor maps' boxes are {64 k, 128 rows} for a
// K-major operand and {64 m, 64 k} for an MN-major one; out-of-range rows and
// columns read zero, so K, M and N need no padding.
struct alignas(64) GemmProblem {
  CUtensorMap mapA, mapB;
  int tilesM, tilesN, kBlocks;
  int aMn, bMn;
};

template <class Epi>
struct alignas(64) PairGemmArgs {
  GemmProblem prob[2];
  CUtensorMap mapPartial;  // [256 slots, 256] fp32, for an Epi that kCuts
  int problems;
  PairSchedule schedule;
  Epi epi;
};

// Operand descriptor without its start address.
__device__ __forceinline__ uint64_t pairDescBase(int mn) {
  uint64_t d = (uint64_t)(mn ? (8192 >> 4) : 1) << 16;  // leading offset, bits [16,30)
  d |= (uint64_t)(1024 >> 4) << 32;                     // stride, bits [32,46)
  d |= (uint64_t)1 << 46;                               // descriptor version 1
  d |= (uint64_t)2 << 61;                               // SWIZZLE_128B
  return d;
}
__device__ __forceinline__ uint64_t pairDesc(uint64_t base, uint32_t addr) {
  return base | (uint64_t)((addr & 0x3FFFFu) >> 4);
}
// kind::f16 instruction descriptor: bf16 x bf16 -> f32, M = N = 256; bits 15
// and 16 say that A / B is MN-major.
__device__ __forceinline__ uint32_t pairInstrDesc(int aMn, int bMn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)aMn << 15) | ((uint32_t)bMn << 16) |
         ((uint32_t)(256 >> 3) << 17) | ((uint32_t)(kPairBM >> 4) << 24);
}
__device__ __forceinline__ void pairMma(uint32_t tmemD, uint64_t a, uint64_t b, uint32_t instr,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, "
      "{%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(tmemD),
      "l"(a), "l"(b), "r"(instr), "r"(accumulate), "r"(0u)
      : "memory");
}
// One CTA's 128 rows (from mn0) of a 64-wide K block (from k0) of an operand.
__device__ __forceinline__ void loadHalf(uint32_t dst, const CUtensorMap* map, int mn, int mn0,
                                         int k0, uint32_t leaderBar) {
  if (mn) {
    tmaLoadPair(dst, map, mn0, k0, leaderBar);
    tmaLoadPair(dst + kHalf / 2, map, mn0 + 64, k0, leaderBar);
  } else {
    tmaLoadPair(dst, map, k0, mn0, leaderBar);
  }
}

// A warp's 32 x 32 block as bf16 (64-byte rows, 64-byte swizzle) or fp32
// (128-byte rows, 128-byte swizzle) in its staging buffer, then one TMA
// store; the map clips rows and columns past the output's edge, and a block
// that starts past it is the caller's to skip (`inside`).
__device__ __forceinline__ void stageWait(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void stageDone() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void storeBf16(const float (&v)[32], int lane, uint32_t buf,
                                          const CUtensorMap* map, int row0, int col0,
                                          bool inside) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = packBf16(v[2 * i], v[2 * i + 1]);
  stageWait(lane);
  const uint32_t rowOff = (uint32_t)lane * 64u, sw = ((uint32_t)lane >> 1) & 3u;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    stShared16(buf + rowOff + 16u * ((uint32_t)g ^ sw), w[4 * g], w[4 * g + 1], w[4 * g + 2],
               w[4 * g + 3]);
  stageDone();
  if (lane == 0 && inside) {
    tmaStore2d(map, col0, row0, buf);
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
__device__ __forceinline__ void tmaAdd2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], "
      "[%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(y), "r"(src)
      : "memory");
}
__device__ __forceinline__ void storeF32(const float (&v)[32], int lane, uint32_t buf,
                                         const CUtensorMap* map, int row0, int col0, bool inside,
                                         bool add) {
  stageWait(lane);
  const uint32_t rowOff = (uint32_t)lane * 128u, sw = (uint32_t)lane & 7u;
#pragma unroll
  for (int g = 0; g < 8; ++g)
    stShared16(buf + rowOff + 16u * ((uint32_t)g ^ sw), __float_as_uint(v[4 * g]),
               __float_as_uint(v[4 * g + 1]), __float_as_uint(v[4 * g + 2]),
               __float_as_uint(v[4 * g + 3]));
  stageDone();
  if (lane == 0 && inside) {
    if (add)
      tmaAdd2d(map, col0, row0, buf);
    else
      tmaStore2d(map, col0, row0, buf);
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}

// Epi: `State begin(problem, row)` once per tile and thread (the thread's row
// of the output), `chunk(state, v, problem, lane, row0, col0, buf)` for each
// 32 x 32 block of a warp (v: the row's 32 columns from col0; buf: the warp's
// 4 KiB of staging), `end(state, row, part)` after the last block (part: the
// 128 columns' number). With Epi::kCuts, parts of cut tiles go to mapPartial
// instead.
template <class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    pairGemmKernel(const __grid_constant__ PairGemmArgs<Epi> args) {
  __shared__ __align__(8) uint64_t sFull[kPairStages];
  __shared__ __align__(8) uint64_t sEmpty[kPairStages];
  __shared__ __align__(8) uint64_t sAccFull[2];
  __shared__ __align__(8) uint64_t sAccEmpty[2];
  __shared__ __align__(8) uint64_t sDone;
  __shared__ uint32_t sTmem;
  __shared__ int sAbort;
  extern __shared__ uint8_t dsmem[];
  const uint32_t base = (smemAddr(dsmem) + 1023u) & ~1023u;
  const uint32_t stageA0 = base, stageB0 = base + kPairStages * kHalf;
  const uint32_t epi0 = base + kPairStages * 2 * kHalf;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
      const int n0 = (w.tile % p.tilesN) * 256 + (int)rank * 128;
      const int aMn = p.aMn, bMn = p.bMn;
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++g) {
        const uint32_t s = g % kPairStages, round = g / kPairStages;
        if (!mbarWait(&sEmpty[s], (round & 1u) ^ 1u, abort, 1)) break;
        if (rank == 0) mbarExpectTx(&sFull[s], 4 * kHalf);  // both CTAs' A and B halves
        const uint32_t bar = inLeader(&sFull[s]);
        loadHalf(stageA0 + s * kHalf, &p.mapA, aMn, m0, kb * kBK, bar);
        loadHalf(stageB0 + s * kHalf, &p.mapB, bMn, n0, kb * kBK, bar);
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
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // MMA issuer (even CTA only).
    uint32_t g = 0, local = 0;
    PairWalk walk;
    PairWork w;
    walk.init(schedule, pair);
    for (; !*abort && walk.next(schedule, &w); ++local) {
      const GemmProblem& p = args.prob[w.which];
      const uint64_t descA = pairDescBase(p.aMn), descB = pairDescBase(p.bMn);
      const uint32_t stepA = p.aMn ? 2048 : 32, stepB = p.bMn ? 2048 : 32;
      const uint32_t instr = pairInstrDesc(p.aMn, p.bMn);
      const uint32_t b = local & 1u, use = local >> 1;
      if (!mbarWait(&sAccEmpty[b], (use & 1u) ^ 1u, abort, 2)) break;
      fenceAfterSync();
      const uint32_t acc = tmem + b * kTmemCols;
      bool ok = true;
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++g) {
        const uint32_t s = g % kPairStages;
        if (!(ok = mbarWait(&sFull[s], (g / kPairStages) & 1u, abort, 2))) break;
        fenceAfterSync();
        const uint32_t a = stageA0 + s * kHalf, bb = stageB0 + s * kHalf;
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k)
          pairMma(acc, pairDesc(descA, a + k * stepA), pairDesc(descB, bb + k * stepB), instr,
                  kb != w.kb0 || k != 0 ? 1u : 0u);
        commitPair(&sEmpty[s]);
      }
      if (!ok) break;
      commitPair(&sAccFull[b]);
    }
    commitPairLocal(&sDone);
    if (*abort) mbarWait(&sDone, 0, abort, 5, true);
  } else if (warp >= 2) {
    // Epilogue (both CTAs): this CTA's 128 rows of the tile; TMEM lane
    // quarter warp % 4, column half (warp - 2) / 4.
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t buf = epi0 + (uint32_t)(warp - 2) * kEpiBuf;
    uint32_t local = 0;
    PairWalk walk;
    PairWork w;
    walk.init(schedule, pair);
    for (; walk.next(schedule, &w); ++local) {
      const uint32_t b = local & 1u, use = local >> 1;
      const GemmProblem& p = args.prob[w.which];
      const int tileN = w.tile % p.tilesN;
      const int row0 = (w.tile / p.tilesN) * kPairBM + (int)rank * 128 + quarter * 32;
      typename Epi::State st = args.epi.begin(w.which, row0 + lane);
      const bool ready = mbarWait(&sAccFull[b], use & 1u, abort, 3);
      if (!__all_sync(0xffffffffu, ready)) break;
      fenceAfterSync();
      const uint32_t acc = tmem + b * kTmemCols + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = half * 128; c < half * 128 + 128; c += 32) {
        float v[32];
        tmemLoad32(acc + (uint32_t)c, v);
        if (c + 32 == half * 128 + 128) {
          // Last read of this buffer: hand it back before the stores.
          fenceBeforeSync();
          __syncwarp();
          if (lane == 0) mbarArriveRemote(inLeader(&sAccEmpty[b]));
        }
        if (Epi::kCuts && w.slot >= 0)
          storeF32(v, lane, buf, &args.mapPartial,
                   w.slot * kPairBM + (int)rank * 128 + quarter * 32, c, true, false);
        else
          args.epi.chunk(st, v, w.which, lane, row0, tileN * 256 + c, buf);
      }
      args.epi.end(st, row0 + lane, tileN * 2 + half);
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

inline bool encode2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t rows,
                     int64_t cols, int64_t ldBytes, int boxCols, int boxRows,
                     CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion) {
  EncodeTiledFn fn = encodeTiled();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ldBytes};
  const cuuint32_t box[2] = {(cuuint32_t)boxCols, (cuuint32_t)boxRows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [rows, cols] bf16 operand, rows `ld` elements apart: K-major when cols is
// the summed index, MN-major when rows is.
inline bool operandMap(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld,
                       bool mn) {
  return encode2d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, rows, cols, ld * 2, 64,
                  mn ? 64 : 128, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
inline bool bf16OutMap(CUtensorMap* map, const void* base, int64_t rows, int64_t cols,
                       int64_t ld) {
  return encode2d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, rows, cols, ld * 2, 32, 32,
                  CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}
inline bool f32OutMap(CUtensorMap* map, const void* base, int64_t rows, int64_t cols,
                      int64_t ld) {
  return encode2d(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, base, rows, cols, ld * 4, 32, 32,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

// Plans the launch for kSMs / 2 pairs; with `cut`, sums may be split. Product
// 0 must be the one with the longer sum.
template <class Epi>
void planGemm(PairGemmArgs<Epi>* args, bool cut) {
  PairSchedule& s = args->schedule;
  s = {};
  s.pairs = kSMs / 2;
  for (int i = 0; i < 2; ++i) {
    s.k[i] = 1;
    if (i >= args->problems) continue;
    s.tiles[i] = args->prob[i].tilesM * args->prob[i].tilesN;
    s.k[i] = args->prob[i].kBlocks;
  }
  planPairs(&s, cut);
}

// Launches the products of `args`, whose schedule is planned. Returns 0, or a
// non-zero code without a launch.
template <class Epi>
int launchPairGemm(const PairGemmArgs<Epi>& args, cudaStream_t stream) {
  auto kernel = pairGemmKernel<Epi>;
  // Opt in to the shared memory once per device (bit d of `done`).
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 3;
  const uint64_t bit = 1ull << dev;
  if (!(done.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kPairSmemBytes) != cudaSuccess)
      return 3;
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  const PairSchedule& s = args.schedule;
  // In a first round, pairs past the last unit have nothing to do.
  const int units = s.units(0) + s.units(1), pairs = units < s.pairs ? units : s.pairs;
  kernel<<<2u * (unsigned)pairs, kThreads, kPairSmemBytes, stream>>>(args);
  return launched(cudaGetLastError());
}

}  // namespace
}  // namespace tnops
