// panel_gemm.cuh - products of rows against a wide matrix, both K-major, with
// the caller's epilogue on the fp32 sums:
//
//   D[m, n] = sum_k A[m, k] B[n, k],  handed to Epi in 32 x 32 blocks
//
// for logits (few hundred to a few thousand k, tens of thousands of n) and
// for an MLP's first layer. A persistent CTA-pair pipeline (tcgen05
// cta_group::2) of 256 x 256 tiles with two accumulators in TMEM, so that a
// tile's epilogue runs under the next tile's main loop; the sums here are too
// short to hide one any other way. What bounds such a pipeline is the 64 bytes
// per clock that each SM then loads while its tensor core works, more than L2
// delivers to all SMs at once; so the first K blocks of A (up to kResident of
// them) stay in shared memory while a pair goes along n through its share of a
// 256-row panel, and only B and the rest of A stream through a ring of 16 KiB
// slots. With eight blocks of twelve resident (k = 768) that is 43 bytes per
// clock.
//
// A pair's tiles are consecutive (n fastest), so A is loaded again only where
// its range passes into the next panel.
#pragma once

#include "pair_parts.cuh"

namespace tnops {
namespace {

constexpr int kPanelSlots = 14;   // of kHalf bytes
constexpr int kPanelRing = 6;     // at least this many slots stream
constexpr uint32_t kPanelSmem = kPanelSlots * kHalf + 1024;

template <class Epi>
struct alignas(64) PanelGemmArgs {
  CUtensorMap mapA, mapB;
  int rows, cols, kBlocks;
  int tilesN, tiles, pairs;
  int resident;  // K blocks of A that stay
  Epi epi;
};

// A place in the ring and its barriers' phase, kept up by counting: a division
// by the number of slots for each load would take the MMA warp longer than the
// MMAs of a K block.
struct RingAt {
  uint32_t slot, phase;
  __device__ __forceinline__ void next(uint32_t slots) {
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Epi: `State begin(row)` once per tile and thread (the thread's row of the
// output), `chunk(state, v, ahead, row, col0)` for its 32 columns from col0 of
// each block (ahead: what `ahead(col0)` loaded while the block before was worked
// on), `end(state, row, part)` after the last block (part: the 128 columns'
// number). What an epilogue writes goes straight from registers: operands in
// and out of shared memory take its whole bandwidth here (107 of 128 bytes per
// clock), and a staged copy of the result cost a fifth of the time.
template <class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    panelGemmKernel(const __grid_constant__ PanelGemmArgs<Epi> args) {
  __shared__ __align__(8) uint64_t sFull[kPanelSlots];
  __shared__ __align__(8) uint64_t sEmpty[kPanelSlots];
  __shared__ __align__(8) uint64_t sPanelFull;   // the resident blocks of A are there
  __shared__ __align__(8) uint64_t sPanelEmpty;  // ... and no longer read
  __shared__ __align__(8) uint64_t sAccFull[2];
  __shared__ __align__(8) uint64_t sAccEmpty[2];
  __shared__ __align__(8) uint64_t sDone;
  __shared__ uint32_t sTmem;
  __shared__ int sAbort;
  extern __shared__ uint8_t dsmem[];
  const uint32_t base = (smemAddr(dsmem) + 1023u) & ~1023u;
  const int resident = args.resident;
  const uint32_t slots = (uint32_t)(kPanelSlots - resident);  // of the ring
  const uint32_t ring = base + resident * kHalf;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = clusterRank();
  const int pair = (int)(blockIdx.x >> 1);
  const int first = (int)((int64_t)args.tiles * pair / args.pairs);
  const int end = (int)((int64_t)args.tiles * (pair + 1) / args.pairs);
  const int tilesN = args.tilesN, kBlocks = args.kBlocks;
  volatile int* abort = &sAbort;

  if (threadIdx.x == 0) {
    sAbort = 0;
    for (int s = 0; s < kPanelSlots; ++s) {
      mbarInit(&sFull[s], 1);
      mbarInit(&sEmpty[s], 1);
    }
    mbarInit(&sPanelFull, 1);
    mbarInit(&sPanelEmpty, 1);
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
    RingAt at{0u, 0u};
    uint32_t g = 0, panels = 0;  // loads through the ring, resident panels
    auto stream = [&](const CUtensorMap* map, int row, int kb) {
      if (!mbarWait(&sEmpty[at.slot], at.phase ^ 1u, abort, 1)) return false;
      if (rank == 0) mbarExpectTx(&sFull[at.slot], 2 * kHalf);  // both CTAs' loads
      tmaLoadPair(ring + at.slot * kHalf, map, kb * kBK, row, inLeader(&sFull[at.slot]));
      at.next(slots);
      ++g;
      return true;
    };
    bool ok = true;
    for (int t = first; ok && t < end; ++t) {
      const int m = t / tilesN, m0 = m * 256 + (int)rank * 128;
      const int n0 = (t - m * tilesN) * 256 + (int)rank * 128;
      if (t == first || t == m * tilesN) {
        if (!(ok = mbarWait(&sPanelEmpty, (panels & 1u) ^ 1u, abort, 1))) break;
        if (rank == 0) mbarExpectTx(&sPanelFull, 2 * kHalf * resident);
        for (int kb = 0; kb < resident; ++kb)
          tmaLoadPair(base + kb * kHalf, &args.mapA, kb * kBK, m0, inLeader(&sPanelFull));
        ++panels;
      }
      for (int kb = 0; ok && kb < kBlocks; ++kb) {
        if (kb >= resident) ok = stream(&args.mapA, m0, kb);
        ok = ok && stream(&args.mapB, n0, kb);
      }
    }
    if (*abort) {
      if (rank == 0) {
        for (uint32_t q = g > slots ? g - slots : 0; q < g; ++q)
          mbarWait(&sFull[q % slots], (q / slots) & 1u, abort, 4, true);
        if (panels > 0) mbarWait(&sPanelFull, (panels - 1) & 1u, abort, 4, true);
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
    const uint64_t desc = pairDescBase(0);
    const uint32_t instr = pairInstrDesc(0, 0);
    RingAt at{0u, 0u};
    uint32_t panels = 0, local = 0;
    int tileN = first % tilesN;
    bool ok = true;
    for (int t = first; ok && t < end; ++t, ++local) {
      const uint32_t b = local & 1u, use = local >> 1;
      if (t == first || tileN == 0) {
        if (!(ok = warpWait(&sPanelFull, panels & 1u, abort, 2))) break;
        ++panels;
      }
      if (!(ok = warpWait(&sAccEmpty[b], (use & 1u) ^ 1u, abort, 2))) break;
      fenceAfterSync();
      const uint32_t acc = tmem + b * kTmemCols;
      for (int kb = 0; kb < kBlocks; ++kb) {
        uint32_t a = base + kb * kHalf, sa = 0;
        if (kb >= resident) {
          sa = at.slot;
          if (!(ok = warpWait(&sFull[sa], at.phase, abort, 2))) break;
          a = ring + sa * kHalf;
          at.next(slots);
        }
        const uint32_t sb = at.slot;
        if (!(ok = warpWait(&sFull[sb], at.phase, abort, 2))) break;
        at.next(slots);
        fenceAfterSync();
        const uint32_t bb = ring + sb * kHalf;
        if (elected) {
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            pairMma(acc, pairDesc(desc, a + k * 32), pairDesc(desc, bb + k * 32), instr,
                    kb != 0 || k != 0 ? 1u : 0u);
          if (kb >= resident) commitPair(&sEmpty[sa]);
          commitPair(&sEmpty[sb]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elected) {
        commitPair(&sAccFull[b]);
        if (t + 1 == end || tileN + 1 == tilesN) commitPair(&sPanelEmpty);
      }
      __syncwarp();
      if (++tileN == tilesN) tileN = 0;
    }
    if (elected) commitPairLocal(&sDone);
    __syncwarp();
    if (*abort) mbarWait(&sDone, 0, abort, 5, true);
  } else if (warp >= 2) {
    // Epilogue (both CTAs): this CTA's 128 rows of the tile; TMEM lane
    // quarter warp % 4, column half (warp - 2) / 4.
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint32_t local = 0;
    for (int t = first; t < end; ++t, ++local) {
      const uint32_t b = local & 1u, use = local >> 1;
      const int m = t / tilesN, tileN = t - m * tilesN;
      const int row0 = m * 256 + (int)rank * 128 + quarter * 32;
      typename Epi::State st = args.epi.begin(row0 + lane);
      if (!warpWait(&sAccFull[b], use & 1u, abort, 3)) break;
      fenceAfterSync();
      const uint32_t acc = tmem + b * kTmemCols + ((uint32_t)(quarter * 32) << 16);
      // The next 32 columns are on their way while these are worked on.
      uint32_t r[2][32];
      tmemIssue32(acc + (uint32_t)(half * 128), r[0]);
      auto ahead = args.epi.ahead(tileN * 256 + half * 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = half * 128 + i * 32;
        tmemWait(r[i & 1]);
        const auto now = ahead;
        if (i < 3) {
          ahead = args.epi.ahead(tileN * 256 + c + 32);
          tmemIssue32(acc + (uint32_t)(c + 32), r[(i + 1) & 1]);
        } else {
          // Everything is read: the accumulator goes back before the stores.
          fenceBeforeSync();
          __syncwarp();
          if (lane == 0) arriveInLeader(&sAccEmpty[b]);
        }
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(r[i & 1][k]);
        args.epi.chunk(st, v, now, row0 + lane, tileN * 256 + c);
      }
      args.epi.end(st, row0 + lane, tileN * 2 + half);
    }
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

// 32 columns of a row as 16 pairs of bf16, straight to memory in 32-byte (`wide`:
// the row's address is a multiple of 32), or 16-byte pieces of which the first
// `pieces` 16-byte ones are inside the row.
__device__ __forceinline__ void storeRow32(uint16_t* out, const uint32_t (&w)[16], bool wide,
                                           int pieces) {
  if (wide && pieces >= 4) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + 2 * i),
                   "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]),
                   "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < pieces)
        reinterpret_cast<uint4*>(out)[i] =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// a [rows, k] against b [cols, k], both contiguous, 16-byte aligned, k % 8 == 0.
// Returns 0, or a non-zero code without a launch; args.epi is the caller's.
template <class Epi>
int launchPanelGemm(PanelGemmArgs<Epi>& args, const void* a, const void* b, int rows, int cols,
                    int k, cudaStream_t stream) {
  auto kernel = panelGemmKernel<Epi>;
  // Opt in to the shared memory once per device (bit d of `done`).
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 3;
  const uint64_t bit = 1ull << dev;
  if (!(done.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kPanelSmem) != cudaSuccess)
      return 3;
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  if (!operandMap(&args.mapA, a, rows, k, k, false) ||
      !operandMap(&args.mapB, b, cols, k, k, false))
    return 4;
  args.rows = rows;
  args.cols = cols;
  args.kBlocks = (k + kBK - 1) / kBK;
  args.tilesN = (cols + 255) / 256;
  const int64_t tiles = (int64_t)args.tilesN * ((rows + 255) / 256);
  if (tiles > (1 << 30)) return 1;
  args.tiles = (int)tiles;
  args.pairs = tiles < kSMs / 2 ? (int)tiles : kSMs / 2;
  const int most = kPanelSlots - kPanelRing;
  args.resident = args.kBlocks < most ? args.kBlocks : most;
  kernel<<<2u * (unsigned)args.pairs, kThreads, kPanelSmem, stream>>>(args);
  return launched(cudaGetLastError());
}

}  // namespace
}  // namespace tnops
