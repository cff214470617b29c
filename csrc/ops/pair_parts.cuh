// pair_parts.cuh - what the CTA-pair products (pair_gemm.cuh, panel_gemm.cuh)
// share: operand layouts and their descriptors, the MMA of a pair, and how a
// warp stores a block of the result.
//
// An operand is "K-major" when k is contiguous in memory ([m, k] rows) and
// "MN-major" when m (or n) is contiguous ([k, m] rows). In shared memory, with
// the 128-byte swizzle:
//   K-major   128 rows of 64 k (128 bytes), 8-row atoms of 1024 bytes; the
//             descriptor's stride is the 1024 bytes from 8 rows to the next 8,
//             and a K = 16 slice starts 32 bytes after the one before it;
//   MN-major  two chunks of 64 m, each 64 rows (one per k) of 128 bytes; the
//             leading offset is the 8192 bytes from one chunk to the next, the
//             stride the 1024 bytes from 8 k to the next 8, and a K = 16
//             slice starts 2048 bytes after the one before it.
#pragma once

#include "packed_f32.cuh"
#include "tcgen05.cuh"

namespace tnops {
namespace {

// The MMA warps run their loops whole and elect the thread that issues, so
// that the operands of tcgen05.mma are warp-uniform: from a branch of one
// thread an MMA of 128 clocks took 290 to issue.
__device__ __forceinline__ bool electOne() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
// tcgen05.ld of 32 columns in two steps: the load is issued, and its registers
// may be read after tmemWait (which names them, so that no use moves ahead).
__device__ __forceinline__ void tmemIssue32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmemWait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
// Hands an accumulator back to the even CTA. The arrival publishes nothing in
// memory (the TMEM reads are over with tcgen05.wait), so it has CTA scope: with
// a release at cluster scope it waited for the thread's stores to global
// memory.
__device__ __forceinline__ void arriveInLeader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(inLeader(bar)) : "memory");
}

// mbarWait by a whole warp, with one answer for all of it: a warp leaves its
// loop together.
__device__ __forceinline__ bool warpWait(uint64_t* bar, uint32_t parity, volatile int* abort,
                                         unsigned code) {
  return __all_sync(0xffffffffu, mbarWait(bar, parity, abort, code));
}

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
         ((uint32_t)(256 >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}
__device__ __forceinline__ void pairMma(uint32_t tmemD, uint64_t a, uint64_t b, uint32_t instr,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmemD),
      "l"(a), "l"(b), "r"(instr), "r"(accumulate)
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
// w: the row's 32 columns as 16 pairs of bf16.
__device__ __forceinline__ void storePacked(const uint32_t (&w)[16], int lane, uint32_t buf,
                                            const CUtensorMap* map, int row0, int col0,
                                            bool inside) {
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
__device__ __forceinline__ void storeBf16(const float (&v)[32], int lane, uint32_t buf,
                                          const CUtensorMap* map, int row0, int col0,
                                          bool inside) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = packBf16(v[2 * i], v[2 * i + 1]);
  storePacked(w, lane, buf, map, row0, col0, inside);
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


}  // namespace
}  // namespace tnops
