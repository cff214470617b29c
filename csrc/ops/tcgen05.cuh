// tcgen05.cuh - what the tensor-core kernels share: bounded mbarrier waits,
// TMA loads and stores, shared-memory operand descriptors, tcgen05.ld, the
// CTA-pair (cta_group::2) forms, and tensor-map encoding. The contents live in
// an anonymous namespace: each kernel file has its own status word.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace tnops {
namespace {

constexpr int kBK = 64;  // bf16: 128 bytes, one swizzle row
constexpr int kEpiWarps = 8;  // two per TMEM lane quarter
constexpr int kThreads = 64 + kEpiWarps * 32;
constexpr uint32_t kTmemCols = 256;  // one accumulator
constexpr uint32_t kEpiBuf = 4096;   // staging bytes of one epilogue warp
constexpr uint32_t kEpiBytes = kEpiWarps * kEpiBuf;
constexpr uint32_t kHalf = 128 * kBK * 2;  // 16 KiB: 128 rows x 64 K of bf16
constexpr uint64_t kWaitNs = 2000000000ull;  // 2 s per wait

__device__ unsigned int gTcgen05Status;  // first failure code (0: none)

__device__ __forceinline__ uint32_t smemAddr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ uint64_t globalTimer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbarInit(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smemAddr(bar)), "r"(count));
}
__device__ __forceinline__ void mbarExpectTx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smemAddr(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbarTryWait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smemAddr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits until the phase of `parity` completed. Gives up when *abort is set
// (unless ignoreAbort) or after kWaitNs; on a timeout records `code`.
__device__ __forceinline__ bool mbarWait(uint64_t* bar, uint32_t parity, volatile int* abort,
                                         unsigned code, bool ignoreAbort = false) {
  if (mbarTryWait(bar, parity)) return true;
  const uint64_t t0 = globalTimer();
  for (uint32_t it = 1;; ++it) {
    if (mbarTryWait(bar, parity)) return true;
    if ((it & 63) == 0) {
      if (!ignoreAbort && *abort) return false;
      if (globalTimer() - t0 > kWaitNs) {
        atomicCAS(&gTcgen05Status, 0u, code);
        *abort = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void tmaLoad2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smemAddr(bar))
      : "memory");
}
__device__ __forceinline__ void fenceBeforeSync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fenceAfterSync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// K-major operand tile in shared memory, 128-byte swizzle (see the header).
__device__ __forceinline__ uint64_t smemDesc(uint32_t addr) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);  // start address, bits [0,14)
  d |= (uint64_t)1 << 16;                           // leading byte offset 16 B, bits [16,30)
  d |= (uint64_t)(1024 >> 4) << 32;                 // 8-row stride 1024 B, bits [32,46)
  d |= (uint64_t)1 << 46;                           // descriptor version 1, bits [46,48)
  d |= (uint64_t)2 << 61;                           // SWIZZLE_128B, bits [61,64)
  return d;
}
__device__ __forceinline__ void tmemLoad32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
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
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}


// tanh-GELU, 0.5 x (1 + tanh(u)) with u = k0 (x + k1 x^3), evaluated in the
// equivalent form x / (1 + e^(-2u)) (1 + tanh(u) = 2 / (1 + e^(-2u))): no
// cancellation where tanh(u) is near -1, so the relative error stays near
// that of the hardware ex2 and the fast division (~1e-6), far below the bf16
// rounding of the result. Saturates correctly: x for large u, -0 for very
// negative u.
__device__ __forceinline__ float ex2Approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float geluTanh(float x) {
  const float k0 = 0.7978845608028654f;  // sqrt(2 / pi)
  const float k0k1 = 0.7978845608028654f * 0.044715f;
  const float m2log2e = -2.0f * 1.4426950408889634f;
  // |u| <= 40 keeps e^(-2u) finite; gelu is x or -0 to float precision there.
  const float u = fminf(fmaxf(x * fmaf(k0k1, x * x, k0), -40.0f), 40.0f);
  return __fdividef(x, 1.0f + ex2Approx(u * m2log2e));
}
__device__ __forceinline__ uint32_t packBf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ void tmaStore2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void stShared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                           uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// Before a warp's staging buffers go away: its stores have completed.
__device__ __forceinline__ void epilogueDrain(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  __syncwarp();
}

__device__ __forceinline__ void mbarArrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smemAddr(bar)) : "memory");
}

__device__ __forceinline__ uint32_t clusterRank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of the same shared variable in CTA 0 of the cluster.
__device__ __forceinline__ uint32_t inLeader(const void* p) {
  uint32_t d;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(d) : "r"(smemAddr(p)));
  return d;
}
__device__ __forceinline__ void clusterSync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void tmaLoadPair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t leaderBar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(leaderBar)
      : "memory");
}
// Arrives on `bar` in both CTAs of the pair once the pair MMAs issued so far
// have completed.
__device__ __forceinline__ void commitPair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smemAddr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void commitPairLocal(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smemAddr(bar))
               : "memory");
}
__device__ __forceinline__ void mbarArriveRemote(uint32_t clusterAddr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(clusterAddr)
               : "memory");
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encodeTiled() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }


// This file's status word (0: no failure); `reset` clears it. Synchronises
// the device.
inline unsigned readStatus(int reset) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, gTcgen05Status, sizeof(v));
  if (reset) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(gTcgen05Status, &z, sizeof(z));
  }
  return v;
}

}  // namespace
}  // namespace tnops
