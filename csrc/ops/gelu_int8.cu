// gelu_int8.cu - the first linear layer of an MLP and its GELU, with the sums
// before the GELU left in 8 bits for the backward pass instead of in bf16:
//
//   pre = x w^T + bias             fp32, from the tensor cores' accumulators
//   act = bf16(gelu_tanh(pre))     rounded once, as nothing keeps pre in bf16
//   pre_q, pre_e = pre in 8-bit blocks (int8_blocks.cuh)
//
// An epilogue of the CTA-pair pipeline of panel_gemm.cuh. A thread of it holds
// 32 neighbouring sums of one row, which is one 8-bit block: its largest
// magnitude, its exponent and its bytes need nothing from another thread, and
// the sums are rounded once, from fp32. A row's 128 columns of a tile half
// give four exponent bytes, written together where they are aligned. Inference
// takes the epilogue without the 8-bit half (65536 x 1024 -> 4096: 414 us, 472 with it).
#include "int8_blocks.cuh"
#include "panel_gemm.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

// tanh-GELU of two numbers, x / (1 + e^(-2u)) with u = k0 (x + k1 x^3). Where
// the power passes the fp32 range its inverse is 0 and so is the result; at the
// other end the power is 0 and the result x.
__device__ __forceinline__ uint64_t geluTanh2(uint64_t x) {
  const float c = -2.0f * 1.4426950408889634f * 0.7978845608028654f;  // -2 log2e sqrt(2 / pi)
  const uint64_t inner = fma2(pack2(c * 0.044715f, c * 0.044715f), mul2(x, x), pack2(c, c));
  float a, b;
  unpack2(mul2(x, inner), a, b);
  unpack2(add2(pack2(ex2Approx(a), ex2Approx(b)), pack2(1.f, 1.f)),
          a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return mul2(x, pack2(a, b));
}

template <bool KEEP>  // the sums in 8 bits
struct GeluInt8Epi {
  uint16_t* act;
  const uint16_t* bias;
  uint8_t* q;
  uint8_t* e;
  int rows, cols, blocks;

  struct State {
    uint32_t e;
  };
  __device__ __forceinline__ State begin(int) const { return {0u}; }
  // The columns' biases, zeros past the last column (cols % 8 == 0).
  struct Bias {
    uint4 b[4];
  };
  __device__ __forceinline__ Bias ahead(int col0) const {
    Bias r;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      r.b[g] = make_uint4(0u, 0u, 0u, 0u);
      // volatile: the load stays where it is, ahead of its use.
      if (col0 + 8 * g < cols)
        asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.b[g].x), "=r"(r.b[g].y), "=r"(r.b[g].z), "=r"(r.b[g].w)
                     : "l"(bias + col0 + 8 * g));
    }
    return r;
  }
  // One block: its 32 sums as bytes at q + at, its exponent in the state.
  __device__ __forceinline__ void keepSums(State& st, const float (&v)[32], size_t at,
                                           int col0) const {
    // Of the magnitudes' bits: a NaN's are above infinity's. Columns past the
    // last have zero sums (the weight's rows read zero).
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 32; i += 2)
      top = max(top, max(__float_as_uint(v[i]) & 0x7fffffffu,
                         __float_as_uint(v[i + 1]) & 0x7fffffffu));
    const uint32_t ex = int8Exponent(__uint_as_float(top));
    st.e |= ex << (((col0 >> 5) & 3) * 8);
    uint32_t o[8];
    if (int8Plain(ex)) {
      // x 2^(133 - e) + 1.5 2^23: the sum's last byte is the whole number that
      // x / step rounds to, in two's complement.
      const float inv = __uint_as_float((260u - ex) << 23);
      const uint64_t inv2 = pack2(inv, inv), magic = pack2(12582912.f, 12582912.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float r[4];
        unpack2(fma2(pack2(v[4 * i], v[4 * i + 1]), inv2, magic), r[0], r[1]);
        unpack2(fma2(pack2(v[4 * i + 2], v[4 * i + 3]), inv2, magic), r[2], r[3]);
        o[i] = __byte_perm(__byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040),
                           __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040),
                           0x5410);
      }
    } else {
      const Int8Inverse inv = int8Inverse(ex);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i] |= int8Quantize(v[4 * i + j], inv) << (8 * j);
      }
    }
    if (cols % 32 == 0) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(q + at),
                   "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]),
                   "r"(o[7])
                   : "memory");
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (col0 + 8 * g < cols)
          *reinterpret_cast<uint2*>(q + at + 8 * g) = make_uint2(o[2 * g], o[2 * g + 1]);
    }
  }
  __device__ __forceinline__ void chunk(State& st, const float (&in)[32], const Bias& ahead,
                                        int row, int col0) const {
    if (row >= rows || col0 >= cols) return;
    float v[32];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint4 b = ahead.b[g];
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* x = v + 8 * g + 2 * i;
        unpack2(add2(pack2(in[8 * g + 2 * i], in[8 * g + 2 * i + 1]),
                     pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u))),
                x[0], x[1]);
      }
    }
    const size_t at = (size_t)row * cols + col0;
    if constexpr (KEEP) keepSums(st, v, at, col0);
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      unpack2(geluTanh2(pack2(v[2 * i], v[2 * i + 1])), a, b);
      w[i] = packBf16(a, b);
    }
    storeRow32(act + at, w, cols % 16 == 0, (cols - col0) / 8);
  }
  __device__ __forceinline__ void end(const State& st, int row, int part) const {
    const int b0 = part * 4;  // the first of this thread's exponent bytes
    if (!KEEP || row >= rows || b0 >= blocks) return;
    uint8_t* out = e + (size_t)row * blocks + b0;
    if (blocks % 4 == 0) {
      *reinterpret_cast<uint32_t*>(out) = st.e;
    } else {
      for (int i = 0; i < 4 && b0 + i < blocks; ++i) out[i] = (uint8_t)(st.e >> (8 * i));
    }
  }
};

template <bool KEEP>
int linearGelu(const void* x, const void* w, const void* bias, void* act, uint8_t* q,
                      uint8_t* e, int rows, int outs, int ins, cudaStream_t stream) {
  PanelGemmArgs<GeluInt8Epi<KEEP>> args{};
  GeluInt8Epi<KEEP>& epi = args.epi;
  epi.act = static_cast<uint16_t*>(act);
  epi.bias = static_cast<const uint16_t*>(bias);
  epi.q = q;
  epi.e = e;
  epi.rows = rows;
  epi.cols = outs;
  epi.blocks = (outs + kInt8Block - 1) / kInt8Block;
  return launchPanelGemm(args, x, w, rows, outs, ins, stream);
}

}  // namespace

unsigned geluInt8Status(int reset) { return readStatus(reset); }

}  // namespace tnops

using namespace tnops;

extern "C" int tnops_linear_gelu_int8(const void* x, const void* w, const void* bias, void* act,
                                      uint8_t* pre_q, uint8_t* pre_e, int rows, int outs, int ins,
                                      cudaStream_t stream) {
  if (rows <= 0 || outs <= 0 || ins <= 0 || outs % 8 != 0 || ins % 8 != 0 || !aligned16(x) ||
      !aligned16(w) || !aligned16(bias) || bias == nullptr ||
      (reinterpret_cast<uintptr_t>(act) & 31) || (reinterpret_cast<uintptr_t>(pre_q) & 31) ||
      (reinterpret_cast<uintptr_t>(pre_e) & 3) || (pre_q == nullptr) != (pre_e == nullptr))
    return 1;
  auto f = pre_q != nullptr ? linearGelu<true> : linearGelu<false>;
  return f(x, w, bias, act, pre_q, pre_e, rows, outs, ins, stream);
}
