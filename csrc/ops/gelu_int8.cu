// gelu_int8.cu - the first linear layer of an MLP and its GELU, with the sums
// before the GELU left in 8 bits for the backward pass instead of in bf16:
//
//   pre = x w^T + bias             fp32, from the tensor cores' accumulators
//   act = bf16(gelu_tanh(bf16(pre)))      as tnops_gemm_bias_act gives it
//   pre_q, pre_e = pre in 8-bit blocks (int8_blocks.cuh)
//
// An epilogue of the CTA-pair pipeline of panel_gemm.cuh. A thread of it holds
// 32 neighbouring sums of one row, which is one 8-bit block: its largest
// magnitude, its exponent and its bytes need nothing from another thread, and
// the sums are rounded once, from fp32. A row's 128 columns of a tile half
// give four exponent bytes, written together where they are aligned.
#include "int8_blocks.cuh"
#include "panel_gemm.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

struct GeluInt8Epi {
  static constexpr bool kStages = true;
  CUtensorMap mapAct;
  const uint16_t* bias;
  uint8_t* q;
  uint8_t* e;
  int rows, cols, blocks;

  struct State {
    uint32_t e;
  };
  __device__ __forceinline__ State begin(int) const { return {0u}; }
  __device__ __forceinline__ void chunk(State& st, const float (&in)[32], int lane, int row0,
                                        int col0, uint32_t buf) const {
    float v[32];
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint4 b = make_uint4(0u, 0u, 0u, 0u);
      const bool in8 = col0 + 8 * g < cols;  // cols % 8 == 0
      if (in8) b = __ldg(reinterpret_cast<const uint4*>(bias + col0) + g);
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float add = __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        const float s = in8 ? in[8 * g + i] + add : 0.f;
        v[8 * g + i] = s;
        // fmaxf drops a NaN: carried as infinity.
        top = fmaxf(top, __uint_as_float(min(__float_as_uint(s) & 0x7fffffffu, 0x7f800000u)));
      }
    }
    const uint32_t ex = int8Exponent(top);
    const Int8Inverse inv = int8Inverse(ex);
    st.e |= ex << (((col0 >> 5) & 3) * 8);
    const int row = row0 + lane;
    if (row < rows) {
      uint8_t* out = q + (size_t)row * cols + col0;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (col0 + 8 * g >= cols) break;
        uint32_t o[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          o[i >> 2] |= int8Quantize(v[8 * g + i], inv) << ((i & 3) * 8);
        *reinterpret_cast<uint2*>(out + 8 * g) = make_uint2(o[0], o[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = geluTanh(bf2f(f2bf(v[i])));
    storeBf16(v, lane, buf, &mapAct, row0, col0, row0 < rows && col0 < cols);
  }
  __device__ __forceinline__ void end(const State& st, int row, int part) const {
    const int b0 = part * 4;  // the first of this thread's exponent bytes
    if (row >= rows || b0 >= blocks) return;
    uint8_t* out = e + (size_t)row * blocks + b0;
    if (blocks % 4 == 0) {
      *reinterpret_cast<uint32_t*>(out) = st.e;
    } else {
      for (int i = 0; i < 4 && b0 + i < blocks; ++i) out[i] = (uint8_t)(st.e >> (8 * i));
    }
  }
};

}  // namespace

unsigned geluInt8Status(int reset) { return readStatus(reset); }

}  // namespace tnops

using namespace tnops;

extern "C" int tnops_linear_gelu_int8(const void* x, const void* w, const void* bias, void* act,
                                      uint8_t* pre_q, uint8_t* pre_e, int rows, int outs, int ins,
                                      cudaStream_t stream) {
  if (rows <= 0 || outs <= 0 || ins <= 0 || outs % 8 != 0 || ins % 8 != 0 || !aligned16(x) ||
      !aligned16(w) || !aligned16(bias) || !aligned16(act) || bias == nullptr ||
      (reinterpret_cast<uintptr_t>(pre_q) & 7) || (reinterpret_cast<uintptr_t>(pre_e) & 3))
    return 1;
  PanelGemmArgs<GeluInt8Epi> args{};
  GeluInt8Epi& epi = args.epi;
  if (!bf16OutMap(&epi.mapAct, act, rows, outs, outs)) return 4;
  epi.bias = static_cast<const uint16_t*>(bias);
  epi.q = pre_q;
  epi.e = pre_e;
  epi.rows = rows;
  epi.cols = outs;
  epi.blocks = (outs + kInt8Block - 1) / kInt8Block;
  return launchPanelGemm(args, x, w, rows, outs, ins, stream);
}
