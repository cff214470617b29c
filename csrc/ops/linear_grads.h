// linear_grads.h - the two products of a linear layer's backward pass, for the
// C++ side of the library (the C launcher is tnops_linear_grads).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime_api.h>

namespace tnops {

// How an output is written.
enum GradStore { kStoreNone = 0, kStoreBf16 = 1, kStoreF32 = 2, kAddF32 = 3 };

// y = x w^T with y [rows, outs], x [rows, ins], w [outs, ins]; g [rows, outs]
// (rows `ldg` elements apart) is the gradient of y. dx [rows, ins] = g w,
// dw [outs, ins] = g^T x, each left out with kStoreNone. dw may have `padded`
// more rows, which get zeros. Both are multiplied by *scale[0] and *scale[1]
// where those are given.
struct LinearGrads {
  const void* g;
  int64_t ldg;
  const void* w;
  const void* x;
  void* dx;
  void* dw;
  void* scratch;  // 16-byte aligned, at least tnops_linear_grads_scratch()
  size_t scratchBytes;
  GradStore dxStore, dwStore;
  int rows, outs, ins, padded;
  const float* scale[2];
};

int linearGrads(const LinearGrads& a, cudaStream_t stream);
// Roughly how long both products take, in K blocks of a tile.
int linearGradsCost(int rows, int outs, int ins);
size_t linearGradsScratch(int rows, int outs, int padded, int ins, bool wantDx, bool wantDw);

// First failure code of the tensor-core kernels of linear_grads.cu,
// linear_ce.cu and gelu_int8.cu.
unsigned linearGradsStatus(int reset);
unsigned linearCeStatus(int reset);
unsigned geluInt8Status(int reset);

}  // namespace tnops
