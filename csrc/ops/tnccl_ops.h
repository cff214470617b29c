// tnccl_ops.h - C launchers of the fused model kernels (libtnccl_ops.so).
//
// All launchers are asynchronous on `stream` and return a cudaError_t cast to
// int (0 = success). Shapes are row-major [rows, cols]; bf16 tensors are
// passed as raw 16-bit storage.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

// x_out = x + delta (delta optional, bf16); y = LayerNorm(x_out) * w + b in
// bf16; mean/rstd saved in fp32. x, x_out fp32 [rows, C]; w, b fp32 [C].
// C % 4 == 0 and C <= 2048; x, x_out, w, b 16-byte aligned, delta and y
// 8-byte aligned; anything else returns 1 (invalid argument), no launch.
int tnops_ln_fwd(const float* x, const uint16_t* delta, const float* w, const float* b,
                 float* x_out, uint16_t* y, float* mean, float* rstd, int rows, int C, float eps,
                 cudaStream_t stream);

// Backward of tnops_ln_fwd. gy bf16 [rows, C]; g_res fp32 [rows, C] (gradient
// arriving through the residual stream; may be null = zeros); x_out, mean,
// rstd from the forward. Writes dx fp32 = g_res + dLN/dx, optionally dx_bf16
// (the same value for the bf16 `delta` input), and dw/db fp32 [C] (overwritten,
// deterministic two-stage reduction through `partial`, which must hold
// 2 * tnops_ln_partial_rows() * C floats). C % 4 == 0 and C <= 1024; g_res,
// x_out, w and dx 16-byte aligned, gy and dx_bf16 8-byte aligned; anything
// else returns 1 (invalid argument) without a launch.
int tnops_ln_bwd(const uint16_t* gy, const float* g_res, const float* x_out, const float* w,
                 const float* mean, const float* rstd, float* dx, uint16_t* dx_bf16, float* dw,
                 float* db, float* partial, int rows, int C, cudaStream_t stream);
int tnops_ln_partial_rows(void);

// Fused softmax cross-entropy over bf16 logits [rows, ld] whose first V
// columns are classes (the rest is padding): loss[r] = logsumexp(logits[r,:V])
// - logits[r, target[r]] (fp32), and logits is overwritten in place with
// d(mean loss)/d(logits) = (softmax - onehot)/valid in bf16 (0 in padding
// columns). Rows whose target is negative are ignored (zero loss and
// gradient); `valid` counts the rows that are not, for the mean.
int tnops_cross_entropy_fwd_bwd(uint16_t* logits, const int64_t* target, float* loss, int rows,
                                int V, int ld, int valid, cudaStream_t stream);

// Bias gradient of a linear layer: db[n] = sum_m g[m, n] (g bf16 [M, N],
// db fp32 [N], N a multiple of 8), deterministic two-pass column sum through
// `partial` (tnops_colsum_parts(M, N) * N floats). The bf16 matrices of this
// and the next function must be 16-byte aligned; otherwise, or with N % 8
// != 0, they return 1 without a launch.
int tnops_bias_grad(const uint16_t* g, float* db, float* partial, int M, int N,
                    cudaStream_t stream);
// Fused tanh-GELU backward and bias gradient of the linear layer feeding the
// GELU: gpre = bf16(gy * gelu'(pre)), db[n] = sum_m gpre[m, n].
int tnops_gelu_bwd_bias(const uint16_t* gy, const uint16_t* pre, uint16_t* gpre, float* db,
                        float* partial, int M, int N, cudaStream_t stream);
int tnops_colsum_parts(int M, int N);
// tnops_bias_grad with db in bf16 (rounded from the fp32 sum).
int tnops_bias_grad_bf16(const uint16_t* g, uint16_t* db, float* partial, int M, int N,
                         cudaStream_t stream);
// tnops_gelu_bwd_bias with pre in 8-bit blocks (tnops_quantize_int8's form):
// pre_q [M, N] 8-byte aligned, pre_e [M, ceil(N / 32)]; db (the sum of the
// products before their rounding to bf16) fp32 with db_f32, else bf16, or null
// (partial may then be null too).
int tnops_gelu_bwd_bias_int8(const uint16_t* gy, const uint8_t* pre_q, const uint8_t* pre_e,
                             uint16_t* gpre, void* db, int db_f32, float* partial, int M, int N,
                             cudaStream_t stream);

// Multiplies a bf16 tensor by the fp32 scalar *scale (device memory); no-op
// on the device when *scale == 1.
int tnops_scale_bf16(uint16_t* x, size_t n, const float* scale, cudaStream_t stream);

// Multi-tensor AdamW step (decoupled weight decay) over up to 64 tensors per
// call: p -= lr * (m_hat / (sqrt(v_hat) + eps) + wd * p). grads may be scaled
// by grad_scale first. bias corrections are computed from `step` (>= 1).
typedef struct {
  int n;
  float* param[64];
  const float* grad[64];
  float* exp_avg[64];
  float* exp_avg_sq[64];
  int64_t numel[64];
  float weight_decay[64];
  // Optional (null entries skip it): a bf16 copy of each updated parameter,
  // written in the same pass, for the next forward's bf16 GEMMs.
  uint16_t* param_bf16[64];
} tnops_adamw_list;

int tnops_adamw(const tnops_adamw_list* list, float lr, float beta1, float beta2, float eps,
                int64_t step, float grad_scale, cudaStream_t stream);
// The same update with the step read from device memory (*step >= 1) when
// the kernel runs: a launch captured in a CUDA graph then takes the step of
// each replay (the caller advances the counter on the same stream).
int tnops_adamw_dev(const tnops_adamw_list* list, float lr, float beta1, float beta2, float eps,
                    const int64_t* step, float grad_scale, cudaStream_t stream);

// bf16 GEMM on the tcgen05 tensor cores with a fused epilogue:
// pre = bf16(x w^T + bias), and with `gelu` act = bf16(gelu_tanh(pre)).
// x [M, K], w [N, K] (nn.Linear layout), bias [N] (may be null), pre / act
// [M, N] (pre may be null with gelu). `persistent`: 0 one CTA per 128 x 256
// tile, 1 one CTA per SM walking the tiles with two TMEM accumulators, 2 CTA
// pairs (cta_group::2) walking 256 x 256 tiles. K % 8 == 0,
// N % 8 == 0, x, w, pre, act 16-byte aligned; 1 (invalid argument) otherwise.
int tnops_gemm_bias_act(const void* x, const void* w, const void* bias, void* pre, void* act,
                        int M, int N, int K, int gelu, int persistent, cudaStream_t stream);
// Both products of the backward pass of y = x w^T: dx [rows, ins] (bf16) =
// g w and dw [outs, ins] (fp32 with dw_f32, else bf16) = g^T x, for g
// [rows, outs] with rows ldg elements apart, w [outs, ins], x [rows, ins],
// all bf16. A null dx or dw is left out. ins % 8 == 0, ldg % 8 == 0, 16-byte
// aligned pointers; 1 (invalid argument) without a launch otherwise. scratch
// (scratch_bytes, at least tnops_linear_grads_scratch(...), which may be 0):
// partial sums of tiles that several SM pairs share.
size_t tnops_linear_grads_scratch(int rows, int outs, int ins, int want_dx, int want_dw);
int tnops_linear_grads(const void* g, int64_t ldg, const void* w, const void* x, void* dx,
                       void* dw, int dw_f32, int rows, int outs, int ins, void* scratch,
                       size_t scratch_bytes, cudaStream_t stream);

// Softmax cross-entropy of l = x w^T without the logits in memory: x
// [rows, width], w [vocab, width] in bf16, of which the first `classes` rows
// are classes. A row whose target is outside [0, classes) does not count
// (zero loss, zero gradient). width % 8 == 0, x, w, dx, dw 16-byte, d 32-byte
// aligned; 1 (invalid argument) without a launch otherwise.
//  * fwd: loss[r] and lse[r] (fp32); partial holds
//    2 * rows * tnops_linear_ce_parts(classes) floats of scratch.
//  * mean: *out = the losses' sum, or with `mean` their mean over the rows that
//    count; *share = 1 / max(1, rows that count).
//  * bwd: dx [rows, width] (bf16) and dw [vocab, width] (fp32 with dw_f32, else
//    bf16; rows from `classes` on are zero) of sum_r k[r] loss[r], with k[r] =
//    grad[r * grad_step] (* *share), grad_step 0 or 1. Works on `piece` classes
//    at a time (piece % 32 == 0); d holds rows * piece bf16 of scratch, dx_f32
//    rows * width floats when piece < classes, and scratch scratch_bytes, at
//    least tnops_linear_ce_scratch(...). A null dx or dw is left out.
//  * piece: a good `piece` whose d takes at most `budget` bytes (256 classes
//    at least).
int tnops_linear_ce_parts(int classes);
int tnops_linear_ce_piece(int rows, int width, int classes, int64_t budget);
size_t tnops_linear_ce_scratch(int rows, int width, int classes, int vocab, int piece,
                               int want_dx, int want_dw);
int tnops_linear_ce_fwd(const void* x, const void* w, const int64_t* target, float* loss,
                        float* lse, float* partial, int rows, int width, int classes,
                        cudaStream_t stream);
int tnops_linear_ce_mean(const float* loss, const int64_t* target, float* out, float* share,
                         int rows, int classes, int mean, cudaStream_t stream);
int tnops_linear_ce_bwd(const void* x, const void* w, const int64_t* target, const float* lse,
                        const float* grad, int grad_step, const float* share, void* d, int piece,
                        float* dx_f32, void* scratch, size_t scratch_bytes, void* dx, void* dw,
                        int dw_f32, int rows, int width, int classes, int vocab,
                        cudaStream_t stream);

// Token and position embedding: y[r] = scale * w[token[r]] + p[position[r]]
// for w [vocab, cols] and p [context, cols] (both fp32 with w_f32, else bf16;
// p may be null), y [rows, cols] (fp32 with y_f32, else bf16). A null
// `position` stands for r % seq. An index outside its table adds nothing.
// token_order and position_order (or null): for the gradient of w and, where
// positions are given, of p; tnops_embedding_order_bytes(rows, vocab or
// context) bytes each, 16-byte aligned.
size_t tnops_embedding_order_bytes(int64_t rows, int size);
int tnops_embedding_fwd(const int64_t* token, const int64_t* position, const void* w,
                        const void* p, int w_f32, void* y, int y_f32, int64_t rows, int seq,
                        int vocab, int context, int cols, float scale, void* token_order,
                        void* position_order, cudaStream_t stream);
// Gradients of the tables for g [rows, cols] (fp32 with g_f32, else bf16), dw
// and dp of one type (fp32 with d_f32, else bf16); a null dw or dp is left
// out. dw[v] = scale * the sum of g[r] over the rows with token[r] = v, for
// every v (rows without a token: zero); dp alike over positions, without the
// scale (a null position_order stands for r % seq; rows must then be a multiple
// of seq). The orders are the forward pass's, of the same rows and table sizes;
// they are only read. Bit-identical from run to run. scratch: 16-byte aligned,
// tnops_embedding_grad_scratch(rows, cols, 1 or 2 tables) bytes. Returns 1
// (invalid argument) without a launch for anything else.
size_t tnops_embedding_grad_scratch(int64_t rows, int cols, int tables);
int tnops_embedding_grad(const void* g, int g_f32, const void* token_order, void* dw, int vocab,
                         float scale, const void* position_order, int seq, void* dp, int context,
                         int d_f32, int64_t rows, int cols, void* scratch, cudaStream_t stream);

// x [rows, cols] (fp32 with x_f32, else bf16) in 8-bit blocks: q [rows, cols]
// signed bytes and one exponent byte per 32 neighbours of a row, e
// [rows, ceil(cols / 32)]; value = q * 2^(e - 133), 255 marks a block that
// holds an infinity or a NaN (it reads back as NaN).
int tnops_quantize_int8(const void* x, int x_f32, uint8_t* q, uint8_t* e, int64_t rows, int cols,
                        cudaStream_t stream);
int tnops_dequantize_int8(const uint8_t* q, const uint8_t* e, void* x, int x_f32, int64_t rows,
                          int cols, cudaStream_t stream);

// act [rows, outs] (bf16) = gelu_tanh(x w^T + bias) for x [rows, ins],
// w [outs, ins], bias [outs] in bf16, and the sums before the GELU in 8-bit
// blocks (rounded from fp32), left out where pre_q and pre_e are null. ins,
// outs % 8 == 0, x, w, bias 16-byte, act and pre_q 32-byte, pre_e 4-byte
// aligned; 1 (invalid argument) otherwise.
int tnops_linear_gelu_int8(const void* x, const void* w, const void* bias, void* act,
                           uint8_t* pre_q, uint8_t* pre_e, int rows, int outs, int ins,
                           cudaStream_t stream);

// First failure code recorded by a tcgen05 kernel (a bounded wait that expired),
// 0 if none; `reset` clears it. Synchronises the device.
unsigned tnops_tcgen05_status(int reset);

// Number of kernels the ops library launched in this process.
unsigned long long tnops_launch_count(void);

#ifdef __cplusplus
}
#endif
