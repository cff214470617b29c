// train_ext.cpp - PyTorch binding of the training operators: embedding,
// linear cross-entropy, and linear layers with 8-bit activations (csrc/ops).
// As in ops_ext.cpp, each entry validates its tensors and calls the C launcher
// on the current CUDA stream; a launcher error raises.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <climits>
#include <string>
#include <vector>

#include "tnccl_ops.h"

namespace py = pybind11;

namespace {

using Opt = c10::optional<at::Tensor>;

cudaStream_t streamOf(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

void need(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
void need(const at::Tensor& t, at::ScalarType st, const char* name) {
  need(t, name);
  TORCH_CHECK(t.scalar_type() == st, name, " has dtype ", t.scalar_type(), ", expected ", st);
}
// 1 for fp32, 0 for bf16.
int f32(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name,
              " must be float32 or bfloat16, not ", t.scalar_type());
  return t.scalar_type() == at::kFloat;
}
void sameDevice(const at::Tensor& a, const at::Tensor& b, const char* name) {
  TORCH_CHECK(a.device() == b.device(), name, " is on ", b.device(), ", expected ", a.device());
}
int asInt(int64_t n, const char* what) {
  TORCH_CHECK(n >= 0 && n <= INT_MAX, what, " (", n, ") is out of range");
  return (int)n;
}

void ok(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, ")"); }

at::Tensor scratchOf(size_t n, const at::Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* orNull(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

uint8_t* bytes(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

// -- embedding -----------------------------------------------------------------

// orderW and orderP (or null) receive what the gradients of w and p need to
// know of token and position.
at::Tensor embeddingFwd(const at::Tensor& token, const Opt& position, const at::Tensor& w,
                        const Opt& p, int64_t seq, double scale, bool outF32,
                        at::Tensor* orderW = nullptr, at::Tensor* orderP = nullptr) {
  need(token, at::kLong, "idx");
  need(w, "weight");
  TORCH_CHECK(w.dim() == 2, "weight must be [vocab, width]");
  const int wF32 = f32(w, "weight");
  sameDevice(token, w, "weight");
  if (p) {
    need(*p, w.scalar_type(), "pos_weight");
    TORCH_CHECK(p->dim() == 2 && p->size(1) == w.size(1), "pos_weight must be [context, width]");
    sameDevice(token, *p, "pos_weight");
  }
  if (position) {
    need(*position, at::kLong, "positions");
    TORCH_CHECK(position->numel() == token.numel(), "positions must have one entry per token");
    sameDevice(token, *position, "positions");
  }
  c10::cuda::CUDAGuard g(token.device());
  const int64_t rows = token.numel();
  auto y = at::empty({rows, w.size(1)}, w.options().dtype(outF32 ? at::kFloat : at::kBFloat16));
  if (y.numel() == 0) return y;
  auto order = [&](at::Tensor* out, const at::Tensor& table) -> void* {
    if (out == nullptr) return nullptr;
    *out = scratchOf(tnops_embedding_order_bytes(rows, asInt(table.size(0), "table size")), w);
    TORCH_CHECK(out->defined(), "embedding: too many rows, or a table without rows");
    return out->data_ptr();
  };
  void* tokenOrder = order(orderW, w);
  void* positionOrder = p && position ? order(orderP, *p) : nullptr;
  ok(tnops_embedding_fwd(token.data_ptr<int64_t>(),
                         position ? position->data_ptr<int64_t>() : nullptr, w.data_ptr(),
                         p ? p->data_ptr() : nullptr, wF32, y.data_ptr(), outF32 ? 1 : 0, rows,
                         asInt(seq, "sequence length"), asInt(w.size(0), "vocabulary"),
                         p ? asInt(p->size(0), "context") : 0, asInt(w.size(1), "width"),
                         (float)scale, tokenOrder, positionOrder, streamOf(token)),
     "tnops_embedding_fwd");
  return y;
}

// grad [rows, width]; the forward pass's orders of token and position
// (undefined for row % seq) -> the gradients of the [vocab, width] and
// [context, width] tables; one with no rows (vocab or context 0) is left out.
std::vector<at::Tensor> embeddingGrad(const at::Tensor& grad, const at::Tensor& tokenOrder,
                                      const at::Tensor& positionOrder, int64_t seq,
                                      int64_t vocab, int64_t context, double scale, bool outF32,
                                      const Opt& dwOut, const Opt& dpOut) {
  need(grad, "grad");
  TORCH_CHECK(grad.dim() == 2, "embedding_grad: want grad [rows, width]");
  const int gF32 = f32(grad, "grad");
  const int64_t rows = grad.size(0), width = grad.size(1);
  TORCH_CHECK(seq > 0 ? rows % seq == 0 : rows == 0,
              "embedding_grad: rows must be whole sequences");
  c10::cuda::CUDAGuard g(grad.device());
  const auto opt = grad.options().dtype(outF32 ? at::kFloat : at::kBFloat16);
  auto table = [&](int64_t n, const Opt& out) {
    if (n == 0) return at::Tensor();
    auto d = out ? *out : at::empty({n, width}, opt);
    need(d, outF32 ? at::kFloat : at::kBFloat16, "out");
    TORCH_CHECK(d.numel() == n * width, "embedding_grad: out has the wrong size");
    sameDevice(grad, d, "out");
    if (rows == 0) d.zero_();
    return d;
  };
  auto dw = table(vocab, dwOut), dp = table(context, dpOut);
  if (rows == 0 || width == 0 || (vocab == 0 && context == 0)) return {dw, dp};
  const int cols = asInt(width, "width");
  auto scratch = at::empty(
      {(int64_t)tnops_embedding_grad_scratch(rows, cols, (vocab > 0) + (context > 0))},
      grad.options().dtype(at::kByte));
  ok(tnops_embedding_grad(grad.data_ptr(), gF32, orNull(tokenOrder), orNull(dw),
                          asInt(vocab, "vocabulary"), (float)scale, orNull(positionOrder),
                          asInt(seq, "sequence length"), orNull(dp), asInt(context, "context"),
                          outF32 ? 1 : 0, rows, cols, scratch.data_ptr(), streamOf(grad)),
     "tnops_embedding_grad");
  return {dw, dp};
}

// -- linear cross-entropy --------------------------------------------------------

struct CeShape {
  int rows, width, classes, vocab;
};
CeShape ceShape(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target,
                int64_t classes) {
  need(x, at::kBFloat16, "x");
  need(w, at::kBFloat16, "weight");
  need(target, at::kLong, "target");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1),
              "linear_cross_entropy: want x [rows, width] and weight [vocab, width]");
  TORCH_CHECK(x.size(1) > 0 && x.size(1) % 8 == 0,
              "linear_cross_entropy: width must be a multiple of 8");
  TORCH_CHECK(target.numel() == x.size(0), "linear_cross_entropy: one target per row");
  TORCH_CHECK(classes > 0 && classes <= w.size(0),
              "linear_cross_entropy: classes must be in [1, ", w.size(0), "]");
  sameDevice(x, w, "weight");
  sameDevice(x, target, "target");
  return {asInt(x.size(0), "rows"), asInt(x.size(1), "width"), asInt(classes, "classes"),
          asInt(w.size(0), "vocabulary")};
}

// -> per-row loss, lse, and (but for kNone) the sum or mean, 1 / rows that count.
// The last two are tensors of their own: the loss may be changed in place.
enum Reduction { kMean = 0, kSum = 1, kNone = 2 };
std::vector<at::Tensor> linearCeFwd(const at::Tensor& x, const at::Tensor& w,
                                    const at::Tensor& target, int64_t classes,
                                    int64_t reduction) {
  const CeShape s = ceShape(x, w, target, classes);
  c10::cuda::CUDAGuard g(x.device());
  const auto opt = x.options().dtype(at::kFloat);
  auto loss = at::empty({s.rows}, opt), lse = at::empty({s.rows}, opt);
  if (s.rows == 0) {
    return {loss, lse, at::zeros({}, opt), at::ones({}, opt)};
  }
  auto partial = at::empty({(int64_t)tnops_linear_ce_parts(s.classes), s.rows, 2}, opt);
  ok(tnops_linear_ce_fwd(x.data_ptr(), w.data_ptr(), target.data_ptr<int64_t>(),
                         loss.data_ptr<float>(), lse.data_ptr<float>(), partial.data_ptr<float>(),
                         s.rows, s.width, s.classes, streamOf(x)),
     "tnops_linear_ce_fwd");
  if (reduction == kNone) return {loss, lse, at::Tensor(), at::Tensor()};
  auto out = at::empty({}, opt), share = at::empty({}, opt);
  ok(tnops_linear_ce_mean(loss.data_ptr<float>(), target.data_ptr<int64_t>(),
                          out.data_ptr<float>(), share.data_ptr<float>(), s.rows, s.classes,
                          reduction == kMean ? 1 : 0, streamOf(x)),
     "tnops_linear_ce_mean");
  return {loss, lse, out, share};
}

// Scratch for a piece of the logits' gradient.
constexpr int64_t kCeBudget = 512ll << 20;

std::vector<at::Tensor> linearCeBwd(const at::Tensor& x, const at::Tensor& w,
                                    const at::Tensor& target, const at::Tensor& lse,
                                    const at::Tensor& grad, const Opt& share, int64_t classes,
                                    bool wantDx, bool wantDw, bool dwF32, const Opt& dwOut,
                                    int64_t budget) {
  const CeShape s = ceShape(x, w, target, classes);
  need(lse, at::kFloat, "lse");
  need(grad, at::kFloat, "grad");
  TORCH_CHECK(lse.numel() == s.rows, "linear_cross_entropy: want one lse per row");
  TORCH_CHECK(grad.numel() == 1 || grad.numel() == s.rows,
              "linear_cross_entropy: want one gradient, or one per row");
  sameDevice(x, lse, "lse");
  sameDevice(x, grad, "grad");
  TORCH_CHECK(budget > 0, "linear_cross_entropy: the scratch budget must be positive");
  if (share) {
    need(*share, at::kFloat, "share");
    TORCH_CHECK(share->numel() == 1, "linear_cross_entropy: want one share");
    sameDevice(x, *share, "share");
  }
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor dx, dw;
  if (wantDx) dx = at::empty_like(x);
  if (wantDw) {
    const auto st = dwF32 ? at::kFloat : at::kBFloat16;
    dw = dwOut ? *dwOut : at::empty({s.vocab, s.width}, w.options().dtype(st));
    need(dw, st, "dw_out");
    TORCH_CHECK(dw.numel() == w.numel(), "linear_cross_entropy: dw_out must match weight");
    sameDevice(x, dw, "dw_out");
    if (s.rows == 0) dw.zero_();
  }
  if (s.rows == 0 || (!wantDx && !wantDw)) return {dx, dw};
  const int64_t piece = tnops_linear_ce_piece(s.rows, s.width, s.classes, budget);
  auto d = at::empty({(int64_t)s.rows, piece}, x.options());
  const size_t scratchBytes =
      tnops_linear_ce_scratch(s.rows, s.width, s.classes, s.vocab, (int)piece, wantDx, wantDw);
  auto scratch = scratchOf(scratchBytes, x);
  at::Tensor dxF32;
  if (wantDx && piece < s.classes) dxF32 = at::empty(x.sizes(), x.options().dtype(at::kFloat));
  ok(tnops_linear_ce_bwd(x.data_ptr(), w.data_ptr(), target.data_ptr<int64_t>(),
                         lse.data_ptr<float>(), grad.data_ptr<float>(),
                         grad.numel() == 1 ? 0 : 1, share ? share->data_ptr<float>() : nullptr,
                         d.data_ptr(), (int)piece,
                         static_cast<float*>(orNull(dxF32)),
                         orNull(scratch), scratchBytes, orNull(dx), orNull(dw),
                         dwF32 ? 1 : 0, s.rows, s.width, s.classes, s.vocab, streamOf(x)),
     "tnops_linear_ce_bwd");
  return {dx, dw};
}

// -- linear layers with 8-bit activations ------------------------------------------

// Scratch of the column sums of an [M, N] matrix; none where one block of rows
// is all.
struct ColumnParts {
  at::Tensor t;
  operator float*() const { return t.defined() ? t.data_ptr<float>() : nullptr; }
};
ColumnParts columnParts(const at::Tensor& like, int M, int N) {
  const int64_t parts = tnops_colsum_parts(M, N);
  return {parts > 1 ? at::empty({parts * N}, like.options().dtype(at::kFloat)) : at::Tensor()};
}

void needSums(const at::Tensor& grad, const at::Tensor& db, at::ScalarType st, int N) {
  need(db, st, "db_out");
  TORCH_CHECK(db.numel() == N, "db_out must have one value per column");
  sameDevice(grad, db, "db_out");
}

// x [rows, cols] -> (q int8 [rows, cols], e uint8 [rows, ceil(cols / 32)])
std::vector<at::Tensor> quantizeInt8(const at::Tensor& x) {
  need(x, "x");
  TORCH_CHECK(x.dim() == 2, "quantize_int8: want [rows, cols]");
  const int xF32 = f32(x, "x");
  c10::cuda::CUDAGuard g(x.device());
  const int64_t rows = x.size(0), cols = x.size(1);
  auto q = at::empty({rows, cols}, x.options().dtype(at::kChar));
  auto e = at::empty({rows, (cols + 31) / 32}, x.options().dtype(at::kByte));
  if (x.numel() == 0) return {q, e};
  ok(tnops_quantize_int8(x.data_ptr(), xF32, bytes(q), bytes(e), rows, asInt(cols, "columns"),
                         streamOf(x)),
     "tnops_quantize_int8");
  return {q, e};
}

void needInt8(const at::Tensor& q, const at::Tensor& e) {
  need(q, at::kChar, "q");
  need(e, at::kByte, "e");
  TORCH_CHECK(q.dim() == 2 && e.dim() == 2 && e.size(0) == q.size(0) &&
                  e.size(1) == (q.size(1) + 31) / 32,
              "8-bit blocks: want q [rows, cols] and e [rows, ceil(cols / 32)]");
  sameDevice(q, e, "e");
}

at::Tensor dequantizeInt8(const at::Tensor& q, const at::Tensor& e, bool outF32) {
  needInt8(q, e);
  c10::cuda::CUDAGuard g(q.device());
  auto x = at::empty(q.sizes(), q.options().dtype(outF32 ? at::kFloat : at::kBFloat16));
  if (x.numel() == 0) return x;
  ok(tnops_dequantize_int8(bytes(q), bytes(e), x.data_ptr(), outF32 ? 1 : 0, q.size(0),
                           asInt(q.size(1), "columns"), streamOf(q)),
     "tnops_dequantize_int8");
  return x;
}

// x bf16 [rows, ins], w bf16 [outs, ins], bias bf16 [outs] -> (act bf16, and
// with `keep` the sums before the GELU in 8-bit blocks, else two undefined tensors)
std::vector<at::Tensor> linearGeluInt8(const at::Tensor& x, const at::Tensor& w,
                                       const at::Tensor& bias, bool keep) {
  need(x, at::kBFloat16, "x");
  need(w, at::kBFloat16, "weight");
  need(bias, at::kBFloat16, "bias");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && bias.numel() == w.size(0),
              "linear_gelu_int8: want x [rows, ins], weight [outs, ins], bias [outs]");
  TORCH_CHECK(w.size(0) % 8 == 0 && w.size(1) % 8 == 0,
              "linear_gelu_int8: the layer's sizes must be multiples of 8");
  sameDevice(x, w, "weight");
  sameDevice(x, bias, "bias");
  c10::cuda::CUDAGuard g(x.device());
  const int rows = asInt(x.size(0), "rows"), outs = asInt(w.size(0), "outputs"),
            ins = asInt(w.size(1), "inputs");
  auto act = at::empty({rows, outs}, x.options());
  at::Tensor q, e;
  if (keep) {
    q = at::empty({rows, outs}, x.options().dtype(at::kChar));
    e = at::empty({rows, (outs + 31) / 32}, x.options().dtype(at::kByte));
  }
  if (rows == 0) return {act, q, e};
  ok(tnops_linear_gelu_int8(x.data_ptr(), w.data_ptr(), bias.data_ptr(), act.data_ptr(),
                            static_cast<uint8_t*>(orNull(q)), static_cast<uint8_t*>(orNull(e)),
                            rows, outs, ins, streamOf(x)),
     "tnops_linear_gelu_int8");
  return {act, q, e};
}

// g bf16 [M, N] -> db [N] (column sums) of type st
at::Tensor biasGradient(const at::Tensor& grad, at::ScalarType st, const Opt& out) {
  need(grad, at::kBFloat16, "grad");
  TORCH_CHECK(grad.dim() == 2 && grad.size(1) % 8 == 0, "bias_grad: want [M, N] with N % 8 == 0");
  c10::cuda::CUDAGuard g(grad.device());
  const int M = asInt(grad.size(0), "rows"), N = asInt(grad.size(1), "columns");
  auto db = out ? *out : at::empty({N}, grad.options().dtype(st));
  needSums(grad, db, st, N);
  if (M == 0) return db.zero_();
  auto part = columnParts(grad, M, N);
  auto* gp = static_cast<uint16_t*>(grad.data_ptr());
  ok(st == at::kFloat
         ? tnops_bias_grad(gp, db.data_ptr<float>(), part, M, N, streamOf(grad))
         : tnops_bias_grad_bf16(gp, static_cast<uint16_t*>(db.data_ptr()), part, M, N,
                                streamOf(grad)),
     "tnops_bias_grad");
  return db;
}

// gy bf16 [M, N], pre in 8-bit blocks -> (gpre bf16 [M, N], db [N] of type st, or
// undefined where it is not wanted)
std::vector<at::Tensor> geluBwdBiasInt8(const at::Tensor& gy, const at::Tensor& q,
                                        const at::Tensor& e, bool wantDb, at::ScalarType st,
                                        const Opt& dbOut) {
  need(gy, at::kBFloat16, "grad_y");
  needInt8(q, e);
  TORCH_CHECK(gy.dim() == 2 && gy.sizes() == q.sizes() && gy.size(1) % 8 == 0,
              "gelu_bwd_bias_int8: want equal [M, N] with N % 8 == 0");
  sameDevice(gy, q, "q");
  c10::cuda::CUDAGuard g(gy.device());
  const int M = asInt(gy.size(0), "rows"), N = asInt(gy.size(1), "columns");
  auto gpre = at::empty_like(gy);
  at::Tensor db;
  ColumnParts part;
  if (wantDb) {
    db = dbOut ? *dbOut : at::empty({N}, gy.options().dtype(st));
    needSums(gy, db, st, N);
    if (M == 0) db.zero_();
    part = columnParts(gy, M, N);
  }
  if (M == 0) return {gpre, db};
  ok(tnops_gelu_bwd_bias_int8(static_cast<uint16_t*>(gy.data_ptr()), bytes(q), bytes(e),
                              static_cast<uint16_t*>(gpre.data_ptr()), orNull(db),
                              st == at::kFloat, part, M, N, streamOf(gy)),
     "tnops_gelu_bwd_bias_int8");
  return {gpre, db};
}

// g [rows, outs], w [outs, ins], x in 8-bit blocks [rows, ins] (none: no dw)
// -> (dx bf16, dw)
std::vector<at::Tensor> linearGradsInt8(const at::Tensor& grad, const at::Tensor& w, const Opt& q,
                                        const Opt& e, bool wantDx, bool dwF32, const Opt& dwOut) {
  need(grad, at::kBFloat16, "grad");
  need(w, at::kBFloat16, "weight");
  TORCH_CHECK(grad.dim() == 2 && w.dim() == 2 && grad.size(1) == w.size(0),
              "linear_grads_int8: want grad [rows, outs], weight [outs, ins]");
  TORCH_CHECK(w.size(0) % 8 == 0 && w.size(1) % 8 == 0,
              "linear_grads_int8: the layer's sizes must be multiples of 8");
  sameDevice(grad, w, "weight");
  const bool wantDw = q.has_value();
  if (wantDw) {
    needInt8(*q, *e);
    TORCH_CHECK(q->size(0) == grad.size(0) && q->size(1) == w.size(1),
                "linear_grads_int8: want q [rows, ins]");
    sameDevice(grad, *q, "q");
  }
  c10::cuda::CUDAGuard g(grad.device());
  const int rows = asInt(grad.size(0), "rows"), outs = asInt(w.size(0), "outputs"),
            ins = asInt(w.size(1), "inputs");
  at::Tensor dx, dw;
  if (wantDx) dx = at::empty({rows, ins}, grad.options());
  if (wantDw) {
    const auto st = dwF32 ? at::kFloat : at::kBFloat16;
    dw = dwOut ? *dwOut : at::empty({outs, ins}, w.options().dtype(st));
    need(dw, st, "dw_out");
    TORCH_CHECK(dw.numel() == w.numel(), "linear_grads_int8: dw_out must match weight");
    sameDevice(grad, dw, "dw_out");
  }
  if (rows == 0 && wantDw) dw.zero_();
  if (rows == 0 || (!wantDx && !wantDw)) return {dx, dw};
  at::Tensor x;
  if (wantDw) x = dequantizeInt8(*q, *e, false);
  const size_t scratchBytes = tnops_linear_grads_scratch(rows, outs, ins, wantDx, wantDw);
  auto scratch = scratchOf(scratchBytes, grad);
  ok(tnops_linear_grads(grad.data_ptr(), outs, w.data_ptr(), orNull(x), orNull(dx), orNull(dw),
                        dwF32 ? 1 : 0, rows, outs, ins, orNull(scratch), scratchBytes,
                        streamOf(grad)),
     "tnops_linear_grads");
  return {dx, dw};
}

// -- autograd ----------------------------------------------------------------------
//
// The operators' autograd functions are C++: a small call's time is the host's,
// and Python functions take several times as long on both ways. Where nothing
// asks for a derivative they are passed by, and nothing is kept for one. They
// have no forward mode and refuse an input with a tangent, also under no_grad;
// passed by, it would come back without one.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wantsDerivative(std::initializer_list<const at::Tensor*> inputs) {
  const bool backward = at::GradMode::is_enabled();
  for (const at::Tensor* t : inputs)
    if (t != nullptr &&
        ((backward && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined()))
      return true;
  return false;
}

void onceDifferentiable(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " cannot be differentiated twice");
}

// Where the gradient of parameter p is to be written: its slice of a flat
// gradient buffer, when it has one (`has`) that the gradient may take now
// (ops.fused.grad_destination, asked when the backward pass runs: it hands a
// slice out once per pass, so that a parameter that is used twice gets two
// gradients to add) and whose type and layout are the gradient's.
Opt destination(const at::Tensor& p, bool has, at::ScalarType st) {
  if (!has) return c10::nullopt;
  py::gil_scoped_acquire gil;
  const py::object d =
      py::module_::import("tiny_nccl_b200.ops.fused").attr("grad_destination")(p);
  if (d.is_none()) return c10::nullopt;
  const auto t = d.cast<at::Tensor>();
  if (t.scalar_type() != st || !t.is_contiguous() ||
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0)
    return c10::nullopt;
  return t.detach();
}
// Whether p may have one: an attribute of the parameter's Python object.
bool hasDestination(const at::Tensor& p) {
  const py::object t = py::cast(p);
  return py::hasattr(t, "_tn_grad_dest") && !t.attr("_tn_grad_dest").is_none();
}
Opt savedOpt(AutogradContext* ctx, const char* key) {
  const auto& v = ctx->saved_data[key];
  return v.isNone() ? Opt() : Opt(v.toTensor());
}
// The products read 16-byte pieces: a tensor that is not contiguous, or starts
// off that boundary, is copied.
at::Tensor packed(const at::Tensor& t) {
  const auto c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
at::Tensor bf16Copy(const at::Tensor& p, const Opt& copy) {
  return packed(copy ? *copy : p.detach().to(at::kBFloat16));
}
// x [*, width] as bf16 rows.
at::Tensor bf16Rows(const at::Tensor& x) {
  return packed(x.reshape({-1, x.size(-1)}).to(at::kBFloat16));
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& w, const Opt& p,
                            const at::Tensor& idx, const Opt& positions, int64_t seq, double scale,
                            bool outF32, bool dwDest, bool dpDest) {
    // The parameters themselves, for what their gradients look like: their
    // values are not needed, so they may change before the backward pass.
    ctx->saved_data["w"] = w;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seq"] = seq;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["dw"] = dwDest;
    ctx->saved_data["dp"] = dpDest;
    at::Tensor orderW, orderP;
    auto y = embeddingFwd(idx, positions, w, p, seq, scale, outF32,
                          w.requires_grad() ? &orderW : nullptr,
                          p && p->requires_grad() ? &orderP : nullptr);
    ctx->save_for_backward({orderW, orderP});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    onceDifferentiable("embedding");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor w = ctx->saved_data["w"].toTensor();
    const Opt p = savedOpt(ctx, "p");
    const bool wantW = ctx->needs_input_grad(0), wantP = p && ctx->needs_input_grad(1);
    const auto st = w.scalar_type();
    const auto g = grads[0].contiguous();
    const auto d = embeddingGrad(
        g, saved[0], saved[1], ctx->saved_data["seq"].toInt(),
        wantW ? w.size(0) : 0, wantP ? p->size(0) : 0, ctx->saved_data["scale"].toDouble(),
        st == at::kFloat, wantW ? destination(w, ctx->saved_data["dw"].toBool(), st) : Opt(),
        wantP ? destination(*p, ctx->saved_data["dp"].toBool(), st) : Opt());
    return {d[0], d[1], {}, {}, {}, {}, {}, {}, {}};
  }
};

// The checks that Python callers see as TypeError and ValueError stand here as
// well: in Python they take a third of a decoding step's call.
at::Tensor embedding(const at::Tensor& idx, const at::Tensor& weight, const Opt& posWeight,
                     const Opt& positions, double scale, c10::optional<at::ScalarType> outType) {
  auto floating = [](at::ScalarType t, const char* name) {
    if (t != at::kFloat && t != at::kBFloat16)
      throw py::type_error(std::string(name) + " must be float32 or bfloat16, not " +
                           c10::toString(t));
  };
  auto index = [](const at::Tensor& t, const char* name) {
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
      throw py::type_error(std::string(name) + " must be int64 or int32, not " +
                           c10::toString(t.scalar_type()));
  };
  floating(weight.scalar_type(), "weight");
  if (weight.dim() != 2) throw py::value_error("weight must be [vocab, width]");
  if (posWeight) {
    if (posWeight->dim() != 2 || posWeight->size(1) != weight.size(1))
      throw py::value_error("pos_weight must be [context, width], of weight's width");
    if (posWeight->scalar_type() != weight.scalar_type())
      throw py::type_error("weight and pos_weight must have one dtype");
  }
  if (outType) floating(*outType, "out_dtype");
  index(idx, "idx");
  if (positions) {
    if (!posWeight) throw py::value_error("positions without pos_weight");
    if (positions->sizes() != idx.sizes())
      throw py::value_error("positions must have idx's shape");
    index(*positions, "positions");
  }
  const auto w = weight.contiguous();
  const Opt p = posWeight ? Opt(posWeight->contiguous()) : Opt();
  auto flat = [](const at::Tensor& t) {
    return (t.dim() == 1 ? t : t.reshape({-1})).to(at::kLong).contiguous();
  };
  const auto token = flat(idx);
  const Opt position = positions ? Opt(flat(*positions)) : Opt();
  const int64_t seq = idx.dim() > 0 ? idx.size(-1) : 1;
  const bool outF32 = outType.value_or(w.scalar_type()) == at::kFloat;
  auto y = wantsDerivative({&w, p ? &*p : nullptr})
               ? EmbeddingFn::apply(w, p, token, position, seq, scale, outF32,
                                    hasDestination(w), p && hasDestination(*p))
               : embeddingFwd(token, position, w, p, seq, scale, outF32);
  if (idx.dim() == 1) return y;
  auto shape = idx.sizes().vec();
  shape.push_back(w.size(1));
  return y.view(shape);
}

struct LinearCeFn : torch::autograd::Function<LinearCeFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const Opt& w16, const at::Tensor& target, int64_t classes,
                            int64_t reduction, bool dwDest) {
    const auto wb = bf16Copy(w, w16);
    const auto r = linearCeFwd(x, wb, target, classes, reduction);
    ctx->save_for_backward({x, wb, target, r[1], r[3]});
    ctx->saved_data["w"] = w;
    ctx->saved_data["classes"] = classes;
    ctx->saved_data["mean"] = reduction == kMean;
    ctx->saved_data["dw"] = dwDest;
    return reduction == kNone ? r[0] : r[2];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    onceDifferentiable("linear_cross_entropy");
    const auto s = ctx->get_saved_variables();
    const at::Tensor w = ctx->saved_data["w"].toTensor();
    const auto st = w.scalar_type();
    const auto g = grads[0].reshape({-1}).to(at::kFloat).contiguous();
    const bool wantW = ctx->needs_input_grad(1);
    const auto d = linearCeBwd(
        s[0], s[1], s[2], s[3], g, ctx->saved_data["mean"].toBool() ? Opt(s[4]) : Opt(),
        ctx->saved_data["classes"].toInt(), ctx->needs_input_grad(0), wantW, st == at::kFloat,
        wantW ? destination(w, ctx->saved_data["dw"].toBool(), st) : Opt(), kCeBudget);
    return {d[0], d[1], {}, {}, {}, {}, {}};
  }
};

at::Tensor linearCrossEntropy(const at::Tensor& x, const at::Tensor& w, const Opt& w16,
                              const at::Tensor& target, int64_t classes, int64_t reduction) {
  const auto xb = bf16Rows(x);
  const auto t = target.reshape({-1}).contiguous();
  at::Tensor loss;
  if (wantsDerivative({&x, &w})) {
    loss = LinearCeFn::apply(xb, w, w16, t, classes, reduction, hasDestination(w));
  } else {
    const auto r = linearCeFwd(xb, bf16Copy(w, w16), t, classes, reduction);
    loss = reduction == kNone ? r[0] : r[2];
  }
  return reduction == kNone ? loss.view(target.sizes()) : loss;
}

// y, and with gelu and `keep` the sums before it in 8-bit blocks.
variable_list linearInt8Out(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b,
                            bool gelu, bool keep) {
  if (gelu) return linearGeluInt8(x, w, b, keep);
  c10::impl::ExcludeDispatchKeyGuard guard(c10::DispatchKey::AutocastCUDA);
  return {at::addmm(b, x, w.t())};
}

struct LinearInt8Fn : torch::autograd::Function<LinearInt8Fn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const at::Tensor& b, const Opt& w16, const Opt& b16, bool gelu,
                            bool dwDest, bool dbDest) {
    const auto wb = bf16Copy(w, w16);
    const auto out = linearInt8Out(x, wb, bf16Copy(b, b16), gelu, true);
    variable_list keep{wb};
    keep.insert(keep.end(), out.begin() + 1, out.end());
    // The inputs are read by the weight's gradient alone.
    const auto q = w.requires_grad() ? quantizeInt8(x) : variable_list(2);
    keep.insert(keep.end(), q.begin(), q.end());
    ctx->save_for_backward(keep);
    ctx->saved_data["w"] = w;
    ctx->saved_data["b"] = b;
    ctx->saved_data["dw"] = dwDest;
    ctx->saved_data["db"] = dbDest;
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    onceDifferentiable("a linear layer with 8-bit activations");
    const auto s = ctx->get_saved_variables();
    const bool gelu = s.size() == 5;
    const at::Tensor w = ctx->saved_data["w"].toTensor(), b = ctx->saved_data["b"].toTensor();
    auto g = packed(grads[0]);
    const bool wantW = ctx->needs_input_grad(1);
    const bool wantB = ctx->needs_input_grad(2);
    const auto bt = b.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
    const Opt dbOut = wantB ? destination(b, ctx->saved_data["db"].toBool(), bt) : Opt();
    at::Tensor db;
    if (gelu) {
      auto r = geluBwdBiasInt8(g, s[1], s[2], wantB, bt, dbOut);
      g = r[0];
      db = r[1];
    } else if (wantB) {
      db = biasGradient(g, bt, dbOut);
    }
    const auto st = w.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
    const at::Tensor &q = s[s.size() - 2], &e = s[s.size() - 1];
    const auto d = linearGradsInt8(
        g, s[0], wantW ? Opt(q) : Opt(), wantW ? Opt(e) : Opt(), ctx->needs_input_grad(0),
        st == at::kFloat, wantW ? destination(w, ctx->saved_data["dw"].toBool(), st) : Opt());
    return {d[0], d[1], db, {}, {}, {}, {}, {}};
  }
};

at::Tensor linearInt8(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b,
                      const Opt& w16, const Opt& b16, bool gelu) {
  TORCH_CHECK(w.dim() == 2 && b.dim() == 1 && b.size(0) == w.size(0) && x.dim() > 0 &&
                  x.size(-1) == w.size(1),
              "linear_int8: want x [*, ins], weight [outs, ins], bias [outs]");
  TORCH_CHECK(w.size(0) % 8 == 0 && w.size(1) % 8 == 0,
              "linear_int8: the layer's sizes must be multiples of 8");
  const auto xb = bf16Rows(x);
  auto y = wantsDerivative({&x, &w, &b})
               ? LinearInt8Fn::apply(xb, w, b, w16, b16, gelu, hasDestination(w),
                                     hasDestination(b))
               : linearInt8Out(xb, bf16Copy(w, w16), bf16Copy(b, b16), gelu, false)[0];
  auto shape = x.sizes().vec();
  shape.back() = w.size(0);
  return y.view(shape);
}

}  // namespace

void registerTrainOps(py::module_& ops) {
  ops.def("embedding", &embedding, py::arg("idx"), py::arg("weight"), py::arg("pos_weight"),
          py::arg("positions"), py::arg("scale"), py::arg("out_dtype"));
  ops.def("linear_cross_entropy", &linearCrossEntropy, py::arg("x"), py::arg("weight"),
          py::arg("weight_bf16"), py::arg("target"), py::arg("classes"), py::arg("reduction"));
  ops.def("linear_int8", &linearInt8, py::arg("x"), py::arg("weight"), py::arg("bias"),
          py::arg("weight_bf16"), py::arg("bias_bf16"), py::arg("gelu"));
  ops.def("linear_gelu_int8", &linearGeluInt8, py::arg("x"), py::arg("weight"), py::arg("bias"),
          py::arg("keep") = true);
  ops.def("linear_ce_fwd", &linearCeFwd, py::arg("x"), py::arg("weight"), py::arg("target"),
          py::arg("classes"), py::arg("reduction"));
  ops.def("linear_ce_piece", &tnops_linear_ce_piece, py::arg("rows"), py::arg("width"),
          py::arg("classes"), py::arg("budget"));
  ops.def("linear_ce_bwd", &linearCeBwd, py::arg("x"), py::arg("weight"), py::arg("target"),
          py::arg("lse"), py::arg("grad"), py::arg("share"), py::arg("classes"),
          py::arg("want_dx"), py::arg("want_dw"), py::arg("dw_f32"),
          py::arg("dw_out") = py::none(), py::arg("budget") = kCeBudget);
  ops.def("quantize_int8", &quantizeInt8, py::arg("x"));
  ops.def("dequantize_int8", &dequantizeInt8, py::arg("q"), py::arg("e"), py::arg("out_f32"));
}
