"""Training operators (csrc/ops): token and position embedding, linear layer +
softmax cross-entropy in pieces of the vocabulary, and 8-bit activation
blocks. Their autograd functions are native too (csrc/torch/train_ext.cpp); a
second differentiation and forward-mode inputs (dual tensors) raise.
Like :mod:`.fused`, every function calls the native kernels; a missing
extension or an unsupported argument raises.
"""
from __future__ import annotations

import torch

from .fused import _ops, current_copy


def _needs_float(name: str, t: torch.Tensor) -> None:
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name} must be float32 or bfloat16, not {t.dtype}")


def _as_rows(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dim() == 0:
        raise ValueError(f"{name} must have at least one dimension")
    return t.reshape(t.shape[:-1].numel(), t.shape[-1]).contiguous()


def embedding(idx: torch.Tensor, weight: torch.Tensor, pos_weight: torch.Tensor | None = None,
              positions: torch.Tensor | None = None, scale: float = 1.0,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """scale * weight[idx] + pos_weight[positions], of shape [*idx.shape, width].

    weight [vocab, width] and pos_weight [context, width] (optional) are both
    float32 or both bfloat16; the sum is formed in fp32 and rounded once to
    ``out_dtype`` (float32 or bfloat16; the tables' type when None).
    ``positions`` (idx's shape) gives each token's position, e.g. when single
    tokens are decoded; None counts along idx's last dimension. idx and
    positions are int64 (int32 is converted). An index outside its table, such
    as a negative one for padding, adds nothing and gets no gradient.

    The gradients of both tables are fp32 sums over the rows sorted by token (in
    row order within blocks, which are then added), bit-identical from run to
    run; a row that no token names gets zero."""
    return _ops().embedding(idx, weight, pos_weight, positions, scale, out_dtype)


_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         classes: int = 0, reduction: str = "mean") -> torch.Tensor:
    """Softmax cross-entropy of the logits x W^T against int64 targets, without
    the [rows, vocabulary] logits in memory.

    x [*, width] is taken in bf16, weight [vocab, width] (e.g. the tied token
    embedding; fp32 or bf16) through its bf16 copy; logits, softmax and losses
    are fp32. The first ``classes`` rows of weight are classes (all when 0),
    the rest is padding with zero gradient. A target outside [0, classes) does
    not count: zero loss, zero gradient, and not part of the mean.
    ``reduction``: "mean" over the rows that count (0 when none does), "sum",
    or "none" for fp32 losses of target's shape.

    Backward: the gradient of x is bf16, that of weight has weight's type; the
    gradient of the logits is rounded to bf16 between the products (a factor
    that all rows share is not), a piece of the vocabulary of at most 512 MiB
    (or 256 classes) at a time. A row of x that is not finite makes the weight's
    gradient NaN also where its target does not count (its share is 0 x), but
    no other row's loss or gradient. width must be a multiple of 8."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    _needs_float("weight", weight)
    if weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"weight must be [vocab, {x.shape[-1]}], not {tuple(weight.shape)}")
    if target.dtype != torch.int64:
        raise TypeError(f"target must be int64, not {target.dtype}")
    if target.numel() * x.shape[-1] != x.numel():
        raise ValueError("target must have one entry per row of x")
    return _ops().linear_cross_entropy(x, weight, current_copy(weight), target,
                                       int(classes) or weight.shape[0], _REDUCTIONS[reduction])


def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (float32 or bfloat16) as (q, e): whole numbers in [-127, 127] (int8,
    x's shape) and one exponent byte for each 32 neighbours of the last
    dimension (uint8); value = q * 2^(e - 133). Off by at most half a step, 1/127.5
    of the block's largest magnitude (magnitudes below 2^-127 have steps of
    2^-133); a block with an infinity or a NaN reads back as NaN."""
    _needs_float("x", x)
    q, e = _ops().quantize_int8(_as_rows("x", x))
    return q.view(x.shape), e.view(*x.shape[:-1], e.shape[1])


def dequantize_int8(q: torch.Tensor, e: torch.Tensor,
                    dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of :func:`quantize_int8`'s blocks (exact in bfloat16 and
    float32)."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"dtype must be float32 or bfloat16, not {dtype}")
    x = _ops().dequantize_int8(_as_rows("q", q), _as_rows("e", e), dtype == torch.float32)
    return x.view(q.shape)
