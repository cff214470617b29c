"""Fused sm_100a model kernels: residual-add + LayerNorm, softmax
cross-entropy, multi-tensor AdamW, the bias / GELU-backward gradients
behind the autograd linears (which may keep their activations in 8 bits),
token and position embedding, and the LM head's cross-entropy without the
logits in memory."""
from .fused import (add_layer_norm, bf16_weight, cross_entropy, launch_count, layer_norm,
                    linear, linear_gelu, linear_nobias)
from .optim import AdamW, gpt2_param_groups
from .train import dequantize_int8, embedding, linear_cross_entropy, quantize_int8

__all__ = ["add_layer_norm", "layer_norm", "cross_entropy", "linear", "linear_gelu",
           "linear_nobias", "bf16_weight", "AdamW", "gpt2_param_groups", "launch_count",
           "embedding", "linear_cross_entropy", "quantize_int8", "dequantize_int8"]
