"""Host side of the training operators at their edges, without a GPU: what the
C launchers refuse before any CUDA call."""
import pytest
import torch

from test_train_ops_cpu import A, I, P, _launcher, _refuses


def test_gelu_launcher_refuses_half_of_the_8_bit_sums(built):
    """Both parts of the 8-bit form are wanted, or neither."""
    f = _launcher("tnops_linear_gelu_int8", P, P, P, P, P, P, I, I, I, P)
    _refuses(f, [A, A, A, A, A, A, 4, 64, 64, None], [(4, None), (5, None)])


def test_gelu_gradient_launcher_with_and_without_a_bias_gradient(built):
    """Without db there are no column sums; the refusals are the same."""
    f = _launcher("tnops_gelu_bwd_bias_int8", P, P, P, P, P, I, P, I, I, P)
    _refuses(f, [A, A, A, A, None, 1, None, 64, 768, None],
             [(0, A + 8), (1, A + 4), (3, A + 8), (7, 0), (8, 770)])
    _refuses(f, [A, A, A, A, A, 1, A, 6400, 768, None], [(6, None)])  # sums without scratch
    f = _launcher("tnops_bias_grad", P, P, P, I, I, P)
    _refuses(f, [A, A, A, 64, 768, None], [(1, None)])


def test_int8_blocks_need_a_dimension(built):
    from tiny_nccl_b200 import ops
    x = torch.zeros(())
    with pytest.raises(ValueError):
        ops.quantize_int8(x)
    with pytest.raises(ValueError):
        ops.dequantize_int8(x.to(torch.int8), torch.zeros(1, dtype=torch.uint8))
