"""Host side of the training operators at their edges, without a GPU: what the
C launchers refuse before any CUDA call."""
from test_train_ops_cpu import A, I, P, _launcher, _refuses


def test_gelu_launcher_refuses_half_of_the_8_bit_sums(built):
    """Both parts of the 8-bit form are wanted, or neither."""
    f = _launcher("tnops_linear_gelu_int8", P, P, P, P, P, P, I, I, I, P)
    _refuses(f, [A, A, A, A, A, A, 4, 64, 64, None], [(4, None), (5, None)])
