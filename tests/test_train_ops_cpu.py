"""Host side of the training operators, without a GPU: refusals in Python, in
the binding and in the C launchers (before any CUDA call), and the piece rule
of the cross-entropy."""
import ctypes
import os

import pytest
import torch

from conftest import ROOT, run

P, I, L, F, S = (ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float,
                 ctypes.c_size_t)
A = 1 << 20  # an aligned address; never dereferenced on these paths


def _launcher(name, *types):
    f = getattr(ctypes.CDLL(os.path.join(ROOT, "tiny_nccl_b200", "lib", "libtnccl_ops.so")), name)
    f.argtypes, f.restype = types, I
    return f


def _scratch(name, *args):
    f = _launcher(name, *[I] * len(args))
    f.restype = S
    return f(*args)


def _refuses(f, good, bad):
    for i, v in bad:
        args = list(good)
        args[i] = v
        assert f(*args) == 1, (i, v)


def test_linear_grads_launcher_refuses(built):
    f = _launcher("tnops_linear_grads", P, L, P, P, P, P, I, I, I, I, P, S, P)
    # 8192 rows of a 768 -> 768 layer: dW's nine tiles are cut.
    need = _scratch("tnops_linear_grads_scratch", 8192, 768, 768, 1, 1)
    assert need > 0 and need % (256 * 256 * 4) == 0
    good = [A, 768, A, A, A, A, 0, 8192, 768, 768, A, need, None]
    _refuses(f, good, [(0, None), (0, A + 8), (1, 764), (1, 760), (2, A + 2), (2, None),
                       (3, A + 4), (3, None), (4, A + 8), (5, A + 8), (7, 0), (8, 0), (9, 0),
                       (9, 764), (10, None), (10, A + 8), (11, need - 1)])
    assert _scratch("tnops_linear_grads_scratch", 0, 768, 768, 1, 1) == 0
    assert _scratch("tnops_linear_grads_scratch", 33, 512, 128, 1, 1) == 0


def test_linear_ce_launchers_refuse(built):
    f = _launcher("tnops_linear_ce_fwd", P, P, P, P, P, P, I, I, I, P)
    good = [A, A, A, A, A, A, 4, 64, 100, None]
    _refuses(f, good, [(0, A + 8), (1, A + 8), (6, 0), (7, 0), (7, 60), (8, 0)])
    f = _launcher("tnops_linear_ce_bwd", P, P, P, P, P, I, P, P, I, P, P, S, P, P, I, I, I, I, I, P)
    good = [A, A, A, A, A, 0, A, A, 256, A, None, 0, A, A, 1, 4, 64, 300, 304, None]
    _refuses(f, good, [(0, A + 8), (1, A + 8), (5, 2), (7, A + 16), (8, 0), (8, 264), (9, None),
                       (9, A + 4), (10, A + 8), (12, A + 8), (13, A + 4), (15, 0),
                       (16, 60), (17, 0), (18, 299)])
    # The scratch of the first pieces and of the last, shorter one.
    a, b, c = (_scratch("tnops_linear_grads_scratch", 1024, n, 768, 1, 1) for n in (768, 232, 1000))
    assert _scratch("tnops_linear_ce_scratch", 1024, 768, 1000, 1000, 768, 1, 1) == max(a, b)
    assert _scratch("tnops_linear_ce_scratch", 1024, 768, 1000, 1000, 1024, 1, 1) == c
    f = _launcher("tnops_linear_ce_mean", P, P, P, P, I, I, I, P)
    assert f(A, A, A, A, 0, 5, 1, None) == 1


def test_embedding_launchers_refuse(built):
    f = _launcher("tnops_embedding_fwd", P, P, P, P, I, P, I, L, I, I, I, I, F, P, P, P)
    good = [A, None, A, A, 1, A, 1, 8, 4, 100, 16, 64, 1.0, A, None, None]
    _refuses(f, good, [(7, 0), (7, 1 << 31), (8, 0), (9, 0), (10, 0), (11, 0), (13, A + 8),
                       (9, (1 << 31) - 1), (14, A)])  # an order of positions that are not given
    f = _launcher("tnops_embedding_grad", P, I, P, P, I, F, P, I, P, I, I, L, I, P, P)
    good = [A, 1, A, A, 100, 1.0, None, 4, A, 50, 1, 8, 64, A, None]
    _refuses(f, good, [(2, None), (4, 0), (7, 0), (7, 3), (9, 0), (11, 0), (11, 1 << 31),
                       (12, 0), (13, None), (13, A + 8), (2, A + 8), (6, A + 8)])
    assert f(A, 1, A, None, 100, 1.0, None, 4, None, 50, 1, 8, 64, A, None) == 1


def test_embedding_scratch_grows_with_its_parts(built):
    f = _launcher("tnops_embedding_grad_scratch", L, I, I)
    f.restype = ctypes.c_size_t
    assert f(0, 64, 2) == 0 and f(1, 1, 1) % 16 == 0
    # Sorted keys and their rows, 8 bytes a row, and two rows of fp32 partial
    # sums for each 16 rows.
    assert f(65536, 1024, 2) == 2 * (8 * 65536 + 8 * 4096 * 1024)


def test_embedding_order_bytes(built):
    """One chunk: sorted indices and rows; more: a key per row, of 64 bits where
    index and place do not fit 32."""
    f = _launcher("tnops_embedding_order_bytes", L, I)
    f.restype = ctypes.c_size_t
    assert [f(n, 50304) for n in (0, 1, 1023, 1024, 1025, 16384, 16385, 1 << 31)] == [
        0, 32, 2 * 4096, 2 * 4096, 4112, 65536, 65552, 0]
    assert f(2000, (1 << 22) - 2) == 8000 and f(2000, (1 << 22) - 1) == 16000
    assert f(30000, (1 << 21) - 2) == 120000 and f(30000, (1 << 21) - 1) == 240000
    assert f(100000, (1 << 20) - 2) == 400000 and f(100000, (1 << 20) - 1) == 800000
    assert f(20000, 0) == 0 and f(20000, (1 << 31) - 1) == 0


def test_int8_launchers_refuse(built):
    f = _launcher("tnops_quantize_int8", P, I, P, P, L, I, P)
    _refuses(f, [A, 0, A, A, 4, 64, None], [(4, 0), (5, 0)])
    f = _launcher("tnops_dequantize_int8", P, P, P, I, L, I, P)
    _refuses(f, [A, A, A, 0, 4, 64, None], [(4, 0), (5, 0)])
    f = _launcher("tnops_linear_gelu_int8", P, P, P, P, P, P, I, I, I, P)
    _refuses(f, [A, A, A, A, A, A, 4, 64, 64, None],
             [(0, A + 8), (1, A + 8), (2, A + 4), (2, None), (3, A + 16), (4, A + 8), (5, A + 2),
              (6, 0), (7, 0), (7, 60), (8, 0), (8, 60)])
    f = _launcher("tnops_gelu_bwd_bias_int8", P, P, P, P, P, I, P, I, I, P)
    for db_f32 in (0, 1):
        _refuses(f, [A, A, A, A, A, db_f32, A, 64, 768, None],
                 [(0, A + 8), (1, A + 4), (3, A + 8), (7, 0), (8, 770)])
    f = _launcher("tnops_bias_grad_bf16", P, P, P, I, I, P)
    _refuses(f, [A, A, A, 64, 768, None], [(0, A + 8), (3, 0), (4, 770)])


def test_pair_schedule(built):
    """Every K block of every tile belongs to one SM pair's part, and the
    joining kernel adds exactly the parts of cut tiles that were written."""
    r = run([os.path.join(ROOT, "build", "bin", "pair_schedule_test")], timeout=300)
    assert r.returncode == 0 and "pair schedule ok" in r.stdout, r.stderr


def test_pair_pipeline_model(built):
    """The barriers of the pair and panel products, as threads: short sums
    behind a slow epilogue, tiles with rows in one half only, panels that
    change."""
    r = run([os.path.join(ROOT, "build", "bin", "pair_pipeline_model_test")], timeout=300)
    assert r.returncode == 0 and "pair pipelines: PASS" in r.stdout, r.stdout + r.stderr


def test_python_refusals(built):
    from tiny_nccl_b200 import ops
    w, p = torch.zeros(10, 8), torch.zeros(6, 8)
    idx = torch.zeros(2, 3, dtype=torch.int64)
    for error, args, kw in [
            (TypeError, (idx.float(), w), {}),
            (TypeError, (idx, w.half()), {}),
            (TypeError, (idx, w, p.bfloat16()), {}),
            (TypeError, (idx, w), dict(out_dtype=torch.float16)),
            (ValueError, (idx, w, torch.zeros(6, 9)), {}),
            (ValueError, (idx, w[0]), {}),
            (ValueError, (idx, w), dict(positions=idx)),
            (ValueError, (idx, w, p), dict(positions=idx[0])),
            (TypeError, (idx, w, p), dict(positions=idx.float())),
            (RuntimeError, (idx, w), {})]:  # not on a GPU
        with pytest.raises(error):
            ops.embedding(*args, **kw)
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for error, args, kw in [
            (ValueError, (x, w, t), dict(reduction="max")),
            (ValueError, (x, torch.zeros(10, 16), t), {}),
            (ValueError, (x, w, t[:3]), {}),
            (TypeError, (x, w, t.int()), {}),
            (TypeError, (x, w.half(), t), {}),
            (RuntimeError, (x, w, t), {})]:
        with pytest.raises(error):
            ops.linear_cross_entropy(*args, **kw)
    with pytest.raises(TypeError):
        ops.quantize_int8(x.half())
    with pytest.raises(TypeError):
        ops.dequantize_int8(x.to(torch.int8), torch.zeros(4, 1, dtype=torch.uint8), torch.float16)
    with pytest.raises(RuntimeError):
        ops.quantize_int8(x)
    for f in (ops.linear, ops.linear_gelu):
        with pytest.raises(ValueError):
            f(x, w, torch.zeros(10), activations="int4")
        # Sizes are refused before anything is computed, not in the backward pass.
        with pytest.raises(RuntimeError, match="multiples of 8"):
            f(x, w, torch.zeros(10), activations="int8")
        with pytest.raises(RuntimeError, match="bias"):
            f(x, w[:8], torch.zeros(10), activations="int8")
        with pytest.raises(RuntimeError, match="weight"):
            f(x[:, :4], w[:8], torch.zeros(8), activations="int8")


def test_gradient_slice_is_handed_out_once_per_backward():
    """A parameter used by two functions in one backward pass: only the first
    gets its flat slice, so that the two gradients add up; the next pass hands
    it out again."""
    from tiny_nccl_b200.ops.fused import grad_destination
    got = []

    class Use(torch.autograd.Function):
        @staticmethod
        def forward(ctx, p, k):
            ctx.p, ctx.k = p, k
            return p.sum() * k

        @staticmethod
        def backward(ctx, g):
            d = grad_destination(ctx.p)
            got.append(d is not None)
            out = d if d is not None else torch.empty(3)
            return out.fill_(float(ctx.k)), None

    p = torch.nn.Parameter(torch.zeros(3))
    flat = torch.zeros(8)
    p._tn_grad_dest = flat[4:7]
    for _ in range(2):
        (Use.apply(p, 2) + Use.apply(p, 5)).backward()
        assert torch.equal(p.grad, torch.full((3,), 7.0))
        p.grad = None
    assert got == [True, False, True, False]


def test_cross_entropy_pieces_cover_the_classes(built):
    """A piece is a multiple of 256 classes and fits the budget where one tile
    does; there are at most five pieces more than the budget asks for."""
    from tiny_nccl_b200._native import load
    piece = load().ops.linear_ce_piece
    for rows in (1, 7, 200, 8192, 32768, 300000):
        for classes in (1, 255, 256, 257, 1000, 50257, 200000):
            for width in (8, 768, 4096):
                for budget in (1 << 12, 1 << 20, 512 << 20):
                    n = piece(rows, width, classes, budget)
                    tiles = (classes + 255) // 256
                    assert n > 0 and n % 256 == 0 and n <= tiles * 256
                    assert n == 256 or n * rows * 2 <= budget
                    most = max(1, budget // (rows * 512))
                    assert -(-tiles * 256 // n) <= -(-tiles // most) + 5
    assert piece(0, 768, 100, 1 << 20) == 0
