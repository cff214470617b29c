"""The training operators at their edges: values that are no number, logits of
hundreds, forward-mode differentiation, parameters that are frozen, very many
rows, and the 8-bit sums of the fused GELU bit by bit.

As in test_train_ops_gpu.py, tolerances count roundings: half a step is eps / 2
of a type relative to the value (bf16 2^-8, fp32 2^-24).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(scope="module")
def ops(built):
    import tiny_nccl_b200.ops as o
    return o


def _normal(*shape, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


# -- cross-entropy: values that are no number ---------------------------------------


@pytest.mark.parametrize("first,count,classes", [
    (0, 32, 300),     # a whole block of 32 classes, the first of its 128
    (128, 32, 300),
    (128, 128, 400),  # all 128
    (128, 1, 129),    # the only class of its block
    (256, 1, 257),    # ... and of its tile
    (5, 1, 300),
    (32, 32, 300),
])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_nan_logits_reach_the_loss(ops, first, count, classes, reduction):
    """A class whose logits are NaN makes every loss that counts NaN, wherever
    the class stands; a row that does not count stays 0."""
    x, w = _normal(20, 64, seed=1, dtype=torch.bfloat16), _normal(classes, 64, seed=2, std=0.2)
    w[first:first + count] = float("nan")
    target = torch.full((20,), 100, device="cuda")  # a class that is a number
    target[3] = -100
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, target, reduction=reduction)
    if reduction == "mean":
        assert bool(loss.isnan())
    else:
        counts = target >= 0
        assert bool(loss[counts].isnan().all()) and bool((loss[~counts] == 0).all())


@pytest.mark.parametrize("first,count,classes", [(0, 32, 300), (128, 128, 400), (256, 1, 257),
                                                 (0, 299, 300)])
def test_classes_at_minus_infinity_are_absent(ops, first, count, classes):
    """Logits of -inf add nothing: the losses are those of the other classes,
    bit for bit where their blocks are the same."""
    x, w = _normal(20, 64, seed=1, dtype=torch.bfloat16), _normal(classes, 64, seed=2, std=0.2)
    x[:, 0] = 1.0
    w[first:first + count, 0] = float("-inf")
    keep = torch.ones(classes, dtype=torch.bool, device="cuda")
    keep[first:first + count] = False
    target = torch.full((20,), int(keep.nonzero()[-1]), device="cuda")
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, target, reduction="none")
    logits = x.double() @ w[keep].to(torch.bfloat16).double().t()
    want = torch.logsumexp(logits, 1) - logits[:, int(keep[:target[0]].sum())]
    # 64 fp32 products and sums a logit, ex2's and the sums' 2^-20.
    size = x.double().abs() @ w[keep].to(torch.bfloat16).double().abs().t()
    off = 2 * 65 * F32 * size.amax(1) + 2.0 ** -20 + 4 * F32 * logits.abs().amax(1)
    assert bool(((loss.double() - want).abs() <= off).all())


# -- cross-entropy: rows that are sure ------------------------------------------------


@pytest.mark.parametrize("at", [0, 31, 32, 127, 130, 299])
def test_sure_rows_have_no_loss_and_no_gradient(ops, at):
    """Logits in the hundreds that fp32 holds exactly, the target's above all
    others by more than exp's range: the softmax is exactly the target's, so
    that loss and gradients are exactly 0, not a rounding of the logits (lse's
    half step is 3e-5 at 1000)."""
    a = torch.arange(129, 256, 2, device="cuda")  # bf16 holds whole numbers to 256
    x = torch.zeros(len(a), 64, device="cuda")
    x[:, 0] = a
    w = torch.zeros(300, 64, device="cuda")
    w[:, 0] = 1.0
    w[at, 0] = 4.0  # the target's logit is 4 a, the others' are a
    w[:, 1:] = _normal(300, 63, seed=1)  # seen by no row, but by dx
    xr, wr = x.requires_grad_(), w.requires_grad_()
    target = torch.full((len(a),), at, device="cuda")
    loss = ops.linear_cross_entropy(xr, wr, target, reduction="none")
    dx, dw = torch.autograd.grad(loss, [xr, wr], torch.ones_like(loss))
    assert bool((loss == 0).all()), loss
    assert not bool(dx.any()) and not bool(dw.any())


def test_loss_is_never_negative(ops):
    """lse is at least the target's logit, in the kernel's arithmetic too."""
    x = _normal(512, 64, seed=3, std=40.0, dtype=torch.bfloat16)
    w = _normal(700, 64, seed=4, dtype=torch.bfloat16)
    target = (x.double() @ w.double().t()).argmax(1)
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, target, reduction="none")
    assert bool((loss >= 0).all()), float(loss.min())


# -- what is asked for ------------------------------------------------------------------


def _small_calls(ops):
    """(call, its differentiable inputs) for each operator, small."""
    idx = torch.arange(6, device="cuda")
    w, p = _normal(10, 64, seed=1), _normal(8, 64, seed=2)
    x, b = _normal(6, 64, seed=3), _normal(24, seed=4)
    x16, lw = x.to(torch.bfloat16), _normal(24, 64, seed=5)
    return [(lambda w, p: ops.embedding(idx, w, p), (w, p)),
            (lambda x, w: ops.linear_cross_entropy(x, w, idx), (x, w)),
            (lambda x, w: ops.linear_cross_entropy(x, w, idx, reduction="none"), (x16, w)),
            (lambda x, w, b: ops.linear(x, w, b, activations="int8"), (x, lw, b)),
            (lambda x, w, b: ops.linear_gelu(x, w, b, activations="int8"), (x16, lw, b))]


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(ops, grad):
    """A dual tensor among the inputs raises, as it does in every other
    autograd function here: the result would come back without its tangent."""
    from torch.autograd import forward_ad
    for call, inputs in _small_calls(ops):
        for i, t in enumerate(inputs):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError):
                    call(*inputs[:i], dual, *inputs[i + 1:])
        with torch.no_grad():
            call(*inputs)


def _peak(call):
    """Bytes that a call has on the device at once, beyond what it found."""
    call()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("rows,ins,outs", [(300, 72, 264), (2048, 256, 1024)])
def test_gelu_keeps_no_8_bit_sums_without_a_gradient(ops, rows, ins, outs):
    """Inference forms the activations alone, the same bits."""
    x = _normal(rows, ins, seed=1, dtype=torch.bfloat16)
    w = _normal(outs, ins, seed=2, dtype=torch.bfloat16)
    b = _normal(outs, seed=3, dtype=torch.bfloat16)
    want = ops.linear_gelu(x, w.clone().requires_grad_(), b, activations="int8").detach()
    with torch.no_grad():
        assert torch.equal(ops.linear_gelu(x, w, b, activations="int8"), want)
        peak = _peak(lambda: ops.linear_gelu(x, w, b, activations="int8"))
    # The activations in bf16, and less than the byte for each of them that the
    # 8-bit sums would take.
    assert 2 * rows * outs <= peak < 2 * rows * outs + rows * outs // 2


def _launches(ops, call):
    before = ops.launch_count()
    out = call()
    return ops.launch_count() - before, out


def test_frozen_weight_keeps_no_inputs(ops):
    """Only the weight's gradient reads the inputs: a frozen weight (the rest
    trained) forms no 8-bit copy of them, and the other gradients are the same."""
    x = _normal(300, 128, seed=1, dtype=torch.bfloat16)
    w, b = _normal(264, 128, seed=2), _normal(264, seed=3).requires_grad_()
    gy = _normal(300, 264, seed=4, dtype=torch.bfloat16)
    for f in (ops.linear, ops.linear_gelu):
        launches, res = [], []
        for frozen in (False, True):
            xr = x.clone().requires_grad_()
            wr = w.clone().requires_grad_(not frozen)
            n, y = _launches(ops, lambda: f(xr, wr, b, activations="int8"))
            launches.append(n)
            res.append((y.detach(), *torch.autograd.grad(y, [xr, b], gy)))
        assert launches[1] == launches[0] - 1  # the quantizing kernel
        for one, other in zip(*res):
            assert torch.equal(one, other)


def test_frozen_bias_is_not_summed(ops):
    """A frozen bias: no column sums behind the GELU's gradient, the other
    gradients the same."""
    rows, outs = 2000, 264
    x = _normal(rows, 128, seed=1, dtype=torch.bfloat16)
    w, b = _normal(outs, 128, seed=2).requires_grad_(), _normal(outs, seed=3)
    gy = _normal(rows, outs, seed=4, dtype=torch.bfloat16)
    launches, res = [], []
    for frozen in (False, True):
        xr, br = x.clone().requires_grad_(), b.clone().requires_grad_(not frozen)
        y = ops.linear_gelu(xr, w, br, activations="int8")
        n, d = _launches(ops, lambda: torch.autograd.grad(y, [xr, w], gy, retain_graph=True))
        launches.append(n)
        res.append(d)
        if not frozen:
            n, d = _launches(ops, lambda: torch.autograd.grad(y, [xr, w, br], gy))
            launches.append(n)
    # Asked for or not makes the difference, not whether the bias is frozen.
    assert launches[0] == launches[2] == launches[1] - 1, launches
    for one, other in zip(*res):
        assert torch.equal(one, other)


# -- embedding: very many rows ------------------------------------------------------------


def _embedding_grad_ms(ops, rows):
    g = torch.Generator(device="cuda").manual_seed(1)
    idx = torch.randint(0, 50000, (rows,), device="cuda", generator=g)
    w = torch.zeros(50000, 4, device="cuda", requires_grad=True)
    gy = torch.ones(rows, 4, device="cuda")
    y = ops.embedding(idx, w)
    times = []
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        torch.autograd.grad(y, [w], gy, retain_graph=True)
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


def test_embedding_gradient_grows_with_the_rows(ops):
    """Eight times the rows take about eight times as long (twice that is
    allowed), where searching every chunk for every row would take 64 times."""
    assert _embedding_grad_ms(ops, 1 << 22) < 16 * _embedding_grad_ms(ops, 1 << 19)


@pytest.mark.parametrize("rows,vocab", [
    (1 << 17, 1000),             # as many chunks as are merged at once
    ((1 << 17) + 1, 1000),       # ... and one row
    ((1 << 18) + 4097, 50000),
    (3 * (1 << 17), 7),          # an odd number of sorted parts
    (1300001, 2100000),          # 64-bit sort keys
    (1300001, 1),                # one run
])
def test_embedding_of_very_many_rows(ops, rows, vocab):
    g = torch.Generator(device="cuda").manual_seed(rows)
    idx = torch.randint(-1, vocab + 1, (rows,), device="cuda", generator=g)
    at = torch.randint(0, 300, (rows,), device="cuda", generator=g)
    w = torch.zeros(vocab, 3, device="cuda", requires_grad=True)
    p = torch.zeros(300, 3, device="cuda", requires_grad=True)
    gy = torch.randint(-2, 3, (rows, 3), device="cuda", generator=g).float()
    dw, dp = torch.autograd.grad(ops.embedding(idx, w, p, positions=at), [w, p], gy)
    # Whole numbers whose sums stay below 2^24: exact in any order.
    keep = (idx >= 0) & (idx < vocab)
    assert torch.equal(dw, torch.zeros_like(w).index_add_(0, idx[keep], gy[keep]))
    assert torch.equal(dp, torch.zeros_like(p).index_add_(0, at, gy))


def test_embedding_of_very_many_rows_adds_in_row_order(ops):
    """The order of equal tokens is the rows': a run's first block is added in
    fp32 in that order, so that a sum of values far apart shows any other."""
    rows = (1 << 17) + 30000
    g = torch.Generator(device="cuda").manual_seed(5)
    idx = torch.randperm(rows // 16 * 16, device="cuda", generator=g) // 16
    vocab = int(idx.max()) + 1
    gy = _normal(len(idx), 4, seed=6) * 10.0 ** torch.randint(-4, 5, (len(idx), 1), device="cuda",
                                                               generator=g)
    w = torch.zeros(vocab, 4, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(ops.embedding(idx, w), [w], gy)
    by_token = gy[torch.sort(idx, stable=True)[1]].view(vocab, 16, 4)
    want = torch.zeros(vocab, 4, device="cuda")
    for i in range(16):  # sixteen rows each: every run lies within its block
        want += by_token[:, i]
    assert torch.equal(dw, want)


# -- the fused GELU's 8-bit sums, bit by bit ------------------------------------------------


def _int8_exponent(top):
    """The exponent byte of a block whose largest magnitude is top: the least
    e >= 0 with round(top / 2^(e - 133)) <= 127, in 64 bits."""
    e = (torch.frexp(top).exponent.long() - 9 + 133).clamp(min=0) * (top > 0)
    for _ in range(4):
        e = torch.where(torch.round(top / _step64(e)) > 127, e + 1, e)
    return e


def _step64(e):
    return ((e - 133 + 1023) << 52).view(torch.float64)  # 2^(e - 133), exactly


def _gelu_slope64(x):
    k0, k1 = (2.0 / torch.pi) ** 0.5, 0.044715
    r = 1 / (1 + torch.exp(-2 * k0 * (x + k1 * x ** 3)))
    return r + 2 * x * r * (1 - r) * k0 * (1 + 3 * k1 * x ** 2)


def _off_by(q, lo, hi):
    return int(((q < lo) | (q > hi)).sum())


GELU_SHAPES = [(1, 8, 8), (33, 128, 512), (130, 72, 264), (300, 520, 136), (70, 64, 40),
               (257, 1600, 1032), (1000, 200, 776)]


@pytest.mark.parametrize("rows,ins,outs", GELU_SHAPES)
def test_gelu_int8_sums_bit_by_bit(ops, rows, ins, outs):
    """q and e of the sums before the GELU: the fp32 sum is off by at most
    (ins + 1) half steps of its magnitudes' sum, and between the whole numbers
    that both ends of that range round to nothing is allowed. Then the gradients
    from these q and e, whose only roundings are the GELU gradient's to bf16 and
    the results'."""
    from tiny_nccl_b200._native import load
    x = _normal(rows, ins, seed=rows, dtype=torch.bfloat16)
    w = _normal(outs, ins, seed=rows + 1, std=ins ** -0.5, dtype=torch.bfloat16)
    b = _normal(outs, seed=rows + 2, std=0.1, dtype=torch.bfloat16)
    # Blocks of every size, and one of zeros.
    w *= (2.0 ** (torch.arange(outs, device="cuda") // 32 % 40 - 20))[:, None].to(torch.bfloat16)
    w[:32] = 0.0
    b[:32] = 0.0
    act, q, e = load().ops.linear_gelu_int8(x, w, b)
    x64, w64, b64 = x.double(), w.double(), b.double()
    pre = x64 @ w64.t() + b64
    err = (ins + 1) * F32 * (x64.abs() @ w64.abs().t() + b64.abs())
    pad = -outs % 32
    block = lambda t: torch.nn.functional.pad(t, (0, pad)).view(rows, -1, 32)  # noqa: E731
    size, eb = block(pre.abs()), block(err)
    lo = _int8_exponent((size - eb).clamp(min=0).amax(2))
    hi = _int8_exponent((size + eb).amax(2))
    assert _off_by(e.long(), lo, hi) == 0
    step = _step64(e.long()).repeat_interleave(32, 1)[:, :outs]
    qlo, qhi = (torch.round(t / step).clamp(-127, 127) for t in (pre - err, pre + err))
    assert _off_by(q.double(), qlo, qhi) == 0
    # Most values leave no choice. Where the weights are small a sum is its bf16
    # bias and a little: with eight significant bits against q's seven, half of
    # the values in a block's top binade lie next to a tie; elsewhere the range
    # is 2 (ins + 1) 2^-24 0.64 sqrt(ins) of a value near 1, a sixth of the step
    # 2^-5 at 1600 inputs.
    assert float((qlo == qhi).double().mean()) > 0.5
    back = q.double() * step
    assert torch.equal(load().ops.dequantize_int8(q, e, True).double(), back)

    xr, wr, br = x.clone().requires_grad_(), w.float().requires_grad_(), b.float().requires_grad_()
    y = ops.linear_gelu(xr, wr, br, activations="int8")
    assert torch.equal(y, act)
    gy = _normal(rows, outs, seed=rows + 3, dtype=torch.bfloat16)
    dx, dw, db = torch.autograd.grad(y, [xr, wr, br], gy)
    g = gy.double() * _gelu_slope64(back)
    # The slope: ex2, a reciprocal and fp32 products, 2^-20 of at most 1.13; g's
    # bf16 rounding, then fp32 sums, then the result's rounding (dx bf16).
    slope = 2.0 ** -20 * gy.double().abs()
    each = BF16 * g.abs() + slope * (1 + BF16)
    xq = load().ops.dequantize_int8(*ops.quantize_int8(x), True).double()
    ex, ew, es = g @ w64, g.t() @ xq, g.sum(0)
    off = (each + (outs + 2) * F32 * g.abs()) @ w64.abs() + BF16 * ex.abs() * 1.01 + 1e-30
    assert bool(((dx.double() - ex).abs() <= off).all())
    off = (each + (rows + 2) * F32 * g.abs()).t() @ xq.abs() + 1e-30
    assert bool(((dw.double() - ew).abs() <= off).all())
    off = (slope + (rows + 2) * F32 * g.abs()).sum(0) + 1e-30
    assert bool(((db.double() - es).abs() <= off).all())


@pytest.mark.parametrize("classes,vocab", [(480, 500), (480, 1000), (700, 704), (1000, 1001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_rows_get_zero_whatever_x_holds(ops, classes, vocab, dtype):
    """The rows of weight behind the classes have a zero gradient also where
    a row of x is no number."""
    x = _normal(600, 64, seed=1, dtype=torch.bfloat16)
    x[5, 3], x[7, 0] = float("nan"), float("inf")
    w = _normal(vocab, 64, seed=2, dtype=dtype).requires_grad_()
    target = torch.arange(600, device="cuda") % classes
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, target, classes=classes), [w])
    assert bool((dw[classes:] == 0).all())
    assert bool(dw[:classes].isnan().any())


def test_int8_blocks_without_values(ops):
    for shape in [(5, 0), (0, 40), (0, 0), (3, 0, 64), (3, 2, 0)]:
        x = torch.empty(shape, device="cuda")
        q, e = ops.quantize_int8(x)
        assert q.shape == shape and e.shape == (*shape[:-1], -(-shape[-1] // 32))
        assert ops.dequantize_int8(q, e).shape == shape


def test_binding_refuses_sizes_that_do_not_match(ops):
    """What the backward pass of the cross-entropy reads has the sizes of its
    forward pass."""
    from tiny_nccl_b200._native import load
    x = _normal(40, 64, seed=1, dtype=torch.bfloat16)
    w = _normal(300, 64, seed=2, dtype=torch.bfloat16)
    target = torch.arange(40, device="cuda")
    _, lse, _, share = load().ops.linear_ce_fwd(x, w, target, 300, 0)
    one = torch.ones(1, device="cuda")
    good = dict(x=x, weight=w, target=target, lse=lse, grad=one, share=share, classes=300,
                want_dx=True, want_dw=True, dw_f32=True)
    load().ops.linear_ce_bwd(**good)
    for bad in (dict(lse=lse[:39]), dict(lse=lse.cpu()), dict(grad=torch.ones(39, device="cuda")),
                dict(grad=one.cpu()), dict(share=torch.empty(0, device="cuda")),
                dict(share=share.cpu()), dict(target=target[:39]),
                dict(dw_out=torch.empty(299, 64, device="cuda"))):
        with pytest.raises(RuntimeError):
            load().ops.linear_ce_bwd(**{**good, **bad})


def test_int8_blocks_bound(ops):
    """Half a step is at most 1 / 127.5 of a block's largest magnitude, reached
    where 127.5 steps become 63.75; 2^-7 does not hold there."""
    x = torch.zeros(2, 32, device="cuda")
    x[0, 0], x[0, 1] = 127.5 / 64, 1 / 64   # 63.75 steps of 2^-5, and half a step
    x[1, 0], x[1, 1] = 127.0 / 64, 1 / 128  # 127 steps of 2^-6, and half a step
    back = ops.dequantize_int8(*ops.quantize_int8(x), torch.float32)
    off = (back.double() - x.double()).abs().amax(1) / x.double().amax(1)
    assert off[0] == 1 / 127.5 and off[0] > 2.0 ** -7 > off[1]
    for seed in range(4):
        scale = 2.0 ** (torch.arange(500, device="cuda")[:, None] % 60 - 30)
        x = _normal(500, 96, seed=seed) * scale
        back = ops.dequantize_int8(*ops.quantize_int8(x), torch.float32)
        top = x.double().view(500, 3, 32).abs().amax(2).repeat_interleave(32, 1)
        assert bool(((back.double() - x.double()).abs() <= top / 127.5).all())


# -- sizes past the tiles ------------------------------------------------------------------


def _blocks64(x):
    """x as its 8-bit blocks hold it, in 64 bits."""
    pad = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).view(len(x), -1, 32)
    step = _step64(_int8_exponent(pad.abs().amax(2)))[..., None]
    return (torch.round(pad / step).clamp(-127, 127) * step).view(len(x), -1)[:, :x.shape[1]]


@pytest.mark.parametrize("rows,ins,outs", [
    (300, 1600, 2560),   # as wide as a layer is timed
    (700, 4096, 1024),   # 64 K blocks
    (2048, 768, 2304),   # few tiles for the SM pairs
    (9001, 776, 264),    # 141 K blocks of dW in few tiles: its sums are cut
])
def test_linear_int8_wide(ops, rows, ins, outs):
    x = _normal(rows, ins, seed=1, dtype=torch.bfloat16).requires_grad_()
    w = _normal(outs, ins, seed=2, std=ins ** -0.5).requires_grad_()
    b = _normal(outs, seed=3, std=0.1).requires_grad_()
    gy = _normal(rows, outs, seed=4, dtype=torch.bfloat16)
    y = ops.linear(x, w, b, activations="int8")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], gy)
    x64, w64, g64 = x.detach().double(), w.detach().to(torch.bfloat16).double(), gy.double()
    xq = _blocks64(x.detach())
    size = x64.abs() @ w64.abs().t() + 1.0
    b64 = b.detach().to(torch.bfloat16).double()
    # fp32 sums of exact products, then the results' rounding.
    for got, want, off in ((y.detach(), x64 @ w64.t() + b64, (ins + 1) * F32 * size),
                           (dx, g64 @ w64, outs * F32 * (g64.abs() @ w64.abs())),
                           (dw, g64.t() @ xq, rows * F32 * (g64.abs().t() @ xq.abs())),
                           (db, g64.sum(0), rows * F32 * g64.abs().sum(0))):
        half = BF16 if got.dtype == torch.bfloat16 else F32
        assert bool(((got.double() - want).abs() <= off + half * 1.01 * want.abs()).all())


@pytest.mark.parametrize("rows,width,classes,vocab", [
    (300, 1600, 2000, 2048),    # a wide head
    (20001, 128, 20000, 20000),  # the logits' gradient in several pieces by the rule itself
])
def test_linear_cross_entropy_wide(ops, rows, width, classes, vocab):
    from tiny_nccl_b200._native import load
    if rows > 10000:
        assert load().ops.linear_ce_piece(rows, width, classes, 512 << 20) < classes
    x = _normal(rows, width, seed=1, dtype=torch.bfloat16)
    w = _normal(vocab, width, seed=2, std=2.0 * width ** -0.5)
    target = torch.arange(rows, device="cuda") * 7919 % classes
    target[::9] = -1
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(xr, wr, target, classes=classes)
    dx, dw = torch.autograd.grad(loss, [xr, wr])
    wc = w.to(torch.bfloat16).double()[:classes]
    keep = target >= 0
    total = 0.0
    ew, sw = torch.zeros_like(wc), torch.zeros_like(wc)
    n = int(keep.sum())
    # A logit's fp32 sum: `width` half steps of its magnitudes; the exponential
    # and the sums 2^-20; d's rounding to bf16.
    logit = 0.0
    for at in range(0, rows, 4096):
        xs, t, k = x[at:at + 4096].double(), target[at:at + 4096].clamp(min=0), keep[at:at + 4096]
        logit = max(logit, width * F32 * float((xs.abs() @ wc.abs().t()).max()))
        logits = xs @ wc.t()
        lse = torch.logsumexp(logits, 1)
        i = torch.arange(len(t), device="cuda")
        total += float((lse - logits[i, t])[k].sum())
        d = torch.exp(logits - lse[:, None])
        d[i, t] -= 1
        d *= k[:, None] / n
        ew += d.t() @ xs
        sw += d.abs().t() @ xs.abs()
        off = BF16 + 3 * logit + 2.0 ** -20 + 2 * classes * F32
        ex, sx = d @ wc, d.abs() @ wc.abs()
        got = dx[at:at + 4096].double()
        assert bool(((got - ex).abs() <= off * sx + 1.01 * BF16 * ex.abs()).all())
    off = BF16 + 3 * logit + 2.0 ** -20 + 2 * rows * F32
    assert bool(((dw[:classes].double() - ew).abs() <= off * sw + 1.01 * F32 * ew.abs()).all())
    assert not bool(dw[classes:].any())
    assert abs(loss.item() - total / n) <= 2 * logit + 2.0 ** -20 + (rows + 4) * F32 * total / n


@pytest.mark.parametrize("dtype", [torch.float64, torch.float16])
def test_linear_int8_gradients_of_other_types(ops, dtype):
    """Parameters of other types are used through bf16 copies, as in the default
    linear layers; their gradients come from fp32 sums, not from bf16 results."""
    x = _normal(300, 128, seed=1, dtype=torch.bfloat16)
    w = _normal(264, 128, seed=2, dtype=torch.bfloat16)
    b = _normal(264, seed=3, dtype=torch.bfloat16)
    gy = _normal(300, 264, seed=4, dtype=torch.bfloat16)
    for f in (ops.linear, ops.linear_gelu):
        res = []
        for t in (torch.float32, dtype):
            wt, bt = w.to(t).requires_grad_(), b.to(t).requires_grad_()
            res.append(torch.autograd.grad(f(x, wt, bt, activations="int8"), [wt, bt], gy))
        for fp32, other in zip(*res):
            assert other.dtype == dtype and torch.equal(fp32.to(dtype), other)
