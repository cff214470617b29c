"""The training operators (embedding, linear cross-entropy, linear layers with
8-bit activations) against plain computations in 64 bits.

Tolerances count roundings: half a step is eps / 2 of a type relative to the
value (bf16 2^-8, fp32 2^-24).
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


def _half(dtype):
    return BF16 if dtype == torch.bfloat16 else F32


def _within(got, want, bound):
    """|got - want| <= bound, elementwise, everything in 64 bits."""
    over = (got.double() - want).abs() - bound
    assert bool((over <= 0).all()), (float(over.max()), int((over > 0).sum()))


def status_ok():
    from tiny_nccl_b200._native import load
    torch.cuda.synchronize()
    assert load().ops.tcgen05_status(True) == 0


# -- embedding ------------------------------------------------------------------


def _embedding_case(batch, seq, vocab, context, width, dtype, seed, positions, repeat):
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.randint(0, vocab, (batch, seq), device="cuda", generator=g)
    if repeat == "one":
        idx.fill_(vocab // 2)
    elif repeat == "few":
        idx %= 3
    idx[0, 0] = -1  # padding
    if idx.numel() > 2:
        idx.view(-1)[-1] = vocab  # past the table
    pos = torch.randint(0, context, (batch, seq), device="cuda", generator=g) if positions else None
    w = _normal(vocab, width, seed=seed + 1, dtype=dtype).requires_grad_()
    p = _normal(context, width, seed=seed + 2, dtype=dtype).requires_grad_()
    return idx, pos, w, p


def _embedding_sums(idx, gy, vocab, scale):
    """(table gradient, sum of magnitudes, tokens per row) in 64 bits."""
    idx, gy = idx.reshape(-1), gy.double().reshape(idx.numel(), -1)
    keep = (idx >= 0) & (idx < vocab)
    z = torch.zeros(vocab, gy.shape[1], dtype=torch.float64, device="cuda")
    total = z.clone().index_put_((idx[keep],), scale * gy[keep], accumulate=True)
    size = z.index_put_((idx[keep],), abs(scale) * gy[keep].abs(), accumulate=True)
    return total, size, torch.bincount(idx[keep], minlength=vocab).double()[:, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,seq,vocab,context,width,positions,repeat", [
    (1, 1, 7, 1, 1, False, ""),             # one token, one column
    (2, 3, 50, 9, 8, True, ""),
    (3, 337, 1009, 512, 250, False, ""),    # odd rows, a width of no vector size
    (8, 1, 50304, 1024, 768, True, ""),     # single tokens
    (4, 1024, 50304, 1024, 768, False, ""),
    (2, 999, 300, 1000, 77, True, "few"),   # three tokens share nearly all rows
    (5, 1024, 40, 1024, 132, False, "one"),  # one token has every row
    (33, 2048, 70000, 2048, 36, False, ""),  # many chunks of the sort
    (3, 700, 4200000, 700, 4, True, ""),     # 64-bit sort keys
    (17, 1024, 1050000, 1024, 4, False, "few"),
    (30, 1000, 2100000, 1000, 4, True, ""),  # chunks of 2048, one list's keys of 64 bits
    (101, 1000, 1050000, 1000, 4, True, "few"),  # chunks of 4096
    (101, 1000, 5000, 1000, 12, True, ""),
    (16, 4096, 11, 4096, 40, False, "one"),  # a run of thousands of blocks
])
def test_embedding(ops, dtype, batch, seq, vocab, context, width, positions, repeat):
    idx, pos, w, p = _embedding_case(batch, seq, vocab, context, width, dtype, 11, positions,
                                     repeat)
    scale = 3.25
    y = ops.embedding(idx, w, p, positions=pos, scale=scale)
    assert y.shape == (batch, seq, width) and y.dtype == dtype
    keep = ((idx >= 0) & (idx < vocab))[..., None]
    at = pos if pos is not None else torch.arange(seq, device="cuda").expand(batch, seq)
    token = torch.where(keep, scale * w.detach().double()[idx.clamp(0, vocab - 1)], 0.0)
    want = token + p.detach().double()[at]
    # fp32 product and sum, one rounding to the result's type.
    size = token.abs() + p.detach().double()[at].abs()
    _within(y, want, 2 * F32 * size + _half(dtype) * want.abs() * (1 + 4 * F32))
    gy = _normal(batch, seq, width, seed=12, dtype=dtype)
    dw, dp = torch.autograd.grad(y, [w, p], gy, retain_graph=True)
    for got, index, n, s in ((dw, idx, vocab, scale), (dp, at, context, 1.0)):
        total, size, count = _embedding_sums(index, gy, n, s)
        assert got.dtype == dtype
        # A chain of fp32 additions is off by at most half a step of the
        # partial sums, which the sum of magnitudes bounds; the scale is one
        # more rounding.
        _within(got, total, (count + 1) * F32 * size * (1 + 1e-3)
                + _half(dtype) * total.abs() * (1 + 1e-3))
    # The same bits every time.
    again = torch.autograd.grad(y, [w, p], gy)
    assert torch.equal(again[0], dw) and torch.equal(again[1], dp)


def test_embedding_runs_at_block_borders(ops):
    """Runs of equal tokens whose lengths put their ends at, before and after
    every multiple of 16 sorted rows, up to runs of more than 32 blocks."""
    lengths = torch.tensor([16, 16, 1, 15, 17, 31, 48, 16, 600, 8, 24, 512, 528, 1, 1, 14, 33],
                           device="cuda")
    idx = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), lengths)
    g = torch.Generator(device="cuda").manual_seed(1)
    for shift in range(17):
        # `shift` rows of token 0 more move every border.
        at = torch.cat([idx.new_zeros(shift), idx])
        at = at[torch.randperm(len(at), device="cuda", generator=g)]
        w = torch.zeros(len(lengths) + 1, 8, device="cuda", requires_grad=True)
        gy = torch.randint(-8, 9, (len(at), 8), device="cuda", generator=g).float()
        (dw,) = torch.autograd.grad(ops.embedding(at, w), [w], gy)
        want = torch.zeros_like(w).index_add_(0, at, gy)  # whole numbers: exact in any order
        assert torch.equal(dw, want)


def test_embedding_without_positions_and_mixed_types(ops):
    idx = torch.tensor([3, 0, 3], device="cuda", dtype=torch.int32)
    w = _normal(5, 12, seed=1, dtype=torch.bfloat16).requires_grad_()
    y = ops.embedding(idx, w, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and torch.equal(y, w.detach().float()[idx.long()])
    gy = _normal(3, 12, seed=2)
    (dw,) = torch.autograd.grad(y, [w], gy)
    want = torch.zeros(5, 12, device="cuda")
    want[0], want[3] = gy[1], gy[0] + gy[2]
    assert torch.equal(dw, want.to(torch.bfloat16))
    # A 0-d index and a transposed gradient.
    assert ops.embedding(idx[0], w).shape == (12,)
    y = ops.embedding(idx, w, out_dtype=torch.float32)
    (dt,) = torch.autograd.grad(y, [w], gy.t().contiguous().t())
    assert torch.equal(dt, dw)


def test_embedding_no_tokens(ops):
    w = _normal(6, 8, seed=1).requires_grad_()
    y = ops.embedding(torch.empty(0, 4, dtype=torch.int64, device="cuda"), w)
    assert y.shape == (0, 4, 8)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))


# -- linear cross-entropy ------------------------------------------------------


def _ce_case(rows, width, vocab, classes, seed, ignored=0.2):
    x = _normal(rows, width, seed=seed, dtype=torch.bfloat16)
    w = _normal(vocab, width, seed=seed + 1, std=2.0 / width ** 0.5, dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    target = torch.randint(0, classes, (rows,), device="cuda", generator=g)
    drop = torch.rand(rows, device="cuda", generator=g) < ignored
    return x, w, torch.where(drop, -100, target)


def _ce_exact(x, w, target, classes, k):
    """(losses, dx, dw, and the sums of magnitudes behind dx and dw) for the
    gradients k of the rows' losses, in 64 bits."""
    x, wf = x.double(), w.double()
    wc = wf[:classes]
    logits = x @ wc.t()
    lse = torch.logsumexp(logits, 1)
    counts = (target >= 0) & (target < classes)
    at = target.clamp(0, classes - 1)
    loss = torch.where(counts, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    d = torch.exp(logits - lse[:, None])
    d[torch.arange(len(x), device="cuda"), at] -= 1
    d = d * torch.where(counts, k.double(), 0.0)[:, None]
    dw, dws = torch.zeros_like(wf), torch.zeros_like(wf)
    dw[:classes] = d.t() @ x
    dws[:classes] = d.abs().t() @ x.abs()
    return loss, d @ wc, dw, d.abs() @ wc.abs(), dws


CE_SHAPES = [
    (1, 8, 1, 1),            # one row, one class: no loss at all
    (1, 64, 300, 300),
    (3, 72, 517, 510),       # neither width nor vocabulary a multiple of a tile
    (77, 256, 1024, 1000),
    (128, 64, 256, 256),
    (257, 200, 4099, 4099),
    (300, 768, 50304, 50257),
    (40, 64, 2000, 900),     # more padding than a tile
]


@pytest.mark.parametrize("rows,width,vocab,classes", CE_SHAPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy(ops, rows, width, vocab, classes, reduction):
    x, w, target = _ce_case(rows, width, vocab, classes, seed=rows + width)
    counts = max(1, int((target >= 0).sum()))
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(xr, wr, target, classes=classes, reduction=reduction)
    if reduction == "none":
        g = _normal(rows, seed=5)
        k = g
    else:
        g = torch.tensor(1.5, device="cuda")
        k = torch.full((rows,), 1.5 / (counts if reduction == "mean" else 1), device="cuda",
                       dtype=torch.float64)
    dx, dw = torch.autograd.grad(loss, [xr, wr], g)
    status_ok()
    each, ex, ew, sx, sw = _ce_exact(x, w, target, classes, k)
    # A logit sums `width` products in fp32 (the size of each is bounded by
    # |x| |w|): width * 2^-24 of that at the most, and the same for lse.
    logit = width * F32 * float((x.double().abs() @ w.double().abs().t()).max()) + 1e-6
    want = each if reduction == "none" else each.sum() / (counts if reduction == "mean" else 1)
    share = 1.0 if reduction == "none" else rows if reduction == "sum" else 1.0
    _within(loss, want, 2 * logit * share + 4 * F32 * want.abs() + rows * F32 * want.abs())
    # d is off by its rounding to bf16, by the logits' error and by that of
    # the exponential (2^-21); the products add in fp32.
    off = BF16 + 3 * logit + 2.0 ** -20
    _within(dx, ex, (off + 2 * vocab * F32) * sx + BF16 * ex.abs() * (1 + off) + 1e-30)
    _within(dw, ew, (off + 2 * rows * F32) * sw + BF16 * ew.abs() * (1 + off) + 1e-30)
    assert dw.dtype == torch.bfloat16 and bool((dw[classes:] == 0).all())


def test_linear_cross_entropy_mean_does_not_scale_the_gradient(ops):
    """1 / rows that count is no bf16 number; rounded into every entry of the
    logits' gradient it would scale all of dx and dw. Projected onto the exact
    gradient, the result's scale is right to a small part of a rounding: the
    entries' own roundings are independent, and average out over
    thousands of them."""
    rows = 1000  # 1 / 1000 is 0.43 of a bf16 step from its neighbour
    x, w, _ = _ce_case(rows, 128, 3000, 3000, seed=77)
    target = torch.randint(0, 3000, (rows,), device="cuda",
                           generator=torch.Generator(device="cuda").manual_seed(1))
    wr = w.float().requires_grad_()
    ops.linear_cross_entropy(x, wr, target).backward()
    k = torch.full((rows,), 1.0 / rows, device="cuda", dtype=torch.float64)
    _, _, ew, _, _ = _ce_exact(x, w, target, 3000, k)
    scale = (wr.grad.double() * ew).sum() / (ew * ew).sum()
    assert abs(float(scale) - 1) < BF16 / 8


def test_linear_cross_entropy_fp32_weight(ops):
    """An fp32 weight is used through its bf16 copy and gets an fp32
    gradient."""
    x, w, target = _ce_case(90, 128, 700, 700, seed=3)
    wr = w.float().requires_grad_()
    xr = x.float().requires_grad_()
    ops.linear_cross_entropy(xr.view(9, 10, 128), wr, target.view(9, 10)).backward()
    n = max(1, int((target >= 0).sum()))
    _, ex, ew, sx, sw = _ce_exact(x, w, target, 700, torch.full((90,), 1.0 / n, device="cuda"))
    assert wr.grad.dtype == torch.float32 and xr.grad.dtype == torch.float32
    _within(wr.grad, ew, (BF16 + 1e-3 * BF16 + 1e-5) * sw)
    _within(xr.grad, ex, (BF16 + 1e-5) * sx + BF16 * ex.abs() * 1.01)


@pytest.mark.parametrize("budget_tiles", [1, 3])
def test_linear_cross_entropy_pieces(ops, budget_tiles):
    """Many pieces of the vocabulary give dw bit for bit as one piece does (its
    rows belong to one piece each), and dx up to the fp32 sums' order."""
    from tiny_nccl_b200._native import load
    x, w, target = _ce_case(200, 136, 1500, 1437, seed=21)
    loss, lse, _, share = load().ops.linear_ce_fwd(x, w, target, 1437, 0)
    one = torch.ones(1, device="cuda")
    args = (x, w, target, lse, one, share, 1437, True, True, True, None)
    dx, dw = load().ops.linear_ce_bwd(*args, 512 << 20)
    px, pw = load().ops.linear_ce_bwd(*args, budget_tiles * 200 * 512)
    status_ok()
    assert load().ops.linear_ce_piece(200, 136, 1437, budget_tiles * 200 * 512) < 1437
    assert torch.equal(dw, pw)
    k = torch.full((200,), 1.0 / max(1, int((target >= 0).sum())), device="cuda")
    _, ex, _, sx, _ = _ce_exact(x, w, target, 1437, k)
    for got in (dx, px):
        _within(got, ex, (BF16 + 2e-5) * sx + BF16 * ex.abs() * 1.01)


def test_linear_cross_entropy_rows_that_do_not_count(ops):
    """All rows ignored: loss 0 and zero gradients; targets past the classes
    and any negative one are ignored; a row of NaN that does not count leaves
    the other rows' losses and gradients of x alone."""
    x, w, _ = _ce_case(40, 64, 500, 480, seed=4)
    for t in (-1, -100, 480, 10 ** 12):
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = ops.linear_cross_entropy(xr, wr, torch.full((40,), t, device="cuda"), classes=480)
        loss.backward()
        assert loss.item() == 0.0
        assert bool((xr.grad == 0).all()) and bool((wr.grad == 0).all())
    target = torch.arange(40, device="cuda")
    target[7] = -1
    bad = x.clone()
    bad[7] = float("nan")
    res = []
    for xi in (x, bad):
        xr = xi.clone().requires_grad_()
        loss = ops.linear_cross_entropy(xr, w, target, classes=480, reduction="none")
        loss.sum().backward()
        res.append((loss.detach(), xr.grad))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


def test_linear_cross_entropy_gradients_of_any_sign(ops):
    """reduction="none" with positive, negative, zero and very small gradients
    of the rows' losses."""
    x, w, target = _ce_case(64, 64, 300, 300, seed=14, ignored=0.1)
    g = _normal(64, seed=15)
    g[::4] = 0.0
    g[1::8] *= -1e-20
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(xr, wr, target, reduction="none")
    dx, dw = torch.autograd.grad(loss, [xr, wr], g)
    _, ex, ew, sx, sw = _ce_exact(x, w, target, 300, g)
    _within(dx, ex, (BF16 + 2e-5) * sx + BF16 * ex.abs() * 1.01)
    _within(dw, ew, (BF16 + 2e-5) * sw + BF16 * ew.abs() * 1.01 + 1e-30)
    assert bool((dx[::4] == 0).all())


def test_linear_cross_entropy_large_logits(ops):
    """Logits in the hundreds: the running maximum keeps every exponential
    finite."""
    x, w, target = _ce_case(50, 64, 900, 900, seed=6, ignored=0.0)
    x = (64 * x.float()).to(torch.bfloat16)
    xr = x.clone().requires_grad_()
    loss = ops.linear_cross_entropy(xr, w, target, reduction="none")
    loss.sum().backward()
    each, *_ = _ce_exact(x, w, target, 900, torch.ones(50, device="cuda"))
    logit = 64 * F32 * float((x.double().abs() @ w.double().abs().t()).max())
    _within(loss, each, 2 * logit + 1e-5 + 4 * F32 * each.abs())
    assert bool(torch.isfinite(xr.grad).all())


def test_linear_cross_entropy_no_rows(ops):
    w = _normal(40, 16, seed=1).requires_grad_()
    x = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    loss = ops.linear_cross_entropy(x, w, torch.empty(0, dtype=torch.int64, device="cuda"))
    loss.backward()
    assert loss.item() == 0.0 and bool((w.grad == 0).all()) and x.grad.shape == (0, 16)


def test_linear_cross_entropy_difference_quotient(ops):
    """The gradient against a central difference of the loss in 64 bits, along
    a random direction."""
    x, w, target = _ce_case(60, 64, 333, 333, seed=31)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    ops.linear_cross_entropy(xr, wr, target).backward()
    u, v = _normal(60, 64, seed=32).double(), _normal(333, 64, seed=33).double()
    n = int((target >= 0).sum())

    def f(h):
        logits = (x.double() + h * u) @ (w.double() + h * v).t()
        return torch.nn.functional.cross_entropy(logits, target, ignore_index=-100)

    h = 1e-5
    slope = (f(h) - f(-h)) / (2 * h)
    got = (xr.grad.double() * u).sum() + (wr.grad.double() * v).sum()
    _, ex, ew, sx, sw = _ce_exact(x, w, target, 333, torch.full((60,), 1.0 / n, device="cuda"))
    bound = ((2 * BF16 + 1e-4) * (sx * u.abs()).sum() + (2 * BF16 + 1e-4) * (sw * v.abs()).sum())
    assert abs(float(got - slope)) <= float(bound) + 1e-8


# -- 8-bit blocks ------------------------------------------------------------------


def _blocks64(x):
    """(values read back, steps) of the 8-bit blocks of x, in 64 bits."""
    rows, n = x.shape
    full = torch.nn.functional.pad(x.double(), (0, -n % 32)).view(rows, -1, 32)
    top = full.abs().amax(2, keepdim=True)
    e = (torch.frexp(top).exponent.long() - 8).clamp(min=-133)
    step = ((e + 1023) << 52).view(torch.float64)  # 2^e, exactly
    for _ in range(3):
        step = torch.where(torch.round(top / step) > 127, 2 * step, step)
    step = step.clamp(min=2.0 ** -133, max=2.0 ** 121)
    q = torch.round(full / step).clamp(-127, 127)
    return (q * step).view(rows, -1)[:, :n], step.expand_as(full).reshape(rows, -1)[:, :n]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (7, 33), (64, 768), (130, 1000),
                                       (2000, 264)])
def test_int8_blocks(ops, dtype, rows, cols):
    x = _normal(rows, cols, seed=cols, dtype=dtype)
    x[0, 0] = 127.5 / 64 * 2.0 ** 3  # rounds to 128 steps: the next exponent
    if rows > 4:
        x[1] = 0.0
        x[2] *= 2.0 ** 100
        x[3] *= 2.0 ** -120
        x[4] *= 2.0 ** -140 if dtype == torch.float32 else 2.0 ** -125
    q, e = ops.quantize_int8(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and e.shape == (rows, -(-cols // 32))
    want, step = _blocks64(x)
    back = ops.dequantize_int8(q, e, torch.float32)
    assert torch.equal(back.double(), want)
    assert torch.equal(ops.dequantize_int8(q, e).double(), want)  # bf16 holds every value
    assert bool(((back.double() - x.double()).abs() <= step / 2).all())


def test_int8_blocks_extremes(ops):
    """The largest bf16 numbers; blocks with NaN or infinity read back as NaN
    and leave their neighbours alone."""
    x = torch.zeros(4, 96, device="cuda", dtype=torch.bfloat16)
    x[0, :3] = torch.tensor([3.38e38, -3.38e38, 1e36])
    x[1, 40], x[2, 95], x[3, 0] = float("nan"), float("inf"), float("-inf")
    x[1, 0] = 5.0
    back = ops.dequantize_int8(*ops.quantize_int8(x), torch.float32)
    want, step = _blocks64(x.nan_to_num(0, 0, 0))
    assert torch.equal(back[0].double(), want[0])
    assert bool(back[1, 32:64].isnan().all()) and not bool(back[1, :32].isnan().any())
    assert back[1, 0] == 5.0
    assert bool(back[2, 64:].isnan().all()) and bool(back[3, :32].isnan().all())


# -- linear layers with 8-bit activations --------------------------------------------


def _gelu64(x):
    u = (2.0 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)
    return x / (1 + torch.exp(-2 * u))


def _gelu_slope64(x):
    x = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(_gelu64(x).sum(), [x])
    return g


LINEAR_SHAPES = [(1, 8, 8), (33, 128, 512), (130, 72, 264), (256, 256, 256), (1000, 768, 768),
                 (2049, 264, 1032), (6001, 520, 776)]  # the last: dW's sums are cut


@pytest.mark.parametrize("rows,ins,outs", LINEAR_SHAPES)
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_int8(ops, rows, ins, outs, gelu, dtype):
    x = _normal(rows, ins, seed=rows, dtype=torch.bfloat16).requires_grad_()
    w = _normal(outs, ins, seed=rows + 1, std=ins ** -0.5, dtype=torch.bfloat16)
    b = _normal(outs, seed=rows + 2, std=0.1, dtype=torch.bfloat16)
    gy = _normal(rows, outs, seed=rows + 3, dtype=torch.bfloat16)
    f = ops.linear_gelu if gelu else ops.linear
    wr, br = w.to(dtype).requires_grad_(), b.to(dtype).requires_grad_()
    y = f(x, wr, br, activations="int8")
    if not gelu:
        assert torch.equal(y, f(x, wr, br))  # the forward pass is the same
    dx, dw, db = torch.autograd.grad(y, [x, wr, br], gy)
    status_ok()
    assert dw.dtype == dtype and db.dtype == dtype
    x64, w64, g64 = x.detach().double(), w.double(), gy.double()
    off = torch.zeros((), dtype=torch.float64, device="cuda")
    if gelu:
        pre = x64 @ w64.t() + b.double()
        # The sum's fp32 error, a slope of at most 1.13, the GELU's own error
        # (ex2, reciprocal: 2^-20) and one rounding.
        sums = (ins + 1) * F32 * (x64.abs() @ w64.abs().t() + b.double().abs())
        gl = _gelu64(pre)
        _within(y, gl, 1.13 * sums + 2.0 ** -20 * pre.abs() + BF16 * gl.abs() * 1.01 + 1e-30)
        # The fp32 sum may fall on the other side of a border than the exact
        # one: a step of its block, or two where it moves the block's exponent;
        # the slope changes by at most 1.13 for a change of one.
        back, step = _blocks64(pre)
        g64 = g64 * _gelu_slope64(back)
        off = gy.double().abs() * 1.13 * 2 * step
    size = g64.abs()
    # g is rounded to bf16 after the GELU's slope; products add in fp32.
    g_off = off + (BF16 * size + 1e-5 * gy.double().abs() if gelu else 0)
    half = _half(dtype)
    xq, _ = _blocks64(x.detach())
    ex, ew, eb = g64 @ w64, g64.t() @ xq, g64.sum(0)
    _within(dx, ex, (g_off + outs * F32 * size) @ w64.abs() + BF16 * ex.abs() * 1.01 + 1e-30)
    _within(dw, ew, (g_off + rows * F32 * size).t() @ xq.abs() + half * ew.abs() * 1.01 + 1e-30)
    _within(db, eb, (g_off + rows * F32 * size).sum(0) + half * eb.abs() * 1.01 + 1e-30)


def test_linear_int8_needs_only_some_gradients(ops):
    x = _normal(40, 64, seed=1, dtype=torch.bfloat16)
    w = _normal(72, 64, seed=2).requires_grad_()
    b = _normal(72, seed=3).requires_grad_()
    gy = _normal(40, 72, seed=4, dtype=torch.bfloat16)
    both = ops.linear(x.clone().requires_grad_(), w, b, activations="int8")
    dw, db = torch.autograd.grad(both, [w, b], gy)
    alone = ops.linear(x, w, b, activations="int8")
    dw2, db2 = torch.autograd.grad(alone, [w, b], gy)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)


def test_linear_int8_no_rows(ops):
    w, b = _normal(24, 16, seed=1).requires_grad_(), _normal(24, seed=2).requires_grad_()
    for f in (ops.linear, ops.linear_gelu):
        x = torch.empty(2, 0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = f(x, w, b, activations="int8")
        assert y.shape == (2, 0, 24)
        dx, dw, db = torch.autograd.grad(y.sum(), [x, w, b])
        assert dx.shape == x.shape and not bool(dw.any()) and not bool(db.any())


def test_nothing_is_kept_without_a_gradient(ops):
    """Under no_grad, and for inputs that ask for no gradient, the results are
    the same bits and belong to no graph."""
    x = _normal(50, 64, seed=1, dtype=torch.bfloat16)
    w, b = _normal(128, 64, seed=2).requires_grad_(), _normal(128, seed=3).requires_grad_()
    t = torch.arange(50, device="cuda")
    calls = (lambda: ops.embedding(t, w, b.view(2, 64), positions=t % 2),
             lambda: ops.linear_cross_entropy(x, w, t),
             lambda: ops.linear_cross_entropy(x, w, t, reduction="none"),
             lambda: ops.linear(x, w, b, activations="int8"),
             lambda: ops.linear_gelu(x, w, b, activations="int8"))
    for f in calls:
        with_graph = f()
        with torch.no_grad():
            without = f()
        assert with_graph.requires_grad and not without.requires_grad
        assert torch.equal(with_graph, without)


# -- used together --------------------------------------------------------------------


def test_operators_together_train_step(ops):
    """Embedding, an MLP with 8-bit activations and the cross-entropy in
    pieces, forward and backward, captured in a CUDA graph: a replay on new
    tokens gives what the eager step gives on them, bit for bit."""
    V, C, R = 1000, 128, 192
    p = {k: _normal(*s, seed=i, std=0.05).requires_grad_() for i, (k, s) in enumerate(
        dict(wte=(1024, C), wpe=(64, C), w1=(4 * C, C), b1=(4 * C,), w2=(C, 4 * C),
             b2=(C,)).items())}
    leaves = list(p.values())

    def step(idx, target):
        h = ops.embedding(idx, p["wte"], p["wpe"], scale=C ** 0.5)
        m = ops.linear_gelu(h, p["w1"], p["b1"], activations="int8")
        m = ops.linear(m, p["w2"], p["b2"], activations="int8")
        loss = ops.linear_cross_entropy(h + m, p["wte"], target, classes=V)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    g = torch.Generator(device="cuda").manual_seed(9)
    data = torch.randint(0, V, (3, 2, 3, R // 3), device="cuda", generator=g)
    idx, target = data[0, 0].clone(), data[0, 1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(idx, target)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(idx, target)
    for i in (1, 2):
        idx.copy_(data[i, 0])
        target.copy_(data[i, 1])
        graph.replay()
        got = [t.clone() for t in out]
        want = step(data[i, 0], data[i, 1])
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    status_ok()


def test_tied_weight_in_a_flat_gradient_buffer(ops):
    """A weight that is both embedding and head, with its place in a flat
    gradient buffer: the head's gradient and the embedding's add up there, as
    without the buffer; a weight used once is written in place."""
    V, C, R = 700, 64, 90
    w = torch.nn.Parameter(_normal(V, C, seed=1, std=0.1))
    p = torch.nn.Parameter(_normal(R, C, seed=2, std=0.1))
    lw = torch.nn.Parameter(_normal(C, C, seed=3, std=0.1))
    lb = torch.nn.Parameter(torch.zeros(C, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(4)
    idx = torch.randint(0, V, (2, R), device="cuda", generator=g)
    leaves = [w, p, lw, lb]

    def backward():
        for t in leaves:
            t.grad = None
        h = ops.embedding(idx, w, p)
        h = ops.linear(h, lw, lb, activations="int8")
        ops.linear_cross_entropy(h, w, idx.roll(1, 1)).backward()
        return [t.grad.clone() for t in leaves]

    want = backward()
    flat = torch.zeros(sum(t.numel() for t in leaves), device="cuda")
    at = 0
    for t in leaves:
        t._tn_grad_dest = flat[at:at + t.numel()].view_as(t)
        at += t.numel()
    for _ in range(2):
        got = backward()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for t in (p, lw, lb):
            assert t.grad.data_ptr() == t._tn_grad_dest.data_ptr()


def test_strided_and_misaligned_inputs(ops):
    """Rows that are not contiguous, and storage that starts off a 16-byte
    boundary (copied or read one value at a time)."""
    w = _normal(50, 12, seed=1)
    base = torch.empty(50 * 12 + 1, device="cuda")
    off = base[1:].view(50, 12).copy_(w).requires_grad_()
    idx = torch.arange(40, device="cuda").view(4, 10)
    gy = _normal(4, 5, 12, seed=2)
    wr = w.clone().requires_grad_()
    y, z = ops.embedding(idx[:, ::2], off), ops.embedding(idx[:, ::2].contiguous(), wr)
    assert torch.equal(y, z)
    assert torch.equal(*(torch.autograd.grad(a, [b], gy)[0] for a, b in ((y, off), (z, wr))))
    x = _normal(64, 128, seed=3, dtype=torch.bfloat16)
    hw = _normal(100, 64, seed=4, dtype=torch.bfloat16)
    t = torch.arange(64, device="cuda")
    a = ops.linear_cross_entropy(x[:, ::2], hw, t)
    b = ops.linear_cross_entropy(x[:, ::2].contiguous(), hw, t)
    assert torch.equal(a, b)
    assert torch.equal(ops.quantize_int8(x.t())[0], ops.quantize_int8(x.t().contiguous())[0])


def test_misaligned_gradients_and_parameters(ops):
    """A gradient, an input and parameters that start off a 16-byte boundary
    give the bits of aligned ones."""
    def off(t):  # the same values, one element past a boundary
        base = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        return base[1:].view(t.shape).copy_(t)
    x = _normal(40, 64, seed=1, dtype=torch.bfloat16)
    w, b = _normal(48, 64, seed=2, dtype=torch.bfloat16), _normal(48, seed=3, dtype=torch.bfloat16)
    t = torch.arange(40, device="cuda")
    flat = torch.cat([torch.zeros(3, device="cuda"), _normal(40 * 48, seed=4)])
    gy = flat[3:].view(40, 48).to(torch.bfloat16)
    for f in (lambda *a: ops.linear(*a, activations="int8"),
              lambda *a: ops.linear_gelu(*a, activations="int8"),
              lambda x, w, b: ops.linear_cross_entropy(x, w, t, reduction="none")):
        out = []
        for move in (lambda v: v, off):
            leaves = [move(v).requires_grad_() for v in (x, w, b)]
            y = f(*leaves)
            # The gradient that arrives is a view of the joined tensor's.
            joined = torch.cat([torch.zeros(3 if move is off else 0, device="cuda", dtype=y.dtype),
                                y.flatten()])
            g = flat.to(joined.dtype)[3 if move is not off else 0:][:joined.numel()]
            out.append([y, *torch.autograd.grad(joined, leaves, g, allow_unused=True)])
        for a, c in zip(*out):
            assert (a is None and c is None) or torch.equal(a, c)
    status_ok()


def test_loss_may_be_changed_in_place(ops):
    x = _normal(40, 64, seed=1, dtype=torch.bfloat16).requires_grad_()
    w = _normal(100, 64, seed=2).requires_grad_()
    t = torch.arange(40, device="cuda")
    for reduction in ("mean", "sum"):
        want = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction=reduction) * 0.5,
                                   [x, w])
        loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
        loss.mul_(0.5)
        for a, b in zip(torch.autograd.grad(loss, [x, w]), want):
            assert torch.equal(a, b)


def test_linear_gelu_int8_far_from_zero(ops):
    """Sums of any size: the GELU is 0 or its argument, the slope 0 or 1, and a
    sum that is no number gives none."""
    values = [20.0, -20.0, 1e12, -1e12, 1e20, -1e20, 3e38, -3e38]
    b = torch.tensor(values, device="cuda").repeat_interleave(32).to(torch.bfloat16)
    x = torch.zeros(5, 64, device="cuda", dtype=torch.bfloat16)
    w = _normal(256, 64, seed=1)
    b.requires_grad_()
    y = ops.linear_gelu(x, w, b, activations="int8")
    gy = _normal(5, 256, seed=2, dtype=torch.bfloat16)
    (db,) = torch.autograd.grad(y, [b], gy)
    up = b.detach() > 0
    assert torch.equal(y[:, up], b.detach()[up].expand(5, -1))
    assert bool((y[:, ~up].abs() <= 1e-30).all())
    g64 = gy.double()
    _within(db[up], g64.sum(0)[up], BF16 * g64.sum(0)[up].abs() * 1.01
            + 5 * F32 * g64.abs().sum(0)[up])
    assert bool((db[~up].abs() <= 1e-25).all())
    with torch.no_grad():
        b[40] = float("nan")
    y = ops.linear_gelu(x, w, b, activations="int8")
    (db,) = torch.autograd.grad(y, [b], gy)
    assert bool(y[:, 40].isnan().all()) and not bool(y[:, :40].isnan().any())
    # 8-bit blocks lose a number's neighbours with it, and no others.
    assert bool(db[32:64].isnan().all()) and not bool(db[:32].isnan().any())
    assert not bool(db[64:].isnan().any())


def test_refuses_to_be_differentiated_twice(ops):
    w = _normal(20, 16, seed=1).requires_grad_()
    y = ops.embedding(torch.arange(4, device="cuda"), w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), [w], create_graph=True)


# -- refusals -----------------------------------------------------------------------


def test_refusals(ops):
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(16, 64, device="cuda")
    b = torch.zeros(16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    odd = torch.zeros(16, 63, device="cuda")
    with pytest.raises(RuntimeError):  # width % 8
        ops.linear_cross_entropy(x[:, :63], odd, t)
    with pytest.raises(RuntimeError):
        ops.linear_cross_entropy(x, w, t, classes=17)
    with pytest.raises(RuntimeError):
        ops.linear_cross_entropy(x, w, t.cpu())
    with pytest.raises(RuntimeError):
        ops.embedding(t, w.cpu())
    with pytest.raises(RuntimeError):
        ops.embedding(t.cpu(), w)
    with pytest.raises(RuntimeError):
        ops.linear(x[:, :60], w[:, :60].contiguous().requires_grad_(), b,
                   activations="int8").sum().backward()
