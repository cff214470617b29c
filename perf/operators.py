"""Cases of the training operators: the embedding with its gradient by sorted
tokens, the linear layer + softmax cross-entropy in pieces of the vocabulary,
and the linear layers that keep their activations in 8 bits for the backward
pass. Each case runs in a plain form (elementary torch operations in fp32) or,
with ``own``, through this package's operators.

Parameters are bf16 where an operator multiplies matrices (the bf16 copies
that the fused linear layers work on), so that both forms start from the same
values and every gradient has the type of what it belongs to.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # One decoding step of a small batch: eight tokens at positions of
        # their own, forward only. Latency counts.
        dict(name="embedding_decode_8", op="embedding", batch=8, seq=1, vocab=50304, context=1024,
             width=768, dtype="float32", scale=1.0, padded=0.0, positions=True, train=False),
        # A small model on short, padded sequences; width and rows odd.
        dict(name="embedding_train_3x337", op="embedding", batch=3, seq=337, vocab=1009,
             context=512, width=250, dtype="float32", scale=1.0, padded=0.2, positions=False,
             train=True),
        # GPT-2 small's micro-batch on one GPU: the package's benchmark.
        dict(name="embedding_train_8x1024", op="embedding", batch=8, seq=1024, vocab=50304,
             context=1024, width=768, dtype="float32", scale=1.0, padded=0.0, positions=False,
             train=True),
        # A large micro-batch of a wider model with bf16 parameters and
        # embeddings scaled by sqrt(width).
        dict(name="embedding_train_64x1024", op="embedding", batch=64, seq=1024, vocab=50304,
             context=1024, width=1024, dtype="bfloat16", scale=32.0, padded=0.0, positions=False,
             train=True),
        # A small model's ragged batch, every row's loss and gradient apart.
        dict(name="cross_entropy_train_77", op="cross_entropy", rows=77, width=256, vocab=1000,
             padded_vocab=1024, ignored=0.1, reduction="none", train=True),
        # Scoring a context of tokens: losses only.
        dict(name="cross_entropy_eval_1024", op="cross_entropy", rows=1024, width=768,
             vocab=50257, padded_vocab=50304, ignored=0.0, reduction="none", train=False),
        # GPT-2 small's head on its micro-batch.
        dict(name="cross_entropy_train_8192", op="cross_entropy", rows=8192, width=768,
             vocab=50257, padded_vocab=50304, ignored=0.05, reduction="mean", train=True),
        # Four such micro-batches at once, where the logits alone would take
        # 3.3 GB in bf16.
        dict(name="cross_entropy_train_32768", op="cross_entropy", rows=32768, width=768,
             vocab=50257, padded_vocab=50304, ignored=0.05, reduction="mean", train=True),
        # A small model's few rows: latency counts.
        dict(name="linear_int8_train_33", op="linear", rows=33, inputs=128, outputs=512,
             gelu=False),
        # GPT-2 small's query-key-value projection on its micro-batch.
        dict(name="linear_int8_train_8192", op="linear", rows=8192, inputs=768, outputs=2304,
             gelu=False),
        # The first layer of an MLP of width 1024.
        dict(name="linear_gelu_int8_train_8192", op="linear", rows=8192, inputs=1024,
             outputs=4096, gelu=True),
        # The same on a large micro-batch, where activations fill the memory.
        dict(name="linear_gelu_int8_train_65536", op="linear", rows=65536, inputs=1024,
             outputs=4096, gelu=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "cross_entropy", "linear"])
    if op == "embedding":
        seq = _log(rng, 1, 1024)
        batch = _log(rng, 1, max(1, 65536 // seq))
        positions = rng.random() < 0.3
        return dict(op=op, batch=batch, seq=seq, vocab=_log(rng, 64, 50304),
                    context=seq + rng.randrange(0, 300), width=_log(rng, 16, 1024),
                    dtype=rng.choice(["float32", "bfloat16"]), scale=rng.choice([1.0, 0.5, 11.25]),
                    padded=rng.choice([0.0, 0.3]), positions=positions,
                    train=rng.random() < 0.8)
    if op == "cross_entropy":
        vocab = _log(rng, 40, 50257)
        return dict(op=op, rows=_log(rng, 1, 16384), width=8 * _log(rng, 4, 96), vocab=vocab,
                    padded_vocab=vocab + rng.choice([0, 1, 47]),
                    ignored=rng.choice([0.0, 0.2]), reduction=rng.choice(["mean", "sum", "none"]),
                    train=rng.random() < 0.75)
    return dict(op=op, rows=_log(rng, 1, 32768), inputs=8 * _log(rng, 4, 200),
                outputs=8 * _log(rng, 4, 320), gelu=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (std * torch.randn(*shape, device="cuda", generator=g)).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] == "embedding":
        dt = DTYPES[case["dtype"]]
        shape = (case["batch"], case["seq"])
        # Token frequencies fall like 1/rank, as in text: rank ~ vocab^u.
        rank = (case["vocab"] ** uniform(*shape).double()).long().sub_(1)
        order = torch.randperm(case["vocab"], device="cuda", generator=g)
        idx = order[rank.clamp_(0, case["vocab"] - 1)]
        if case["padded"]:
            idx = torch.where(uniform(*shape) < case["padded"], -1, idx)
        s["idx"] = idx
        s["positions"] = (torch.randint(0, case["context"], shape, device="cuda", generator=g)
                          if case["positions"] else None)
        s["weight"] = normal(case["vocab"], case["width"], std=0.02, dtype=dt)
        s["pos_weight"] = normal(case["context"], case["width"], std=0.02, dtype=dt)
        s["grad"] = normal(*shape, case["width"], std=1e-3, dtype=dt) if case["train"] else None
    elif case["op"] == "cross_entropy":
        R, C, V = case["rows"], case["width"], case["vocab"]
        # Outputs of the last LayerNorm against a head whose logits spread by
        # about two.
        s["x"] = normal(R, C, dtype=torch.bfloat16)
        s["weight"] = normal(case["padded_vocab"], C, std=2.0 / math.sqrt(C),
                             dtype=torch.bfloat16)
        target = torch.randint(0, V, (R,), device="cuda", generator=g)
        if case["ignored"]:
            target = torch.where(uniform(R) < case["ignored"], -100, target)
        s["target"] = target
        s["grad"] = uniform(R).add_(0.5) if case["reduction"] == "none" else None
    else:
        R, K, N = case["rows"], case["inputs"], case["outputs"]
        s["x"] = normal(R, K, dtype=torch.bfloat16)
        s["weight"] = normal(N, K, std=1.0 / math.sqrt(K), dtype=torch.bfloat16)
        s["bias"] = normal(N, std=0.1, dtype=torch.bfloat16)
        s["grad"] = normal(R, N, std=1e-2, dtype=torch.bfloat16)
    for k in ("x", "weight", "pos_weight", "bias"):
        if k in s and case.get("train", True):
            s[k].requires_grad_()
    return s


def run(s):
    if own:
        return _OWN[s["op"]](s)
    with torch.no_grad():
        return _PLAIN[s["op"]](s)


# -- the package's operators ------------------------------------------------------


def _own_embedding(s):
    from tiny_nccl_b200 import ops
    y = ops.embedding(s["idx"], s["weight"], s["pos_weight"], positions=s["positions"],
                      scale=s["scale"])
    if not s["train"]:
        return y
    return (y, *torch.autograd.grad(y, [s["weight"], s["pos_weight"]], s["grad"]))


def _own_cross_entropy(s):
    from tiny_nccl_b200 import ops
    loss = ops.linear_cross_entropy(s["x"], s["weight"], s["target"], classes=s["vocab"],
                                    reduction=s["reduction"])
    if not s["train"]:
        return loss
    return (loss, *torch.autograd.grad(loss, [s["x"], s["weight"]], s["grad"]))


def _own_linear(s):
    from tiny_nccl_b200 import ops
    f = ops.linear_gelu if s["gelu"] else ops.linear
    y = f(s["x"], s["weight"], s["bias"], activations="int8")
    return (y, *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["grad"]))


# -- plain forms ------------------------------------------------------------------


def _plain_embedding(s):
    dt = s["weight"].dtype
    idx = s["idx"].reshape(-1)
    pos = s["positions"]
    if pos is None:
        pos = torch.arange(s["seq"], device=idx.device).expand(s["batch"], s["seq"])
    pos = pos.reshape(-1)
    real = (idx >= 0)[:, None]
    token = torch.where(real, s["weight"][idx.clamp(min=0)].float() * s["scale"], 0.0)
    y = (token + s["pos_weight"][pos].float()).to(dt).view(s["batch"], s["seq"], -1)
    if not s["train"]:
        return y
    g = s["grad"].reshape(idx.numel(), -1).float()
    gt = torch.where(real, g * s["scale"], 0.0)
    dw = torch.zeros(s["weight"].shape, device=g.device).index_add_(0, idx.clamp(min=0), gt)
    dp = torch.zeros(s["pos_weight"].shape, device=g.device).index_add_(0, pos, g)
    return y, dw.to(dt), dp.to(dt)


def _plain_cross_entropy(s):
    x, w, V = s["x"].float(), s["weight"].float(), s["vocab"]
    target, rows = s["target"], s["x"].shape[0]
    logits = x @ w[:V].t()
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp_().sum(1, keepdim=True).log_().add_(top)
    valid = target >= 0
    at = target.clamp(min=0)
    loss = torch.where(valid, lse[:, 0] - logits.gather(1, at[:, None])[:, 0], 0.0)
    share = 1.0 / valid.sum().clamp(min=1) if s["reduction"] == "mean" else 1.0
    out = loss if s["reduction"] == "none" else loss.sum() * share
    if not s["train"]:
        return out
    g = torch.where(valid, s["grad"] if s["reduction"] == "none" else share, 0.0)
    d = logits.sub_(lse).exp_()
    d[torch.arange(rows, device=x.device), at] -= 1.0
    d *= g[:, None]
    dw = torch.zeros_like(w)
    torch.mm(d.t(), x, out=dw[:V])
    return out, (d @ w[:V]).to(s["x"].dtype), dw.to(s["weight"].dtype)


def _int8_blocks(x):
    """x as 8-bit whole numbers with one power of two for each 32 neighbours
    of a row, read back: the smallest power of two whose 127 steps, with
    rounding to the nearest (ties to even), hold the block's largest value."""
    rows, n = x.shape
    b = torch.nn.functional.pad(x, (0, -n % 32)).view(rows, -1, 32)
    top = b.abs().amax(2, keepdim=True)
    e = torch.frexp(top).exponent - 7  # top / 2^e in [64, 128)
    e = e + (top >= 127.5 * _power_of_two(e)).to(e.dtype)
    step = _power_of_two(e)
    return ((b / step).round_() * step).view(rows, -1)[:, :n]


def _power_of_two(e):
    """2^e in fp32, exactly, from the exponent's bits (normal numbers)."""
    return ((e.clamp(min=-126) + 127) << 23).view(torch.float32)


_K0, _K1 = math.sqrt(2.0 / math.pi), 0.044715


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(_K0 * (x + _K1 * x * x * x)))


def _gelu_slope(x):
    t = torch.tanh(_K0 * (x + _K1 * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * _K0 * (1.0 + 3.0 * _K1 * x * x)


def _plain_linear(s):
    x, w, b, g = (s[k].float() for k in ("x", "weight", "bias", "grad"))
    pre = x @ w.t() + b
    y = _gelu(pre) if s["gelu"] else pre
    if s["gelu"]:
        g = g * _gelu_slope(_int8_blocks(pre))
    dw = g.t() @ _int8_blocks(x)
    return tuple(t.to(torch.bfloat16) for t in (y, g @ w, dw, g.sum(0)))


_OWN = {"embedding": _own_embedding, "cross_entropy": _own_cross_entropy, "linear": _own_linear}
_PLAIN = {"embedding": _plain_embedding, "cross_entropy": _plain_cross_entropy,
          "linear": _plain_linear}


# -- 64 bits ----------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s)


def _exact_embedding(s):
    rows = s["batch"] * s["seq"]
    idx = s["idx"].reshape(rows)
    pos = (s["positions"].reshape(rows) if s["positions"] is not None
           else torch.arange(rows, device=idx.device) % s["seq"])
    keep = idx >= 0
    y = s["pos_weight"].double()[pos]
    y[keep] += s["scale"] * s["weight"].double()[idx[keep]]
    y = y.view(s["batch"], s["seq"], s["width"])
    if not s["train"]:
        return y
    g = s["grad"].double().reshape(rows, s["width"])
    dw = torch.zeros(s["vocab"], s["width"], dtype=torch.float64, device=idx.device)
    dw.index_put_((idx[keep],), s["scale"] * g[keep], accumulate=True)
    dp = torch.zeros(s["context"], s["width"], dtype=torch.float64, device=idx.device)
    dp.index_put_((pos,), g, accumulate=True)
    return y, dw, dp


def _exact_cross_entropy(s):
    w = s["weight"].double()[:s["vocab"]]
    n = int((s["target"] >= 0).sum())
    losses, dxs = [], []
    dw = torch.zeros(s["weight"].shape, dtype=torch.float64, device=w.device)
    for at in range(0, s["rows"], 4096):
        x, t = s["x"][at:at + 4096].double(), s["target"][at:at + 4096]
        keep = (t >= 0).double()
        logits = torch.einsum("rc,vc->rv", x, w)
        lse = torch.logsumexp(logits, 1)
        rows = torch.arange(len(t), device=w.device)
        losses.append((lse - logits[rows, t.clamp(min=0)]) * keep)
        if s["train"]:
            p = torch.exp(logits - lse[:, None])
            p[rows, t.clamp(min=0)] -= 1.0
            c = keep * (s["grad"][at:at + 4096].double() if s["reduction"] == "none"
                        else 1.0 / max(n, 1) if s["reduction"] == "mean" else 1.0)
            p *= c[:, None]
            dxs.append(p @ w)
            dw[:s["vocab"]] += p.t() @ x
    loss = torch.cat(losses)
    if s["reduction"] != "none":
        loss = loss.sum() / (max(n, 1) if s["reduction"] == "mean" else 1)
    return (loss, torch.cat(dxs), dw) if s["train"] else loss


def _exact_int8(x):
    """The same blocks from the definition: for each block the least power of
    two s with round(max / s) <= 127, then s * round(x / s)."""
    rows, n = x.shape
    blocks = -(-n // 32)
    full = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    full[:, :n] = x
    full = full.view(rows, blocks, 32)
    top = full.abs().max(dim=2, keepdim=True).values
    p = torch.floor(torch.log2(torch.where(top > 0, top, 1.0))).long() - 8
    step = ((p + 1023) << 52).view(torch.float64)  # 2^p, exactly
    for _ in range(4):
        step = torch.where(torch.round(top / step) > 127, 2.0 * step, step)
    return (torch.round(full / step) * step).view(rows, -1)[:, :n]


def _exact_linear(s):
    x, w = s["x"].double(), s["weight"].double()
    pre = torch.addmm(s["bias"].double(), x, w.t())
    g, y = s["grad"].double(), pre
    if s["gelu"]:
        y = pre / (1.0 + torch.exp(-2.0 * _K0 * (pre + _K1 * pre ** 3)))
        h = _exact_int8(pre)
        r = 1.0 / (1.0 + torch.exp(-2.0 * _K0 * (h + _K1 * h ** 3)))
        g = g * (r + 2.0 * h * r * (1.0 - r) * _K0 * (1.0 + 3.0 * _K1 * h ** 2))
    return y, g @ w, g.t() @ _exact_int8(x), g.sum(0)


_EXACT = {"embedding": _exact_embedding, "cross_entropy": _exact_cross_entropy,
          "linear": _exact_linear}


# -- what a pass cannot do without ------------------------------------------------


def work(case):
    if case["op"] == "embedding":
        R, C = case["batch"] * case["seq"], case["width"]
        size = 4 if case["dtype"] == "float32" else 2
        used = min(case["context"], R if case["positions"] else case["seq"])
        moved = 8 * R + size * C * (min(R, case["vocab"]) + used + R)
        if case["positions"]:
            moved += 8 * R
        flops = 2 * R * C
        if case["train"]:  # the gradient read, both tables' gradients written
            moved += size * C * (R + case["vocab"] + case["context"])
            flops += 3 * R * C
        return {"bytes": moved, "flops": flops}
    if case["op"] == "cross_entropy":
        R, C, V, P = case["rows"], case["width"], case["vocab"], case["padded_vocab"]
        moved = 2 * R * C + 2 * V * C + 8 * R + (4 * R if case["reduction"] == "none" else 4)
        flops = 2 * R * C * V
        if case["train"]:
            moved += 2 * R * C + 2 * P * C
            flops *= 3
        return {"bytes": moved, "flops": flops}
    R, K, N = case["rows"], case["inputs"], case["outputs"]
    moved = 2 * (2 * R * K + 2 * N * K + 2 * N + 2 * R * N)
    # What is kept in 8 bits is written in the forward and read in the
    # backward pass: the inputs, and before a GELU the sums too.
    moved += 2 * R * (K + -(-K // 32))
    if case["gelu"]:
        moved += 2 * R * (N + -(-N // 32))
    return {"bytes": moved, "flops": 6 * R * K * N}
