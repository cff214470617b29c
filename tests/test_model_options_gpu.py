"""GPT-2 with the training operators as options of the fused model, against
the default fused model: gradients, a captured trainer step, and the memory
that the options save."""
import pytest
import torch

pytestmark = pytest.mark.gpu

OPTIONS = [dict(embedding="fused"), dict(head="pieces"), dict(activations="int8"),
           dict(embedding="fused", head="pieces", activations="int8")]


def _model(cfg, **kw):
    from tiny_nccl_b200.models import GPT2
    torch.manual_seed(0)
    return GPT2(cfg, impl="fused", **kw).cuda()


def _loss_and_grads(model, idx, tgt):
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = model(idx, tgt)
    loss.backward()
    return loss.item(), {n: p.grad for n, p in model.named_parameters()}


@pytest.mark.parametrize("kw", OPTIONS, ids=lambda kw: "+".join(kw))
def test_options_match_the_default(built, kw):
    from tiny_nccl_b200.models import GPT2Config
    cfg = GPT2Config(n_layer=2, n_head=4, n_embd=256, vocab_size=1000, block_size=128)
    g = torch.Generator(device="cuda").manual_seed(3)
    idx, tgt = torch.randint(0, 1000, (2, 3, 120), device="cuda", generator=g)
    want, gw = _loss_and_grads(_model(cfg), idx, tgt)
    got, gg = _loss_and_grads(_model(cfg, **kw), idx, tgt)
    # The default rounds logits to bf16 (half a step of values below 4 is
    # 2^-7) before the loss; 8-bit activations do not enter the forward pass.
    assert abs(got - want) <= 2 ** -7
    # A gradient's relative error: 8 bits round an activation by at most
    # 2^-7 of its block's largest value, bf16 by 2^-8 of a value; some ten such
    # roundings lie between the loss and the first layer.
    for n in gw:
        off = (gg[n] - gw[n]).norm() / gw[n].norm()
        assert off < 10 * 2 ** -7, (n, float(off))


def test_options_are_checked():
    from tiny_nccl_b200.models import GPT2, GPT2Config
    cfg = GPT2Config(n_layer=1, n_head=1, n_embd=8, vocab_size=16, block_size=4)
    for kw in (dict(embedding="sorted"), dict(head="chunks"), dict(activations="int4"),
               dict(impl="torch", head="pieces")):
        with pytest.raises(ValueError):
            GPT2(cfg, **kw)
    m = GPT2(cfg, embedding="fused").cuda()
    with pytest.raises(ValueError):
        m(torch.zeros(1, 5, dtype=torch.int64, device="cuda"))


def test_last_position_logits(built):
    """Inference through the fused embedding: the same bits as the default.
    8-bit activations skip a bf16 rounding (2^-8) before each GELU."""
    from tiny_nccl_b200.models import GPT2Config
    cfg = GPT2Config(n_layer=2, n_head=4, n_embd=128, vocab_size=500, block_size=64)
    idx = torch.randint(0, 500, (2, 33), device="cuda")
    models = _model(cfg), _model(cfg, embedding="fused", head="pieces"), _model(cfg, **OPTIONS[-1])
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        a, b, c = (m(idx).double() for m in models)
    assert torch.equal(a, b)
    assert (c - a).norm() <= 4 * 2 ** -8 * a.norm()


def test_trainer_step_with_all_options(built):
    """The trainer (flat gradient buffer, AdamW's bf16 copies, CUDA graph) with
    all three options follows its own eager steps."""
    import datetime
    import os

    import torch.distributed as dist

    import tiny_nccl_b200 as tn
    from conftest import free_port
    from tiny_nccl_b200.models import GPT2Config
    from tiny_nccl_b200.parallel import DataParallelTrainer

    own_group = not dist.is_initialized()
    if own_group:
        os.environ.update({"MASTER_ADDR": "127.0.0.1", "MASTER_PORT": str(free_port())})
        dist.init_process_group("nccl", rank=0, world_size=1,
                                device_id=torch.device("cuda", 0),
                                timeout=datetime.timedelta(seconds=60))
    cfg = GPT2Config(n_layer=2, n_head=4, n_embd=128, vocab_size=500, block_size=64)
    g = torch.Generator(device="cuda").manual_seed(5)
    data = torch.randint(0, 500, (6, 4, 65), device="cuda", generator=g)
    runs = {}
    try:
        for graph in (False, True):
            comm = tn.init_from_torch_distributed(device=0)
            model = _model(cfg, **OPTIONS[-1])
            tr = DataParallelTrainer(model, comm, lr=1e-3, reducer="flat", cuda_graph=graph)
            losses = [tr.step(d[:, :-1], d[:, 1:]).item() for d in data]
            runs[graph] = (losses, [p.detach().clone() for p in model.parameters()])
            tr.close()
            comm.destroy()
    finally:
        if own_group:
            dist.destroy_process_group()
    (le, pe), (lg, pg) = runs[False], runs[True]
    for a, b in zip(le, lg):
        assert abs(a - b) < 1e-3 * abs(a), (le, lg)
    for a, b in zip(pe, pg):
        torch.testing.assert_close(a, b, rtol=1e-2, atol=1e-3)


def test_options_save_memory(built):
    """A step of a model whose logits and activations count: the options lower
    the peak by what the logits (bf16) and half of the kept activations take."""
    from tiny_nccl_b200.models import GPT2Config
    cfg = GPT2Config(n_layer=4, n_head=4, n_embd=256, vocab_size=50000, block_size=512)
    idx = torch.randint(0, 50000, (2, 16, 512), device="cuda")
    peak = []
    for kw in ({}, OPTIONS[-1]):
        m = _model(cfg, **kw)
        _loss_and_grads(m, *idx)
        torch.cuda.synchronize()
        for p in m.parameters():
            p.grad = None
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        _loss_and_grads(m, *idx)
        torch.cuda.synchronize()
        peak.append(torch.cuda.max_memory_allocated() - before)
        del m
    rows = 16 * 512
    logits, kept = rows * 50048 * 2, 4 * rows * 256 * 11  # bytes; 11 widths of bf16, halved
    scratch = 512 << 20
    assert peak[0] - peak[1] > logits + kept - scratch, peak
