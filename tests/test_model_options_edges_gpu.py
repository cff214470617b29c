"""GPT-2's options where some targets are ignored: which rows each loss is the
mean of."""
import pytest
import torch

from test_model_options_gpu import _loss_and_grads, _model

pytestmark = pytest.mark.gpu


def test_ignored_targets_and_the_means(built):
    """head="pieces" is the mean over the rows that count, as impl="torch" is;
    the default head divides by all rows. Loss and gradients differ by that
    factor and nothing else."""
    from tiny_nccl_b200.models import GPT2, GPT2Config
    cfg = GPT2Config(n_layer=2, n_head=4, n_embd=256, vocab_size=1000, block_size=128)
    g = torch.Generator(device="cuda").manual_seed(3)
    idx, tgt = torch.randint(0, 1000, (2, 3, 120), device="cuda", generator=g)
    tgt = torch.where(torch.rand(tgt.shape, device="cuda", generator=g) < 0.2, -100, tgt)
    share = float((tgt >= 0).double().mean())
    assert 0.7 < share < 0.9
    logits, gl = _loss_and_grads(_model(cfg), idx, tgt)
    pieces, gp = _loss_and_grads(_model(cfg, head="pieces"), idx, tgt)
    torch.manual_seed(0)
    model = GPT2(cfg, impl="torch").cuda()
    model.load_state_dict(_model(cfg).state_dict())
    with torch.no_grad():
        plain = model(idx, tgt).item()  # fp32
    # Logits below 4 in bf16 (half a step 2^-7), activations in bf16 before them.
    assert abs(pieces - plain) <= 2 * 2 ** -7
    assert abs(pieces * share - logits) <= 2 ** -7
    for n in gl:
        off = (gp[n] * share - gl[n]).norm() / gl[n].norm()
        assert off < 10 * 2 ** -8, (n, float(off))
