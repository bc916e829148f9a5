"""MiniGPT's options, what of them needs no GPU."""
import pytest
import torch

from fusedkernels_b200 import FusedMoEMLPSorted
from fusedkernels_b200.mini_gpt import MiniGPT

CFG = dict(vocab_size=50, dim=64, n_layers=2, n_heads=2, hidden_dim=64, max_seq_len=8)


@pytest.mark.parametrize("kw", [dict(), dict(fused=False), dict(fused_residual=True),
                                dict(n_experts=4), dict(n_experts=4, balance_coef=0.0)], ids=str)
def test_balance_loss_is_zero_where_nothing_asks_for_one(kw):
    assert MiniGPT(**CFG, **kw).balance_loss() == 0


def as_pickled_before(module, names):
    """What unpickling gives for a module saved by a version without these attributes."""
    for m in module.modules():
        for name in names:
            m.__dict__.pop(name, None)
    return module


def test_models_pickled_before_the_options():
    torch.manual_seed(0)
    model = MiniGPT(**CFG, fused=False)
    idx = torch.randint(0, 50, (2, 9))
    want = model(idx[:, :-1], idx[:, 1:])
    old = as_pickled_before(model, ("fused_residual", "n_experts"))
    assert torch.equal(old(idx[:, :-1], idx[:, 1:]), want)


def test_layers_pickled_before_the_options():
    old = as_pickled_before(FusedMoEMLPSorted(64, 64, 4, 2),
                            ("balance_coef", "z_coef", "balance_loss", "expert_counts"))
    assert old.balance_coef == 0.0 and old.z_coef == 0.0
    assert old.balance_loss is None and old.expert_counts is None
