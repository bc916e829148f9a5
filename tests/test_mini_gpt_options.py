"""MiniGPT's options, what of them needs no GPU."""
import pytest

from fusedkernels_b200.mini_gpt import MiniGPT

CFG = dict(vocab_size=50, dim=64, n_layers=2, n_heads=2, hidden_dim=64, max_seq_len=8)


@pytest.mark.parametrize("kw", [dict(), dict(fused=False), dict(fused_residual=True),
                                dict(n_experts=4), dict(n_experts=4, balance_coef=0.0)], ids=str)
def test_balance_loss_is_zero_where_nothing_asks_for_one(kw):
    assert MiniGPT(**CFG, **kw).balance_loss() == 0
