"""Forward-mode derivatives are refused by every operator, whichever input carries the tangent,
with reverse mode switched on or off: a tangent must not be dropped in silence."""
import pytest
import torch
from torch.autograd import forward_ad

import fusedkernels_b200 as fk

pytestmark = pytest.mark.gpu


def calls():
    G = torch.Generator("cuda").manual_seed(0)
    x, r, top = (torch.randn(6, 64, generator=G, device="cuda") for _ in range(3))
    w = torch.ones(64, device="cuda")
    idx = torch.arange(12, device="cuda").view(6, 2)
    return [("add_norm", lambda x, r, w: fk.fused_add_rms_norm(x, r, w), [x, r, w], 3),
            ("quant", lambda x, r, w: fk.fused_add_rms_norm_quant(x, r, w), [x, r, w], 3),
            ("quant alone", lambda x, w: fk.fused_add_rms_norm_quant(x, None, w), [x, w], 2),
            ("balance", lambda x, i: fk.fused_moe_balance_loss(x, i), [x, idx], 1),
            ("distillation", lambda x, t, i: fk.fused_distillation_loss(x, i, t),
             [x, top[:, :2].contiguous(), idx], 2)]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("case", range(5))
def test_tangents_are_refused(case, reverse):
    name, fn, args, floats = calls()[case]
    for which in range(floats):
        with torch.set_grad_enabled(reverse), forward_ad.dual_level():
            given = list(args)
            given[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises((NotImplementedError, AssertionError)):
                fn(*given)
    with torch.no_grad(), forward_ad.dual_level():  # no tangent: as ever
        assert all(torch.is_tensor(t) for t in torch.utils._pytree.tree_leaves(fn(*args)))


def test_module_refuses_with_and_without_a_residual():
    norm = fk.FusedAddRMSNorm(64).cuda().requires_grad_(False)
    x = torch.randn(6, 64, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for residual in (None, x):
            with pytest.raises(NotImplementedError):
                norm(dual, residual)
