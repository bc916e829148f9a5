"""Balance loss of logits far from zero and beside masks of their type's lowest value, against
64-bit arithmetic.

The bounds do not grow with the logits, but for the z-loss's logsumexp itself: each exponential is
formed of x - max, so its error is 2 ulp and 3 roundings of x - max, which is at most 90 where the
exponential is not 0 in 32 bits; sums of at most 256 terms in a tree, and 32 roundings around them."""
import pytest
import torch

import fusedkernels_b200 as fk
from conftest import gen
from operator_reference import U, assert_within, half_step, tiny

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def check(logits, idx, z_coef, xg=None):
    xg = logits.cuda().requires_grad_(True) if xg is None else xg
    loss, counts = fk.fused_moe_balance_loss(xg, idx.cuda(), z_coef=z_coef)
    (got,) = torch.autograd.grad(loss, xg)
    x = logits.double()
    n, e = x.shape
    assert torch.equal(counts.cpu(), torch.bincount(idx.reshape(-1), minlength=e))
    g = counts.cpu().double() / idx.numel() - 1 / e
    d = x - x.amax(1, keepdim=True)
    far = (-d).clamp(max=90.0)
    p = torch.softmax(d, 1)
    lse = torch.logsumexp(x, 1, keepdim=True)
    share = (p * g).sum(1, keepdim=True)
    p_err = 64 + 8 * far + 8 * (p * far).sum(1, keepdim=True)  # relative
    share_err = (p * g.abs() * p_err).sum(1, keepdim=True)
    lse_err = 4 * lse.abs() + 64 + 8 * (p * far).sum(1, keepdim=True)
    want = (1 + e * share.sum() / n + z_coef * lse.square().sum() / n)
    bound = U * ((1 + e * share_err.sum() / n) + z_coef * (2 * lse.abs() * lse_err).sum() / n +
                 8 * want.abs())
    assert_within(loss, want, bound, "loss")
    ce, cz = e / n, 2 * z_coef / n
    grad = p * (ce * (g - share) + cz * lse)
    err = p * (p_err * (ce * (g.abs() + share.abs()) + cz * lse.abs()) +
               ce * (share_err + 8 * g.abs()) + cz * lse_err)
    t = logits.dtype
    assert_within(got, grad, U * err + 1.01 * half_step(t) * grad.abs() + tiny(t) + 2.0 ** -126,
                  "grad")


def inputs(e, k, dtype, seed):
    G = gen(seed)
    s = 2.0 * torch.randn(40, e, generator=G) + torch.randn(e, generator=G)
    return s, s.topk(k, dim=1).indices, G


# Whole packets, tiles of odd rows, and (in the last test) other strides.
EXPERTS = [8, 64, 128, 256, 7, 61, 161]


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
@pytest.mark.parametrize("z_coef", [0.0, 1e-3])
@pytest.mark.parametrize("e", EXPERTS)
def test_offsets(e, z_coef, dtype):
    s, idx, _ = inputs(e, 2, dtype, e)
    s += torch.tensor([0.0, 1000.0, -1000.0, 30000.0, -30000.0]).repeat(8)[:, None]
    check(s.to(dtype), idx, z_coef)


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
@pytest.mark.parametrize("e", EXPERTS)
def test_lowest_value_masks(e, dtype):
    """Experts switched off by the type's lowest value: some, all but one, all of them (uniform),
    and beside minus infinity."""
    s, idx, _ = inputs(e, 2, dtype, e + 1)
    s = s.to(dtype)
    low = torch.finfo(dtype).min
    s[::4, e // 2:] = low
    s[1::4] = low
    s[1::8, e // 3] = 1.0
    s[2::4, : e // 2] = -float("inf")
    s[2::4, e // 2:] = low
    check(s, idx, 0.0)


@pytest.mark.parametrize("dtype", [FP, BF], ids=str)
def test_other_strides(dtype):
    s, idx, _ = inputs(40, 2, dtype, 3)
    s[::3] += 1000.0
    s = s.to(dtype)
    s[1::3, 20:] = torch.finfo(dtype).min
    wide = torch.zeros(40, 99, dtype=dtype, device="cuda")
    wide[:, 3:43] = s.cuda()
    check(s, idx, 1e-3, wide[:, 3:43].detach().requires_grad_(True))
