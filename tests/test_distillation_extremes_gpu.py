"""Distillation of logits far from zero and beside masks of their type's lowest value, against
64-bit arithmetic.

The bounds do not grow with the logits: each exponential is formed of x - max, so its error is 2
to 4 ulp and 3 roundings of (x - max) / T, which is at most 88 where the exponential is not 0 in 32
bits; factors that join partial sums have the same."""
import pytest
import torch

import fusedkernels_b200 as fk
from conftest import gen
from operator_reference import U, assert_within, half_step, tiny

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def reference(logits, idx, top, targets, temperature, hard_weight):
    """Loss, gradient and their bounds (without the rounding to the type); rows all count."""
    x = logits.double()
    n, v = x.shape
    t, a = temperature, (0.0 if targets is None else hard_weight)
    s = 1.0 if targets is None else 1.0 - a
    d = x - x.amax(1, keepdim=True)
    far = (-d * max(1.0, 1.0 / t)).clamp(max=90.0)
    p = torch.softmax(top.double() / t, 1)
    teacher_far = ((top.double().amax(1, keepdim=True) - top.double()) / t).clamp(max=90.0)
    dense = torch.zeros_like(x).scatter_add_(1, idx, p)
    # a sum: v / 256 terms by one thread, then a tree
    base = v / 256 + 64
    loss = loss_err = torch.zeros(n, dtype=torch.float64)
    grad, err = torch.zeros_like(x), torch.zeros_like(x)
    for weight, temp, soft in ((s, t, True), (a, 1.0, False)):
        if weight == 0.0:
            continue
        q = torch.softmax(d / temp, 1)
        z_err = base + 8 * (q * far).sum(1)
        lz = torch.logsumexp(d / temp, 1)
        q_err = q * (z_err[:, None] + 8 * far)
        if soft:
            picked = d.gather(1, idx) / t
            loss = loss + weight * t * t * ((p * (p.log() - picked)).sum(1) + lz)
            size = (p * (p.log().abs() + picked.abs())).sum(1) + lz + 1
            p_err = 64 + 8 * (p * teacher_far).sum(1) + 8 * teacher_far.amax(1)
            loss_err = loss_err + weight * t * t * (size * p_err + z_err)
            grad = grad + weight * t * (q - dense)
            err = err + weight * t * (q_err + dense * p_err[:, None])
        else:
            at = targets[:, None]
            hit = d.gather(1, at)[:, 0]
            loss = loss + weight * (lz - hit)
            loss_err = loss_err + weight * (64 * (lz + hit.abs() + 1) + z_err)
            one = torch.zeros_like(x).scatter_(1, at, 1.0)
            grad = grad + weight * (q - one)
            err = err + weight * (q_err + 8 * one)
    return loss.mean(), grad / n, U * loss_err.mean(), U * err / n


def check(logits, idx, top, targets, temperature, hard_weight=0.5, xg=None):
    xg = logits.cuda().requires_grad_(True) if xg is None else xg
    loss = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda(),
                                      None if targets is None else targets.cuda(),
                                      temperature=temperature, hard_weight=hard_weight)
    (grad,) = torch.autograd.grad(loss, xg)
    want, wgrad, lb, gb = reference(logits, idx, top, targets, temperature, hard_weight)
    t = logits.dtype
    assert_within(loss, want, lb + half_step(FP) * want.abs(), "loss")
    assert_within(grad, wgrad, gb + 1.01 * half_step(t) * wgrad.abs() + tiny(t) + 2.0 ** -126, "grad")
    return loss.detach(), grad


def inputs(n, v, k, dtype, seed, hard):
    G = gen(seed)
    s = 2.5 * torch.randn(n, v, generator=G)
    top, idx = (0.8 * s + torch.randn(n, v, generator=G)).topk(k, dim=1)
    targets = torch.randint(0, v, (n,), generator=G) if hard else None
    return s, idx, top.to(dtype), targets


# One packet a thread, four, sixteen; clusters of CTAs; an odd width.
VOCABS = [1000, 1024, 3001, 20000, 60000]
# One temperature, a square, powers, two exponentials; below 1.
TEMPERATURES = [1.0, 2.0, 3.0, 2.3, 0.7]


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
@pytest.mark.parametrize("temperature", TEMPERATURES)
@pytest.mark.parametrize("hard", [False, True])
@pytest.mark.parametrize("v", VOCABS)
def test_offsets(v, hard, temperature, dtype):
    """Rows that lie around +-1000 and +-30000."""
    s, idx, top, targets = inputs(6, v, 8, dtype, v, hard)
    for i, offset in enumerate((0.0, 1000.0, -1000.0, 30000.0, -30000.0, 3.0)):
        s[i] += offset
    check(s.to(dtype), idx, top, targets, temperature)


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
@pytest.mark.parametrize("temperature", TEMPERATURES)
@pytest.mark.parametrize("hard", [False, True])
@pytest.mark.parametrize("v", VOCABS)
def test_lowest_value_masks(v, hard, temperature, dtype):
    """Logits masked with the type's lowest value: a padded tail, the first half, a quarter in the
    middle, all but one, and a whole row (its softmax is uniform)."""
    s, idx, top, targets = inputs(6, v, 8, dtype, v + 1, hard)
    low = torch.finfo(dtype).min
    s = s.to(dtype)
    kept = torch.ones(6, v, dtype=torch.bool)
    kept[0, v - v // 40:] = False
    kept[1, :v // 2] = False
    kept[2, v // 4:v // 2] = False
    kept[3] = False
    kept[3, v // 3] = True
    s = s.masked_fill(~kept, low)
    s[4] = low
    s[5, : v // 2] = -float("inf")  # beside minus infinity
    s[5, v // 2:] = low
    G = gen(v + 2)
    for i in range(6):  # the teacher's ids and the label are not masked
        open_ = torch.arange(v // 2, v) if i == 5 else kept[i].nonzero()[:, 0]
        pick = open_[torch.randperm(len(open_), generator=G)[:8]]
        idx[i] = pick[torch.arange(8) % len(pick)]
        if hard:
            targets[i] = idx[i, 3]
    loss, grad = check(s, idx, top, targets, temperature)
    assert torch.isfinite(loss) and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", [FP, BF], ids=str)
@pytest.mark.parametrize("temperature", [1.0, 2.3])
def test_other_offset_from_16_bytes(dtype, temperature):
    """The element loops give the same bounds."""
    s, idx, top, targets = inputs(6, 1001, 8, dtype, 5, True)
    s[1] += 1000.0
    s[2, 900:] = torch.finfo(dtype).min
    s[3] = torch.finfo(dtype).min
    s = s.to(dtype)
    idx[2], targets[2] = torch.arange(8), 5
    wide = torch.zeros(6, 1105, dtype=dtype, device="cuda")
    wide[:, 3:1004] = s.cuda()
    check(s, idx, top, targets, temperature, xg=wide[:, 3:1004].detach().requires_grad_(True))
