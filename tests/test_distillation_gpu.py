"""Distillation loss and gradient against 64-bit arithmetic: operator_reference.distill's bounds
plus one rounding to the output's type."""
import pytest
import torch

import fusedkernels_b200 as fk
from conftest import gen
from fusedkernels_b200.distillation import last_distillation_error
from operator_reference import assert_within, distill, half_step, tiny

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def inputs(n, v, k, dtype=FP, seed=0, hard=True, ragged=True):
    G = gen(seed)
    s = 2.5 * torch.randn(n, v, generator=G)
    top, idx = (0.8 * s + torch.randn(n, v, generator=G)).topk(k, dim=1)
    if ragged:
        used = torch.randint(0, k + 1, (n, 1), generator=G)
        idx = idx.masked_fill(torch.arange(k)[None] >= used, -1)
    targets = None
    if hard:
        targets = torch.randint(0, v, (n,), generator=G)
        targets[1::7] = -100
        targets[2::5] = idx[2::5, 0].clamp(min=0)  # labels among the teacher's ids too
    return s.to(dtype), idx, top.to(dtype), targets


def check(logits, idx, top, targets, temperature=1.0, hard_weight=0.5, scale=1.0, go=None,
          inplace=False, xg=None, **kw):
    xg = logits.cuda().requires_grad_(True) if xg is None else xg
    tg = None if targets is None else targets.cuda()
    args = dict(temperature=temperature, hard_weight=hard_weight, **kw)
    with torch.no_grad():
        only = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda(), tg, inplace_grad=inplace,
                                          **args)
        assert torch.equal(xg.cpu(), logits)  # no gradient wanted: nothing is written
    loss = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda(), tg, inplace_grad=inplace,
                                      loss_scale=scale, **args)
    go = scale if go is None else go
    (grad,) = torch.autograd.grad(loss, xg, torch.tensor(go, device="cuda"))
    assert grad.dtype == logits.dtype and loss.dtype == FP
    if inplace:
        assert grad.data_ptr() == xg.data_ptr()
    want, wgrad, lb, gb = distill(logits, idx, top, targets, loss_scale=go, **args)
    t = logits.dtype
    assert_within(loss, want, lb + half_step(FP) * want.abs(), "loss")
    assert_within(only, want, lb + half_step(FP) * want.abs(), "loss alone")
    again = 2 if go != scale else 1
    assert_within(grad, wgrad, gb + again * 1.01 * half_step(t) * wgrad.abs() +
                  tiny(t) * (1 + abs(go / scale)), "grad")
    return loss.detach(), grad


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("hard", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 1.5, 3.0, 4.0, 2.3, 0.7])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 50, 3), (5, 7, 7), (40, 1000, 16),
                                   (9, 4099, 33), (3, 32000, 64), (2, 50257, 100)])
def test_matches_64_bits(n, v, k, temperature, hard, dtype):
    logits, idx, top, targets = inputs(n, v, k, dtype, seed=n + v, hard=hard)
    check(logits, idx, top, targets, temperature, scale=256.0 if dtype == HF else 1.0)
    assert last_distillation_error() == 0


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("v", [1024, 1001, 128256])
def test_inplace_and_weights(dtype, v):
    logits, idx, top, targets = inputs(6, v, 20, dtype, seed=v)
    for hw in (0.0, 0.3, 1.0):
        check(logits, idx, top, targets, hard_weight=hw, inplace=True)
    check(logits, idx, top, targets, temperature=3.0, inplace=True)


def test_more_rows_than_the_grid_twice():
    logits, idx, top, targets = inputs(1700, 264, 8, BF, seed=1)
    a = check(logits, idx, top, targets, 2.0)
    b = check(logits, idx, top, targets, 2.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("k", [1, 31, 256, 1024])
def test_slots(k):
    logits, idx, top, targets = inputs(5, 2500, k, FP, seed=k, ragged=False)
    check(logits, idx, top, targets)
    check(logits, idx, top, None)
    check(logits, idx.flip(1), top.flip(1), targets)  # any order


def test_ids_standing_twice():
    logits, idx, top, targets = inputs(30, 300, 12, FP, seed=2, ragged=False)
    idx[:, 5] = idx[:, 0]
    idx[::2, 7:10] = idx[::2, 3:4]
    idx[4] = 17
    targets[4], targets[6], targets[8] = 17, idx[6, 0], idx[8, 3]
    a = check(logits, idx, top, targets)
    assert all(torch.equal(p, q) for p, q in zip(a, check(logits, idx, top, targets)))
    check(logits, idx, top, None, temperature=2.0)
    check(logits.bfloat16(), idx, top, targets, inplace=True)


@pytest.mark.parametrize("hard", [False, True])
def test_empty_teacher_rows(hard):
    logits, idx, top, targets = inputs(20, 100, 6, FP, seed=3, hard=hard)
    idx[3] = -1
    top[5] = -float("inf")
    top[6, 1:] = -float("inf")
    top[7, 2] = -1e30
    top[8] = torch.finfo(FP).min  # a mask of the type's lowest value: all slots alike
    check(logits, idx, top, targets)
    check(logits, idx, top, targets, temperature=2.0)


@pytest.mark.parametrize("hard", [False, True])
@pytest.mark.parametrize("k", [5, 64])
def test_empty_teacher_rows_among_many(k, hard):
    """Batches of 4096 rows and more share a warp between teacher rows: rows without a teacher,
    with NaN, ids out of range or ids standing twice lie beside ordinary ones."""
    logits, idx, top, targets = inputs(4200, 96, k, FP, seed=15, hard=hard)
    idx[5::3] = -1
    top[7::11] = -float("inf")
    idx[8::13, 0] = idx[8::13, 1].clamp(min=0)
    idx[8::13, 1] = idx[8::13, 0]
    check(logits, idx, top, targets)
    idx[100, 0] = 7
    top[100, 0] = float("nan")
    idx[201, 0] = 96
    if hard:
        targets[100] = targets[201] = 3
    xg = logits.cuda().requires_grad_(True)
    loss = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda(),
                                      None if targets is None else targets.cuda())
    loss.backward()
    assert torch.isnan(loss) and last_distillation_error() == 1
    assert torch.isnan(xg.grad[201]).all() and torch.isnan(xg.grad[100]).any()
    rest = [i for i in range(4200) if i not in (100, 201)]
    assert torch.isfinite(xg.grad[rest]).all()


def test_nothing_counts():
    logits, idx, top, targets = inputs(4, 60, 3, BF, seed=4)
    loss, grad = check(logits, idx, top, torch.full_like(targets, -100))
    assert loss == 0 and torch.count_nonzero(grad) == 0
    loss, grad = check(logits, torch.full_like(idx, -1), top, None)
    assert loss == 0 and torch.count_nonzero(grad) == 0
    x = torch.zeros(0, 60, device="cuda", requires_grad=True)
    loss = fk.fused_distillation_loss(x, idx[:0].cuda(), top[:0].cuda())
    loss.backward()
    assert loss == 0 and x.grad.shape == (0, 60)


def test_ignore_index():
    logits, idx, top, targets = inputs(12, 80, 4, FP, seed=5)
    targets[targets == -100] = 9
    check(logits, idx, top, targets, ignore_index=9)


def test_infinite_and_nan_logits():
    logits, idx, top, _ = inputs(8, 90, 5, FP, seed=6, hard=False, ragged=False)
    logits[:, 70:] = -float("inf")  # a padded vocabulary
    idx = idx.clamp(max=69)
    check(logits, idx, top, None)
    logits[1, idx[1, 0]] = -float("inf")  # the teacher's id has no probability: an infinite loss
    xg = logits.cuda().requires_grad_(True)
    loss = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda())
    loss.backward()
    assert loss == float("inf") and torch.isfinite(xg.grad).all()
    logits[2, 3] = float("nan")
    xg = logits.cuda().requires_grad_(True)
    loss = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda())
    loss.backward()
    assert torch.isnan(loss) and torch.isnan(xg.grad[2]).all()
    assert torch.isfinite(xg.grad[[0, 1, 3, 4, 5, 6, 7]]).all()


@pytest.mark.parametrize("which", ["idx", "target", "negative target"])
@pytest.mark.parametrize("v", [50, 4096])
def test_out_of_range_is_nan(which, v):
    logits, idx, top, targets = inputs(6, v, 4, FP, seed=7, ragged=False)
    targets[1] = 0
    if which == "idx":
        idx[3, 2] = v
    else:
        targets[3] = v if which == "target" else -7
    idx[2, 0] = 10 ** 12
    targets[2] = -100  # an ignored row may hold anything
    xg = logits.cuda().requires_grad_(True)
    loss = fk.fused_distillation_loss(xg, idx.cuda(), top.cuda(), targets.cuda())
    loss.backward()
    assert torch.isnan(loss) and last_distillation_error() == 1
    assert torch.isnan(xg.grad[3]).all() and torch.isfinite(xg.grad[[0, 1, 2, 4, 5]]).all()
    assert torch.count_nonzero(xg.grad[2]) == 0


def test_extreme_values():
    """Logits far apart: the largest fp32 values that a difference of two does not overflow."""
    logits, idx, top, targets = inputs(6, 64, 4, FP, seed=8, ragged=False)
    logits[0] *= 1e4
    logits[1, 5] = 1e30
    logits[2] -= 1e6
    targets[0], idx[0, 0] = int(logits[0].argmax()), int(logits[0].argmax())
    for i in range(3):
        check(logits[i:i + 1], idx[i:i + 1], top[i:i + 1], targets[i:i + 1].clamp(min=0))


@pytest.mark.parametrize("dtype", [FP, BF])
def test_strides(dtype):
    logits, idx, top, targets = inputs(30, 512, 8, dtype, seed=9)
    wide = torch.zeros(30, 1200, dtype=dtype, device="cuda")
    for a in (0, 8, 3, 600):
        wide[:, a:a + 512] = logits.cuda()
        before = wide.clone()
        check(logits, idx, top, targets, xg=wide[:, a:a + 512].detach().requires_grad_(True))
        assert torch.equal(wide, before)
        check(logits, idx, top, targets, inplace=True,
              xg=wide[:, a:a + 512].detach().requires_grad_(True))
        outside = torch.ones(1200, dtype=torch.bool)
        outside[a:a + 512] = False
        assert torch.equal(wide[:, outside], before[:, outside])
        wide.copy_(before)
    check(logits, idx, top, targets, xg=logits.t().contiguous().cuda().t().detach()
          .requires_grad_(True))
    one = logits[:1].expand(30, 512)
    check(one, idx, top, targets, xg=one.cuda()[:1].expand(30, 512).detach().requires_grad_(True))
    check(logits, idx.int(), top.t().contiguous().t(), targets.int())
    check(logits, idx, top.float(), targets)
    check(logits, idx, top.half(), targets)


@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_other_factors(dtype):
    logits, idx, top, targets = inputs(16, 640, 8, dtype, seed=10)
    check(logits, idx, top, targets, scale=512.0)
    check(logits, idx, top, targets, scale=64.0, go=16.0)
    check(logits, idx, top, targets, scale=64.0, go=100.0)


def test_gradient_against_differences():
    """Central differences in fp32 with steps of 2^-6: third derivatives below 1 for a mean over
    3 rows (error 2^-12 / 6), the loss's roundings 2^-22 * 8 / 2^-5."""
    logits, idx, top, targets = inputs(3, 20, 4, FP, seed=11, ragged=False)
    _, grad = check(logits, idx, top, targets, 2.0, 0.3)
    for i in range(logits.numel()):
        ends = []
        for step in (2.0 ** -6, -2.0 ** -6):
            s = logits.clone()
            s.view(-1)[i] += step
            loss = fk.fused_distillation_loss(s.cuda(), idx.cuda(), top.cuda(), targets.cuda(),
                                              2.0, 0.3)
            ends.append((float(loss), float(s.view(-1)[i])))
        diff = (ends[0][0] - ends[1][0]) / (ends[0][1] - ends[1][1])
        assert abs(diff - float(grad.view(-1)[i])) <= 2e-4


def test_hard_weight_one_is_cross_entropy():
    logits, idx, top, targets = inputs(40, 1000, 8, FP, seed=12)
    a, ga = check(logits, idx, top, targets, hard_weight=1.0)
    xg = logits.cuda().requires_grad_(True)
    b = fk.fused_cross_entropy(xg, targets.cuda())
    b.backward()
    assert abs(a.item() - b.item()) <= 2e-6 * abs(b.item())
    torch.testing.assert_close(ga, xg.grad, rtol=2e-5, atol=1e-8)


def test_second_backward_raises_and_refusals():
    logits, idx, top, targets = (t.cuda() for t in inputs(6, 40, 4))
    x = logits.requires_grad_(True)
    loss = fk.fused_distillation_loss(x, idx, top, targets)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="handed over"):
        loss.backward()
    big = torch.zeros(6, 1025, device="cuda")
    for a, kw in (((x, idx[:5], top[:5]), {}), ((x, idx, top[:, :3]), {}),
                  ((x, idx[:, :0], top[:, :0]), {}), ((x, big.long(), big), {}),
                  ((x, idx.float(), top), {}), ((x, idx.cpu(), top), {}),
                  ((x, idx, top.cpu()), {}), ((x, idx, top.clone().requires_grad_(True)), {}),
                  ((x, idx, top, targets[:5]), {}), ((x, idx, top, targets.cpu()), {}),
                  ((x, idx, top, targets.float()), {}), ((x, idx, top), dict(temperature=0.0)),
                  ((x, idx, top, targets), dict(hard_weight=1.5)), ((x[0], idx, top), {}),
                  ((x, idx, top), dict(loss_scale=-2.0)), ((x.cpu(), idx.cpu(), top.cpu()), {})):
        with pytest.raises(AssertionError):
            fk.fused_distillation_loss(*a, **kw)
    with pytest.raises(TypeError):
        fk.fused_distillation_loss(x.double(), idx, top)


def test_graph_replay_beside_another_stream():
    """Two captured graphs replayed at once on two streams, against the eager results."""
    sets = [inputs(200, 2048, 16, BF, seed=s) for s in (13, 14)]
    graphs = []
    for logits, idx, top, targets in sets:
        x, i, p, y = (t.cuda() for t in (logits, idx, top, targets))
        x.requires_grad_(True)
        fk.fused_distillation_loss(x, i, p, y)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = fk.fused_distillation_loss(x, i, p, y)
            (grad,) = torch.autograd.grad(loss, x)
        graphs.append((g, loss, grad, (x, i, p, y)))  # a graph reads its inputs where they are
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for s, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (logits, idx, top, targets), (_, loss, grad, _) in zip(sets, graphs):
        eager = check(logits, idx, top, targets)
        assert torch.equal(eager[0], loss) and torch.equal(eager[1], grad)


@pytest.mark.parametrize("v", [600, 601])
def test_mean_of_equal_rows(v):
    """n times the same row: the sum in 64 bits is n times that row's loss, so the mean is the one
    row's loss, bit for bit (601 with a gradient at another offset takes the element loops)."""
    logits, idx, top, targets = inputs(1, v, 6, FP, seed=16, ragged=False)
    targets[:] = 5

    def loss(n):
        x = logits.expand(n, v).contiguous().cuda()
        if v == 601:
            x = torch.nn.functional.pad(x, (1, 2))[:, 1:602]
        x.requires_grad_(True)
        return fk.fused_distillation_loss(x, idx.expand(n, -1).cuda(), top.expand(n, -1).cuda(),
                                          targets.expand(n).cuda()).detach()

    one = loss(1)
    for n in (3, 7, 13, 14, 15, 26, 41, 47, 55):  # 1 / (1 / n) is not n in 32 bits for most
        assert torch.equal(loss(n), one), n


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("v", [1000, 1003, 4096])
def test_hard_weight_one_leaves_the_teacher_out(v, dtype):
    """Even where its logits are NaN or infinite."""
    logits, idx, top, targets = inputs(8, v, 6, dtype, seed=17, ragged=False)
    targets[:] = idx[:, 1]
    top[0, 1], top[1, 1], top[2, 3] = float("nan"), float("inf"), float("inf")
    top[4] = float("nan")
    for temperature in (1.0, 2.0):
        _, grad = check(logits, idx, top, targets, temperature, hard_weight=1.0)
        assert torch.isfinite(grad).all()
    wide = torch.zeros(8, v + 13, dtype=dtype, device="cuda")
    wide[:, 3:v + 3] = logits.cuda()  # the element loops
    check(logits, idx, top, targets, 2.0, hard_weight=1.0,
          xg=wide[:, 3:v + 3].detach().requires_grad_(True))
