"""Router balance loss with counts against 64-bit arithmetic.  Counts have to be equal; loss and
gradient are held to operator_reference.balance's bounds plus one rounding to their type."""
import pytest
import torch

import fusedkernels_b200 as fk
from conftest import gen
from operator_reference import assert_within, balance, half_step, tiny

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def inputs(n, e, k, dtype=FP, masked=False, seed=0):
    G = gen(seed)
    logits = (torch.randn(n, e, generator=G) + torch.randn(e, generator=G)).to(dtype)
    idx = logits.float().topk(k, dim=1).indices
    mask = torch.rand(n, generator=G) < 0.7 if masked else None
    return logits, idx, mask


def check(logits, idx, mask, z=0.0, scale=1.0, go=None, xg=None):
    xg = logits.cuda().requires_grad_(True) if xg is None else xg
    loss, counts = fk.fused_moe_balance_loss(xg, idx.cuda(),
                                             None if mask is None else mask.cuda(), z, scale)
    assert counts.dtype == torch.int64 and not counts.requires_grad and loss.dtype == FP
    go = scale if go is None else go
    (grad,) = torch.autograd.grad(loss, xg, torch.tensor(go, device="cuda"))
    assert grad.dtype == logits.dtype
    want, wcounts, wgrad, lb, gb = balance(logits, idx, mask, z, go)
    assert torch.equal(counts.cpu(), wcounts)
    assert_within(loss, want, lb + half_step(FP) * want.abs(), "loss")
    t = logits.dtype
    again = 2 if go != scale else 1  # another factor rounds once more
    # what is rounded first is the gradient for `scale`, among the subnormals too
    assert_within(grad, wgrad, gb + again * 1.01 * half_step(t) * wgrad.abs() +
                  tiny(t) * (1 + abs(go / scale)), "grad")
    with torch.no_grad():
        l2, c2 = fk.fused_moe_balance_loss(xg, idx.cuda(), None if mask is None else mask.cuda(), z)
    assert torch.equal(l2, loss.detach()) and torch.equal(c2, counts)
    return loss.detach(), counts, grad


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (1, 8, 2), (3, 2, 2), (17, 5, 3), (64, 64, 2),
                                   (255, 100, 7), (1000, 128, 8), (513, 161, 6), (77, 256, 4),
                                   (5000, 60, 4), (300, 255, 255)])
def test_matches_64_bits(n, e, k, masked, dtype):
    logits, idx, mask = inputs(n, e, k, dtype, masked, seed=n + e)
    check(logits, idx, mask, z=1e-2, scale=1024.0 if dtype == HF else 1.0)


def test_many_tokens_and_equal_bits():
    logits, idx, mask = inputs(70001, 128, 8, FP, True, seed=2)
    a = check(logits, idx, mask, 1e-3)
    b = check(logits, idx, mask, 1e-3)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [FP, BF])
def test_other_factors(dtype):
    logits, idx, mask = inputs(200, 24, 3, dtype, seed=3)
    check(logits, idx, mask, scale=0.01)
    check(logits, idx, mask, scale=1.0, go=0.25)
    check(logits, idx, mask, scale=8.0, go=3.0)


def test_strides_and_index_types():
    logits, idx, mask = inputs(90, 40, 4, BF, True, seed=4)
    wide = torch.zeros(90, 100, dtype=BF, device="cuda")
    wide[:, 3:43] = logits.cuda()
    check(logits, idx, mask, xg=wide[:, 3:43].detach().requires_grad_(True))
    check(logits, idx, mask, xg=logits.t().contiguous().cuda().t().detach().requires_grad_(True))
    check(logits, idx.int(), mask)
    check(logits, idx.t().contiguous().t(), mask)
    one = logits[:1].expand(90, 40)
    check(one, idx, mask, xg=one.cuda()[:1].expand(90, 40).detach().requires_grad_(True))


def test_masked_away_and_unused_slots():
    logits, idx, _ = inputs(50, 16, 4, FP, seed=5)
    loss, counts, grad = check(logits, idx, torch.zeros(50, dtype=torch.bool), 1e-3)
    assert loss == 0 and counts.sum() == 0 and torch.count_nonzero(grad) == 0
    idx[::3, 1:] = -1
    check(logits, idx, None, 1e-3)
    idx.fill_(-1)
    loss, counts, _ = check(logits, idx, None, 0.0)
    assert loss == 0 and counts.sum() == 0
    # padding may hold anything
    logits[7], logits[9] = float("nan"), float("inf")
    idx[:] = torch.arange(4)
    idx[7] = 10 ** 12
    mask = torch.ones(50, dtype=torch.bool)
    mask[[7, 9]] = False
    kept = logits.clone()
    kept[[7, 9]] = 0
    want, wcounts, wgrad, lb, gb = balance(kept, idx.clamp(max=15), mask, 1e-3)
    xg = logits.cuda().requires_grad_(True)
    loss, counts = fk.fused_moe_balance_loss(xg, idx.cuda(), mask.cuda(), 1e-3)
    loss.backward()
    assert torch.equal(counts.cpu(), wcounts)
    assert_within(loss, want, 2 * lb + half_step(FP) * want)
    assert_within(xg.grad, wgrad, 2 * gb + half_step(FP) * wgrad.abs())


@pytest.mark.parametrize("e", [8, 7, 100])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_even_load(e, dtype):
    """Every expert chosen by every token: f is 1/E, the loss 1 and the gradient nothing but 0.
    With one expert spared per token the gradient is all cancellation; it keeps its bits: 64
    roundings of p (f - 1/E) terms, not of p f ones."""
    logits, idx, _ = inputs(300, e, e, dtype, seed=e)
    loss, _, grad = check(logits, idx, None)
    assert loss == 1.0 and torch.count_nonzero(grad) == 0
    logits = logits.float()
    idx = logits.topk(e - 1, dim=1).indices
    _, _, grad = check(logits, idx, None)
    _, counts, want, _, _ = balance(logits, idx, None, 0.0)
    g = counts.double() / idx.numel() - 1 / e
    p = torch.softmax(logits.double(), 1)
    size = e / 300 * p * (g.abs() + (p * g.abs()).sum(1, keepdim=True))
    far = float(logits.abs().max())
    assert_within(grad, want, (64 + 4 * far) * 2.0 ** -24 * size)


def test_infinite_logits():
    logits, idx, _ = inputs(20, 12, 2, FP, seed=6)
    logits[:, 3] = -float("inf")  # an expert that is switched off
    logits[5] = -float("inf")
    check(logits, idx, None, 1e-2)
    logits[8, 2] = float("nan")
    xg = logits.cuda().requires_grad_(True)
    loss, _ = fk.fused_moe_balance_loss(xg, idx.cuda())
    loss.backward()
    assert torch.isnan(loss) and torch.isnan(xg.grad[8]).all()
    rows = [i for i in range(20) if i != 8]
    assert torch.isfinite(xg.grad[rows]).all()


def test_index_out_of_range_is_nan():
    logits, idx, _ = inputs(20, 12, 2, FP, seed=7)
    idx[4, 1] = 12
    xg = logits.cuda().requires_grad_(True)
    loss, _ = fk.fused_moe_balance_loss(xg, idx.cuda())
    loss.backward()
    assert torch.isnan(loss) and torch.isnan(xg.grad).all()


def test_gradient_against_differences():
    """Central differences in fp32, steps of 2^-6: third derivatives of a loss of order 1 over 6
    tokens are below 1 (error 2^-12 / 6), the loss's roundings give 2^-23 * 4 / 2^-5."""
    logits, idx, _ = inputs(6, 7, 2, FP, seed=8)
    _, _, grad = check(logits, idx, None, 0.05)
    for i in range(logits.numel()):
        ends = []
        for step in (2.0 ** -6, -2.0 ** -6):
            v = logits.clone()
            v.view(-1)[i] += step
            ends.append((float(fk.fused_moe_balance_loss(v.cuda(), idx.cuda(), None, 0.05)[0]),
                         float(v.view(-1)[i])))
        diff = (ends[0][0] - ends[1][0]) / (ends[0][1] - ends[1][1])
        assert abs(diff - float(grad.view(-1)[i])) <= 1.5e-4


def test_empty_batch():
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    loss, counts = fk.fused_moe_balance_loss(x, torch.zeros(0, 2, dtype=torch.long, device="cuda"))
    loss.backward()
    assert loss == 0 and counts.tolist() == [0] * 8 and x.grad.shape == (0, 8)


def test_second_backward_raises_and_refusals():
    logits, idx, mask = (t if t is None else t.cuda() for t in inputs(9, 8, 2, masked=True))
    x = logits.requires_grad_(True)
    loss, _ = fk.fused_moe_balance_loss(x, idx)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="handed over"):
        loss.backward()
    big = torch.zeros(9, 257, device="cuda")
    for a in ((big, idx), (x, idx[:8]), (x, idx[:, 0]), (x, idx[:, :0]), (x, idx.float()),
              (x, idx.cpu()), (x, idx, mask[:8]), (x, idx, mask.float()), (x, idx, mask.cpu()),
              (x[0], idx), (x.cpu(), idx.cpu())):
        with pytest.raises(AssertionError):
            fk.fused_moe_balance_loss(*a)
    with pytest.raises(AssertionError):
        fk.fused_moe_balance_loss(x, idx, loss_scale=0.0)
    with pytest.raises(TypeError):
        fk.fused_moe_balance_loss(x.double(), idx)


def test_follows_the_router_on_another_stream():
    logits, _, _ = inputs(500, 32, 4, BF, seed=9)
    side = torch.cuda.Stream()
    x = logits.cuda().requires_grad_(True)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w, idx = fk.fused_moe_route_v2(x, 4)
        loss, counts = fk.fused_moe_balance_loss(x, idx)
        (grad,) = torch.autograd.grad(loss, x)
    side.synchronize()
    want, wcounts, wgrad, lb, gb = balance(logits, idx.cpu(), None, 0.0)
    assert torch.equal(counts.cpu(), wcounts) and int(counts.sum()) == 2000
    assert_within(loss, want, lb + half_step(FP) * want)
    assert_within(grad, wgrad, gb + 1.01 * half_step(BF) * wgrad.abs() + tiny(BF))


def test_graph_replay_two_graphs():
    """Two captured graphs, replayed in turn on changing inputs."""
    sets = [inputs(300, 48, 4, FP, seed=s) for s in (10, 11)]
    state = []
    for logits, idx, _ in sets:
        x, i = logits.cuda().requires_grad_(True), idx.cuda()
        fk.fused_moe_balance_loss(x, i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, counts = fk.fused_moe_balance_loss(x, i, None, 1e-3)
            (grad,) = torch.autograd.grad(loss, x)
        state.append((g, x, i, loss, counts, grad))
    for turn in range(2):
        for j, (g, x, i, loss, counts, grad) in enumerate(state):
            logits, idx, _ = sets[(j + turn) % 2]
            with torch.no_grad():
                x.copy_(logits)
                i.copy_(idx)
        for g, *_ in state:
            g.replay()
        torch.cuda.synchronize()
        for j, (g, x, i, loss, counts, grad) in enumerate(state):
            logits, idx, _ = sets[(j + turn) % 2]
            want, wcounts, wgrad, lb, gb = balance(logits, idx, None, 1e-3)
            assert torch.equal(counts.cpu(), wcounts)
            assert_within(loss, want, lb + half_step(FP) * want)
            assert_within(grad, wgrad, gb + half_step(FP) * wgrad.abs())
