"""MiniGPT with the residual stream through FusedAddRMSNorm, MoE blocks with their balance loss
and a teacher's top logits: the operators together, as a training step uses them.

The whole step is restated in 64 bits on the CPU (plain autograd) and every parameter's gradient
compared.  The model runs in fp32: about 20 operations deep, each within 2^-20 of the norm of its
result (3xTF32 products 2^-21, sums of at most 320 terms), 20 * 2^-20 = 2e-5 of a gradient's
norm, taken five times for cancellation between branches: 1e-4."""
import copy
import os
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F

from fusedkernels_b200 import FusedMoEMLPSorted
from fusedkernels_b200.mini_gpt import MiniGPT, train_step

pytestmark = pytest.mark.gpu
CFG = dict(vocab_size=500, dim=128, n_layers=2, n_heads=4, hidden_dim=192, max_seq_len=32)
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def make(seed=0, **kw):
    torch.manual_seed(seed)
    return MiniGPT(**CFG, **kw).cuda()


def batch(seed=1, rows=3, length=32):
    G = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, CFG["vocab_size"], (rows, length + 1), generator=G)
    return idx[:, :-1].contiguous(), idx[:, 1:].contiguous()


def reference_step(model, x, y, teacher, temperature, hard_weight, n_experts, k, coef):
    """The loss and every parameter's gradient in 64 bits."""
    P = {n: p.detach().cpu().double().requires_grad_(True) for n, p in model.named_parameters()}

    def norm(h, name):
        return h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + 1e-6) * P[name]

    B, T = x.shape
    h = P["tok_emb.weight"][x] + P["pos_emb.weight"][:T][None]
    balance = 0.0
    for i in range(CFG["n_layers"]):
        b = f"blocks.{i}."
        a = norm(h, b + "norm1.weight")
        qkv = (a @ P[b + "attn.qkv.weight"].T).view(B, T, 3, CFG["n_heads"], -1).permute(2, 0, 3, 1, 4)
        o = F.scaled_dot_product_attention(qkv[0], qkv[1], qkv[2], is_causal=True)
        h = h + o.transpose(1, 2).reshape(B, T, -1) @ P[b + "attn.proj.weight"].T
        a = norm(h, b + "norm2.weight").reshape(B * T, -1)
        if n_experts:
            logits = a @ P[b + "mlp.router.weight"].T
            top, idx = logits.topk(k, dim=1)
            w = torch.softmax(top, 1)
            out = torch.zeros_like(a)
            for e in range(n_experts):
                m = b + f"mlp.experts.{e}."
                act = F.silu(a @ P[m + "w_gate.weight"].T) * (a @ P[m + "w_up.weight"].T)
                we = (w * (idx == e)).sum(1, keepdim=True)
                out = out + we * (act @ P[m + "w_down.weight"].T)
            f = torch.bincount(idx.reshape(-1), minlength=n_experts).double() / idx.numel()
            balance = balance + coef * n_experts * (f * torch.softmax(logits, 1).mean(0)).sum()
        else:
            m = b + "mlp."
            act = F.silu(a @ P[m + "w_gate.weight"].T) * (a @ P[m + "w_up.weight"].T)
            out = act @ P[m + "w_down.weight"].T
        h = h + out.view(B, T, -1)
    logits = norm(h, "norm_f.weight").reshape(B * T, -1) @ P["lm_head.weight"].T
    loss = F.cross_entropy(logits, y.reshape(-1))
    if teacher is not None:
        ids, top = (t.cpu() for t in teacher)
        p = torch.softmax(top.double() / temperature, 1)
        logq = torch.log_softmax(logits / temperature, 1).gather(1, ids)
        soft = (p * (p.log() - logq)).sum(1).mean() * temperature ** 2
        loss = hard_weight * loss + (1 - hard_weight) * soft
    loss = loss + balance
    loss.backward()
    return loss.detach(), {n: p.grad for n, p in P.items()}


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n_experts", [0, 4])
@pytest.mark.parametrize("distil", [False, True])
def test_gradients_of_a_step(residual, n_experts, distil):
    model = make(fused_residual=residual, n_experts=n_experts, balance_coef=0.05)
    x, y = batch()
    teacher = make(seed=9).top_logits(x.cuda(), 16) if distil else None
    args = (teacher, 2.0, 0.3) if distil else ()
    loss = model(x.cuda(), y.cuda(), *args)
    loss.backward()
    want, grads = reference_step(model, x, y, teacher, 2.0, 0.3, n_experts, 2, 0.05)
    assert abs(float(loss) - float(want)) <= 1e-4 * abs(float(want))
    for n, p in model.named_parameters():
        g = grads[n] if grads[n] is not None else torch.zeros(p.shape, dtype=torch.float64)
        off = (p.grad.cpu().double() - g).norm()
        assert off <= 1e-4 * g.norm() + 1e-12, (n, float(off / g.norm()))


def test_residual_form_is_the_plain_model_in_bf16():
    """bf16: the carried stream rounds where the additions did, so the losses are equal but for
    the library products' own order (none here: same shapes, same calls)."""
    a, b = make(fused_residual=False).bfloat16(), make(fused_residual=True).bfloat16()
    assert all(torch.equal(p, q) for p, q in zip(a.state_dict().values(), b.state_dict().values()))
    x, y = (t.cuda() for t in batch())
    with torch.no_grad():
        la, lb = a(x, y), b(x, y)
    assert abs(float(la) - float(lb)) <= 2 ** -8 * abs(float(la))


def test_training_steps_with_everything():
    model = make(fused_residual=True, n_experts=4).bfloat16()
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    x, y = (t.cuda() for t in batch())
    teacher = make(seed=9).bfloat16().top_logits(x, 8)
    for _ in range(3):
        assert torch.isfinite(train_step(model, opt, x, y, teacher))
    counts = [blk.mlp.expert_counts for blk in model.blocks]
    assert all(int(c.sum()) == x.numel() * 2 and c.dtype == torch.int64 for c in counts)


def test_layer_attributes():
    layer = FusedMoEMLPSorted(64, 64, 4, 2).cuda()
    x = torch.randn(8, 64, device="cuda")
    layer(x)
    assert layer.balance_loss is None and layer.expert_counts is None
    layer = FusedMoEMLPSorted(64, 64, 4, 2, balance_coef=0.01, z_coef=0.001).cuda()
    out = layer(x)
    assert layer.balance_loss.requires_grad and layer.balance_loss.ndim == 0
    twin = copy.deepcopy(layer)  # after a forward, before its backward
    assert twin.balance_loss is None and torch.equal(twin(x), out)
    (out.sum() + layer.balance_loss).backward()
    with torch.no_grad():
        layer(x)
    assert not layer.balance_loss.requires_grad
    with pytest.raises(AssertionError):
        FusedMoEMLPSorted(64, 64, 4, 2, z_coef=0.1)


def test_fp16_layer_keeps_its_balance_gradient():
    """The gradient of a mean over 4096 tokens, times 0.01, is below fp16's smallest step where
    the loss scaler's factor comes after its rounding; here that factor comes first.  Bound: the
    fp16 products of the router's backward (half_step 2^-11 per factor, three of them) over sums
    of 4096 terms."""
    layer = FusedMoEMLPSorted(64, 64, 8, 2, balance_coef=0.01).cuda().half()
    x = torch.randn(4096, 64, device="cuda").half()
    layer(x)
    (layer.balance_loss * 65536.0).backward()
    xd = x.double().cpu()
    logits = (x @ layer.router.weight.T).detach().double().cpu()  # the layer's own, rounded
    idx = logits.sort(dim=1, descending=True, stable=True).indices[:, :2]  # fp16 logits tie
    assert torch.equal(torch.bincount(idx.reshape(-1), minlength=8), layer.expert_counts.cpu())
    f = torch.bincount(idx.reshape(-1), minlength=8).double() / idx.numel()
    p = torch.softmax(logits, 1)
    dlogits = 65536 * 0.01 * 8 / 4096 * p * (f - (p * f).sum(1, keepdim=True))
    want = dlogits.T @ xd
    size = dlogits.abs().T @ xd.abs()
    got = layer.router.weight.grad.double().cpu()
    assert torch.count_nonzero(got) == got.numel()
    assert ((got - want).abs() <= 3 * 2 ** -11 * size + 2 ** -24).all()


def test_command_line():
    cmd = [sys.executable, "-m", "fusedkernels_b200.mini_gpt", "--steps", "2", "--warmup", "1",
           "--batch-size", "2", "--seq-len", "64", "--dim", "128", "--layers", "2",
           "--fused-residual", "--experts", "4", "--distill", "8"]
    r = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "mode=fused" in r.stdout and "loss=nan" not in r.stdout


def test_no_second_derivatives():
    """A backward pass with create_graph gives the gradient; a derivative of it is refused."""
    from fusedkernels_b200 import (fused_add_rms_norm, fused_distillation_loss,
                                   fused_moe_balance_loss)
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda")
    idx = torch.arange(12, device="cuda").view(6, 2) % 32
    top = torch.randn(6, 2, device="cuda")
    for loss in (fused_add_rms_norm(x, x.detach(), w)[0].sum(), fused_moe_balance_loss(x, idx)[0],
                 fused_distillation_loss(x, idx, top)):
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.square().sum().backward()


def captured_and_eager(step, params):
    """Gradients of `step` run eagerly on the default stream, then captured and replayed."""
    step()
    eager = [p.grad.clone() for p in params]
    for p in params:
        p.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for p in params:
        p.grad.zero_()
    graph.replay()
    torch.cuda.synchronize()
    return eager, [p.grad for p in params], graph


@pytest.mark.parametrize("backward", [True, False])
def test_layer_keeps_no_graph(backward):
    """After an eager step nothing of its graph lives on, so the next one can be captured."""
    layer = FusedMoEMLPSorted(64, 64, 4, 2, balance_coef=0.01).cuda()
    x = torch.randn(32, 64, device="cuda")
    params = list(layer.parameters())

    def step():
        out = layer(x)
        (out.square().mean() + layer.balance_loss).backward()

    layer(x)
    if backward:
        step()
        assert layer.balance_loss.grad_fn is None and not layer.balance_loss.requires_grad
        assert float(layer.balance_loss) > 0.0
        for p in params:
            p.grad = None
    eager, replayed, _ = captured_and_eager(step, params)
    for a, b in zip(eager, replayed):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-8)


def test_model_step_is_captured_after_an_eager_one():
    model = make(fused_residual=True, n_experts=4)
    x, y = (t.cuda() for t in batch())
    params = list(model.parameters())

    def step():
        model(x, y).backward()

    eager, replayed, graph = captured_and_eager(step, params)
    for a, b in zip(eager, replayed):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-7)
    assert float(model.balance_loss()) > 0.0
    with torch.enable_grad():
        model.logits(x)  # a forward alone, whose graph lives in the blocks
    for p in params:
        p.grad = None
    captured_and_eager(step, params)
