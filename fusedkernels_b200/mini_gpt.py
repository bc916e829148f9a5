"""Small GPT training harness wiring the fused ops into a model (end-to-end integration).

Mirrors fusedkernels' examples/train_mini_gpt.py (MiniGPT at train_mini_gpt.py:81-110 with
RMSNorm, a SwiGLU MLP and the cross-entropy loss, and the fused / native toggle of
train_mini_gpt.py:60-105): ``fused=True`` uses ``FusedRMSNorm``, ``fused_swiglu`` and
``fused_cross_entropy`` (gradient written in place over the logits); ``fused=False`` uses
the eager PyTorch formulation of the same ops.  Attention and the linear layers are
PyTorch's (SDPA / cuBLAS) in both modes.

Options beyond the reference's example, for the fused mode: ``fused_residual`` carries the
residual stream through ``FusedAddRMSNorm`` (the addition in front of every norm is part of
it), ``n_experts`` puts ``FusedMoEMLPSorted`` in the place of the MLPs, with the routers'
balance loss added to the loss, and a ``teacher`` (ids and logits of its top tokens) turns the
loss into ``fused_distillation_loss``.

``train_step`` runs forward, backward and an AdamW step; ``python -m
fusedkernels_b200.mini_gpt --mode fused`` prints tokens/s.  Under torchrun every rank trains
its own batch and DistributedDataParallel all-reduces the gradients of the replicated
parameters (data parallelism); tokens/s is then the sum over ranks.
"""
from __future__ import annotations

import argparse
import os
import time

import torch
import torch.nn as nn
import torch.nn.functional as F

from .cross_entropy import fused_cross_entropy
from .distillation import fused_distillation_loss
from .moe_layer_sorted import FusedMoEMLPSorted
from .rmsnorm import FusedAddRMSNorm, FusedRMSNorm
from .swiglu import fused_swiglu


class RefRMSNorm(nn.Module):
    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x):
        var = x.float().pow(2).mean(-1, keepdim=True)
        return (x.float() * torch.rsqrt(var + self.eps) * self.weight.float()).to(x.dtype)


class CausalSelfAttention(nn.Module):
    def __init__(self, dim, n_heads):
        super().__init__()
        self.n_heads = n_heads
        self.head_dim = dim // n_heads
        self.qkv = nn.Linear(dim, 3 * dim, bias=False)
        self.proj = nn.Linear(dim, dim, bias=False)

    def forward(self, x):
        B, T, D = x.shape
        qkv = self.qkv(x).view(B, T, 3, self.n_heads, self.head_dim).permute(2, 0, 3, 1, 4)
        out = F.scaled_dot_product_attention(qkv[0], qkv[1], qkv[2], is_causal=True)
        return self.proj(out.transpose(1, 2).reshape(B, T, D))


class MLP(nn.Module):
    def __init__(self, dim, hidden_dim, fused: bool):
        super().__init__()
        self.fused = fused
        self.w_gate = nn.Linear(dim, hidden_dim, bias=False)
        self.w_up = nn.Linear(dim, hidden_dim, bias=False)
        self.w_down = nn.Linear(hidden_dim, dim, bias=False)

    def forward(self, x):
        g, u = self.w_gate(x), self.w_up(x)
        return self.w_down(fused_swiglu(g, u) if self.fused else F.silu(g) * u)


class Block(nn.Module):
    fused_residual = False  # of a model that was pickled before it had the option

    def __init__(self, dim, n_heads, hidden_dim, fused: bool, fused_residual: bool = False,
                 n_experts: int = 0, k: int = 2, balance_coef: float = 0.0):
        super().__init__()
        Norm = FusedAddRMSNorm if fused_residual else FusedRMSNorm if fused else RefRMSNorm
        self.fused_residual = fused_residual
        self.norm1, self.norm2 = Norm(dim), Norm(dim)
        self.attn = CausalSelfAttention(dim, n_heads)
        self.mlp = (FusedMoEMLPSorted(dim, hidden_dim, n_experts, k, balance_coef=balance_coef)
                    if n_experts else MLP(dim, hidden_dim, fused))

    def forward(self, x, residual=None):
        if self.fused_residual:  # (what the block before it put out, the stream so far)
            y, residual = self.norm1(x, residual)
            y, residual = self.norm2(self.attn(y), residual)
            return self.mlp(y), residual
        x = x + self.attn(self.norm1(x))
        return x + self.mlp(self.norm2(x))


class MiniGPT(nn.Module):
    fused_residual, n_experts = False, 0  # of a model that was pickled before it had the options

    def __init__(self, vocab_size=32000, dim=1024, n_layers=12, n_heads=16, hidden_dim=2752,
                 max_seq_len=1024, fused: bool = True, fused_residual: bool = False,
                 n_experts: int = 0, moe_k: int = 2, balance_coef: float = 0.01):
        super().__init__()
        assert fused or not (fused_residual or n_experts), "options of the fused mode"
        self.fused = fused
        self.fused_residual = fused_residual
        self.n_experts = n_experts
        self.tok_emb = nn.Embedding(vocab_size, dim)
        self.pos_emb = nn.Embedding(max_seq_len, dim)
        self.blocks = nn.ModuleList([
            Block(dim, n_heads, hidden_dim, fused, fused_residual, n_experts, moe_k, balance_coef)
            for _ in range(n_layers)])
        self.norm_f = (FusedAddRMSNorm if fused_residual else FusedRMSNorm if fused
                       else RefRMSNorm)(dim)
        self.lm_head = nn.Linear(dim, vocab_size, bias=False)

    def logits(self, idx):
        """Logits [B * T, vocab_size] of a batch of tokens."""
        B, T = idx.shape
        if self.n_experts:
            for blk in self.blocks:  # a later block's would keep the graph of the earlier ones
                blk.mlp.balance_loss = None
        x = self.tok_emb(idx) + self.pos_emb(torch.arange(T, device=idx.device))[None]
        if self.fused_residual:
            residual = None
            for blk in self.blocks:
                x, residual = blk(x, residual)
            x, _ = self.norm_f(x, residual)
        else:
            for blk in self.blocks:
                x = blk(x)
            x = self.norm_f(x)
        return self.lm_head(x).reshape(B * T, -1)

    def balance_loss(self):
        """Sum of the MoE blocks' balance losses of the last forward (0 where none asks, and for a
        model without MoE blocks)."""
        losses = [getattr(b.mlp, "balance_loss", None) for b in self.blocks]
        return sum(x for x in losses if x is not None)

    @torch.no_grad()
    def top_logits(self, idx, k):
        """The k largest logits per position and their ids, as a teacher's: ([B * T, k] int64,
        [B * T, k])."""
        values, ids = self.logits(idx).topk(k, dim=1)
        return ids, values

    def forward(self, idx, targets, teacher=None, temperature=1.0, hard_weight=0.5):
        logits = self.logits(idx)
        t = targets.reshape(-1)
        if not self.fused:
            assert teacher is None, "a teacher needs the fused mode"
            return F.cross_entropy(logits.float(), t)
        if teacher is None:
            loss = fused_cross_entropy(logits, t, inplace_grad=True)
        else:
            loss = fused_distillation_loss(logits, *teacher, targets=t, temperature=temperature,
                                           hard_weight=hard_weight, inplace_grad=True)
        return loss + self.balance_loss() if self.n_experts else loss


def train_step(model, opt, x, y, teacher=None):
    loss = model(x, y) if teacher is None else model(x, y, teacher)
    loss.backward()
    opt.step()
    opt.zero_grad(set_to_none=True)
    return loss


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--mode", choices=["fused", "native"], default="fused")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=5)
    ap.add_argument("--batch-size", type=int, default=8)
    ap.add_argument("--seq-len", type=int, default=1024)
    ap.add_argument("--dim", type=int, default=1024)
    ap.add_argument("--layers", type=int, default=12)
    ap.add_argument("--fused-residual", action="store_true",
                    help="carry the residual stream through FusedAddRMSNorm")
    ap.add_argument("--experts", type=int, default=0,
                    help="MoE blocks with this many experts instead of the MLPs")
    ap.add_argument("--distill", type=int, default=0, metavar="K",
                    help="distil from the top K logits of a second model of the same shape")
    args = ap.parse_args()
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    dev = torch.device("cuda", int(os.environ.get("LOCAL_RANK", "0")))
    torch.cuda.set_device(dev)
    if world > 1:
        torch.distributed.init_process_group("nccl", device_id=dev)
    torch.manual_seed(0)  # identical initial weights on every rank
    hidden = args.dim * 43 // 16
    cfg = dict(dim=args.dim, n_layers=args.layers, max_seq_len=args.seq_len,
               hidden_dim=hidden // 64 * 64 if args.experts else hidden,
               fused=args.mode == "fused", fused_residual=args.fused_residual,
               n_experts=args.experts)
    model = MiniGPT(**cfg).to(dev, torch.bfloat16)
    teacher = MiniGPT(**cfg).to(dev, torch.bfloat16) if args.distill else None
    V = model.lm_head.out_features

    def step(x, y):
        return train_step(model, opt, x, y, teacher.top_logits(x, args.distill) if teacher else None)

    if world > 1:
        model = torch.nn.parallel.DistributedDataParallel(model, device_ids=[dev.index])
    opt = torch.optim.AdamW(model.parameters(), lr=3e-4)
    torch.manual_seed(1000 + rank)  # each rank draws its own batches
    for _ in range(args.warmup):
        idx = torch.randint(0, V, (args.batch_size, args.seq_len + 1), device=dev)
        step(idx[:, :-1], idx[:, 1:])
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(args.steps):
        idx = torch.randint(0, V, (args.batch_size, args.seq_len + 1), device=dev)
        loss = step(idx[:, :-1], idx[:, 1:])
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    if world > 1:
        t = torch.tensor([dt], device=dev)
        torch.distributed.all_reduce(t, op=torch.distributed.ReduceOp.MAX)
        dt = float(t.item())
    if rank == 0:
        tok = world * args.steps * args.batch_size * args.seq_len
        print(f"mode={args.mode} ranks={world} tokens/s={tok / dt:,.0f} loss={loss.item():.4f}")
    if world > 1:
        torch.distributed.destroy_process_group()


if __name__ == "__main__":
    main()
