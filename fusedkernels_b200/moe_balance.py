"""Balance loss of a routed layer, with the per-expert counts.

For router logits [N, E] and the experts that the router chose, idx [N, k]:

    counts_e = number of slots that name expert e,   f_e = counts_e / sum(counts)
    p_t = softmax(logits_t),  P_e = mean over the tokens of p_te
    loss = E * sum_e f_e P_e + z_coef * mean over the tokens of logsumexp(logits_t)^2

The first part is smallest where load and probability are spread evenly (1 there), the
second keeps the logits from growing.  The gradient goes through P and the logsumexp; the
counts have none.  ``fk_moe_balance`` counts the slots, then reads each logit once and writes
its gradient with the loss, so the backward pass launches nothing but the check of
grad_output.
"""
import torch

from . import _lib
from .moe_routing_v2 import MAX_EXPERTS


def _balance(logits, topk_idx, token_mask, z_coef, loss_scale, want_grad):
    """loss, counts and (want_grad) the gradient of loss * loss_scale."""
    n_rows, n_experts = logits.shape
    x, stride = _lib.rows_of(logits, n_experts)
    idx = topk_idx.to(torch.int64).contiguous()
    mask = None if token_mask is None else token_mask.contiguous()
    grad = x.new_empty((n_rows, n_experts)) if want_grad else None
    counts = x.new_empty(n_experts, dtype=torch.int64)
    loss = x.new_empty((), dtype=torch.float32)
    size = _lib.workspace_bytes("fk_moe_balance_workspace_size", logits.device)
    ws = x.new_empty(size, dtype=torch.uint8)
    with _lib.on_device(logits):
        _lib.call("fk_moe_balance", x.data_ptr(), stride, idx.data_ptr(), _lib.ptr(mask), n_rows,
                  n_experts, idx.shape[1], z_coef, loss_scale, _lib.ptr(grad), counts.data_ptr(),
                  loss.data_ptr(), ws.data_ptr(), size, _lib.dtype_code(x.dtype),
                  _lib.stream_of(logits))
    return loss, counts, grad


class _FusedMoEBalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args):
        loss, counts, ctx.grad = _balance(logits, *args, True)
        ctx.loss_scale = args[-1]
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, grad_output, _counts):
        return None if grad_output is None else _lib.hand_over_gradient(ctx, grad_output), None


def fused_moe_balance_loss(router_logits: torch.Tensor, topk_idx: torch.Tensor,
                           token_mask: torch.Tensor | None = None, z_coef: float = 0.0,
                           loss_scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Balance loss of one routing and its per-expert counts: ``(loss, counts)``, a scalar
    fp32 loss (see the module's docstring) and int64 counts [E].

    router_logits: [N, E] fp32, fp16 or bf16, E <= 256.  topk_idx: [N, k] expert indices as
    the routers return them; a negative one is an unused slot, one >= E in a counted token makes
    the loss and the whole gradient NaN.  token_mask: [N] bool; tokens that are False (padding)
    count nowhere and get a zero gradient.  With no counted token the loss is 0.  A token whose
    logits are all -inf has no probabilities: it adds 0 to both sums.

    loss_scale: the factor that the backward pass will be started with (a GradScaler's scale,
    or the weight the loss is added with).  It is folded into the gradient in 32 bits, before
    the rounding to the logits' dtype; any other factor gives the right gradient too, at one
    more pass over it and within what the logits' dtype held before (in fp16 what has overflowed
    or vanished stays so).  The returned loss is not scaled.  The gradient is handed over once: a
    second backward pass through the same graph raises."""
    assert router_logits.is_cuda and router_logits.ndim == 2
    n_rows, n_experts = router_logits.shape
    assert 1 <= n_experts <= MAX_EXPERTS, f"n_experts={n_experts} outside 1..{MAX_EXPERTS}"
    assert topk_idx.ndim == 2 and topk_idx.shape[0] == n_rows and topk_idx.shape[1] >= 1
    assert topk_idx.dtype in (torch.int64, torch.int32) and topk_idx.device == router_logits.device
    if token_mask is not None:
        assert token_mask.shape == (n_rows,) and token_mask.dtype == torch.bool
        assert token_mask.device == router_logits.device
    assert 0.0 < loss_scale < float("inf")
    args = (topk_idx, token_mask, float(z_coef), float(loss_scale))
    if _lib.wants_derivative(router_logits):
        return _FusedMoEBalanceLoss.apply(router_logits, args)
    return _balance(router_logits, *args, False)[:2]
