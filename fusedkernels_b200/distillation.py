"""Distillation loss from a teacher's top logits, alone or mixed with the hard label.

A teacher's full logits are too large to store; what is kept per row is its top k, ids and
logits.  Over the used slots of a row (id >= 0), with temperature T and s the student's row:

    p = softmax(teacher / T) over the slots,   q = softmax(s / T) over the vocabulary
    soft = T^2 * KL(p || q) = T^2 * sum_j p_j (log p_j - log q_{id_j})
    row  = (1 - hard_weight) * soft + hard_weight * (logsumexp(s) - s_target)
    loss = mean of row over the counted rows

``fk_distill`` gives the loss and its gradient with each logit read from memory once and its
gradient written once, as ``fused_cross_entropy`` does; the two losses share that pass.
"""
import torch

from . import _lib

MAX_SLOTS = 1024
_last_err = None


def _distill(logits, teacher_idx, teacher_logits, targets, temperature, hard_weight,
             ignore_index, inplace_grad, loss_scale, want_grad):
    """loss and (want_grad) the gradient of loss * loss_scale."""
    global _last_err
    n_rows, n_cols = logits.shape
    x, stride = _lib.rows_of(logits, n_cols)
    idx = teacher_idx.to(torch.int64).contiguous()
    top = teacher_logits.contiguous()
    if targets is not None:
        targets = targets.to(torch.int64).contiguous()
    grad, grad_stride = None, n_cols
    if want_grad:
        if inplace_grad:
            grad, grad_stride = x, stride
        else:
            grad = x.new_empty((n_rows, n_cols))
    loss = x.new_empty((), dtype=torch.float32)
    err = x.new_empty(1, dtype=torch.int32)
    k = idx.shape[1]
    size = _lib.workspace_bytes("fk_distill_workspace_size", logits.device, n_rows, k)
    ws = x.new_empty(size, dtype=torch.uint8)
    with _lib.on_device(logits):
        _lib.call("fk_distill", x.data_ptr(), stride, _lib.ptr(grad), grad_stride,
                  idx.data_ptr(), top.data_ptr(), _lib.dtype_code(top.dtype), k,
                  _lib.ptr(targets), n_rows, n_cols, ignore_index, temperature, hard_weight,
                  loss_scale, _lib.dtype_code(x.dtype), loss.data_ptr(), err.data_ptr(),
                  ws.data_ptr(), size, _lib.stream_of(logits))
    _last_err = err
    return loss, grad


class _FusedDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args):
        loss, ctx.grad = _distill(logits, *args, True)
        ctx.loss_scale = args[-1]
        return loss

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, grad_output):
        return _lib.hand_over_gradient(ctx, grad_output), None


def fused_distillation_loss(logits: torch.Tensor, teacher_idx: torch.Tensor,
                            teacher_logits: torch.Tensor, targets: torch.Tensor | None = None,
                            temperature: float = 1.0, hard_weight: float = 0.5,
                            ignore_index: int = -100, inplace_grad: bool = False,
                            loss_scale: float = 1.0) -> torch.Tensor:
    """Scalar mean loss of the student's logits [N, V] against a teacher's top logits (see
    the module's docstring).

    teacher_idx, teacher_logits: [N, k], k <= 1024, in any order.  A negative id is an unused
    slot; an id that stands twice counts as two entries; logits of -inf have probability 0.  A
    row with no used slot, or none above -inf, has no soft part.
    targets: [N] hard labels.  With them the counted rows are those whose target is not
    ignore_index, and hard_weight mixes the two parts; without them the counted rows are those
    that hold a teacher, and the loss is the soft part alone (hard_weight is not used).
    With hard_weight 1 (or 0) the soft (hard) part is left out, whatever the teacher's logits hold.
    inplace_grad=True writes the gradient over the logits buffer, as in fused_cross_entropy;
    where no gradient is wanted the logits are left as they are.
    loss_scale: the factor that the backward pass will be started with (a GradScaler's scale).
    It is folded into the gradient in 32 bits, before the rounding to the logits' dtype; any
    other factor gives the right gradient too, at one more pass over it and within what the
    logits' dtype held before (in fp16 what has overflowed or vanished stays so).  The returned
    loss is not scaled.  The gradient is handed over once: a second backward pass through the same
    graph raises.

    A teacher id or target >= V (or a negative target that is not ignore_index) makes the loss
    and that row's gradient NaN; ``last_distillation_error()`` reads the flag."""
    assert logits.is_cuda and logits.ndim == 2 and logits.shape[1] >= 1
    n_rows = logits.shape[0]
    assert teacher_idx.ndim == 2 and teacher_idx.shape == teacher_logits.shape
    assert teacher_idx.shape[0] == n_rows and 1 <= teacher_idx.shape[1] <= MAX_SLOTS, \
        f"the teacher has one row of 1..{MAX_SLOTS} slots for each row of logits"
    assert teacher_idx.dtype in (torch.int64, torch.int32)
    assert teacher_idx.device == logits.device and teacher_logits.device == logits.device
    assert not teacher_logits.requires_grad and not _lib.has_tangent(teacher_logits), \
        "the teacher gets no gradient: detach its logits"
    if targets is not None:
        assert targets.shape == (n_rows,) and targets.device == logits.device
        assert not targets.is_floating_point()
    assert 0.0 < temperature < float("inf") and 0.0 <= hard_weight <= 1.0
    assert 0.0 < loss_scale < float("inf")
    args = (teacher_idx, teacher_logits, targets, float(temperature), float(hard_weight),
            int(ignore_index), inplace_grad, float(loss_scale))
    if _lib.wants_derivative(logits):
        return _FusedDistillation.apply(logits, args)
    return _distill(logits, *args, False)[0]


def last_distillation_error() -> int:
    """Device error flag of the last fused_distillation_loss call: 0 ok, 1 an id or target was
    out of range.  Synchronises."""
    return 0 if _last_err is None else int(_last_err.item())
