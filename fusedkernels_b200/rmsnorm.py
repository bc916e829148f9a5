"""Fused RMSNorm forward + backward.

Mirrors fusedkernels/rmsnorm.py (``_FusedRMSNormFn`` at rmsnorm.py:74-113,
``FusedRMSNorm`` at rmsnorm.py:116-125): y = x * rsqrt(mean(x^2) + eps) * weight with
fp32 accumulation, output in x's dtype, weight an fp32 ``ones`` parameter by default and
its gradient returned in the weight's dtype.  The weight gradient is reduced on the
device in a fixed order (per-CTA partial rows + a column reduce), replacing the
[rows, cols] fp32 partial and torch ``.sum(0)`` of rmsnorm.py:104 and :112.
"""
import torch
import torch.nn as nn

from . import _lib


class _FusedRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        assert x.is_cuda and weight.is_cuda
        orig_shape = x.shape
        x2 = x.reshape(-1, orig_shape[-1]).contiguous()
        n_rows, n_cols = x2.shape
        assert weight.numel() == n_cols
        w = weight.contiguous()
        y = torch.empty_like(x2)
        rstd = torch.empty(n_rows, dtype=torch.float32, device=x.device)
        _lib.call("fk_rmsnorm_fwd", x2.data_ptr(), n_cols, w.data_ptr(),
                  _lib.dtype_code(w.dtype), y.data_ptr(), n_cols, rstd.data_ptr(), n_rows,
                  n_cols, float(eps), _lib.dtype_code(x2.dtype), _lib.stream_of(x2))
        ctx.save_for_backward(x2, w, rstd)
        ctx.orig_shape = orig_shape
        ctx.weight_shape = weight.shape
        return y.reshape(orig_shape)

    @staticmethod
    def backward(ctx, dy):
        x, w, rstd = ctx.saved_tensors
        n_rows, n_cols = x.shape
        dy2 = dy.reshape(-1, n_cols).to(x.dtype).contiguous()
        dx = torch.empty_like(x)
        dw = torch.empty(n_cols, dtype=w.dtype, device=x.device)
        ws_bytes = _lib.rmsnorm_bwd_workspace_bytes(n_rows, n_cols, x.device)
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=x.device)
        _lib.call("fk_rmsnorm_bwd", dy2.data_ptr(), x.data_ptr(), w.data_ptr(),
                  _lib.dtype_code(w.dtype), rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                  ws.data_ptr(), ws.numel(), n_rows, n_cols, _lib.dtype_code(x.dtype),
                  _lib.stream_of(x))
        return dx.reshape(ctx.orig_shape), dw.reshape(ctx.weight_shape), None


class FusedRMSNorm(nn.Module):
    """Drop-in replacement for LlamaRMSNorm / nn.RMSNorm."""

    def __init__(self, hidden_size: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _FusedRMSNormFn.apply(x, self.weight, self.eps)


# ---------------------------------------------------------------- with the residual's addition
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _check_add_norm(x, residual, weight):
    assert x.is_cuda and x.ndim >= 1 and weight.device == x.device
    assert x.dtype in _FLOATS and weight.dtype in _FLOATS, "fp32, fp16 or bf16 tensors"
    assert weight.numel() == x.shape[-1] >= 1
    if residual is not None:
        assert residual.shape == x.shape, "residual and x have one shape (nothing is broadcast)"
        assert residual.device == x.device
        assert residual.dtype is x.dtype or residual.dtype is torch.float32, \
            "the residual has x's dtype or fp32"


def _add_norm(x, residual, w, eps, save):
    """y, h and (save) rstd."""
    n_cols = x.shape[-1]
    n_rows = x.numel() // n_cols
    x2, xs = _lib.rows_of(x, n_cols)
    r2, rs = _lib.rows_of(residual, n_cols)
    y = x.new_empty(x.shape)  # (new_empty: the cheapest of torch's allocating calls)
    h = residual.new_empty(x.shape)
    rstd = x.new_empty(n_rows, dtype=torch.float32) if save else None
    code = _lib._DTYPE_CODES
    with _lib.on_device(x):
        _lib.call("fk_add_rmsnorm_fwd", x2.data_ptr(), xs, r2.data_ptr(), rs, code[h.dtype],
                  w.data_ptr(), code[w.dtype], y.data_ptr(), h.data_ptr(), _lib.ptr(rstd), n_rows,
                  n_cols, eps, code[y.dtype], _lib.stream_of(x))
    return y, h, rstd


class _FusedAddRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        w = weight.contiguous()
        y, h, rstd = _add_norm(x, residual, w, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, w, rstd)
        ctx.x_dtype = x.dtype
        ctx.weight_shape = weight.shape
        return y, h

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy, dh):
        h, w, rstd = ctx.saved_tensors
        n_cols = h.shape[-1]
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if dy is None:  # only the sum was used: its gradient passes through
            if dh is None:
                return None, None, None, None
            return (dh.to(ctx.x_dtype) if need_x else None, dh if need_r else None,
                    torch.zeros(ctx.weight_shape, dtype=w.dtype, device=w.device)
                    if need_w else None, None)
        dy2, dys = _lib.rows_of(dy, n_cols)
        dh2, dhs = (None, 0) if dh is None else _lib.rows_of(dh, n_cols)
        n_rows = h.numel() // n_cols
        dx = h.new_empty(h.shape, dtype=ctx.x_dtype)
        dr = dx if h.dtype == ctx.x_dtype else h.new_empty(h.shape)
        dw = w.new_empty(ctx.weight_shape)
        size = _lib.workspace_bytes("fk_add_rmsnorm_bwd_workspace_size", h.device, n_rows,
                                    n_cols)
        ws = h.new_empty(size, dtype=torch.uint8)
        code = _lib._DTYPE_CODES
        with _lib.on_device(h):
            _lib.call("fk_add_rmsnorm_bwd", dy2.data_ptr(), dys, _lib.ptr(dh2), dhs, h.data_ptr(),
                      code[h.dtype], w.data_ptr(), code[w.dtype], rstd.data_ptr(), dx.data_ptr(),
                      None if dr is dx else dr.data_ptr(), dw.data_ptr(), ws.data_ptr(), size,
                      n_rows, n_cols, code[dx.dtype], _lib.stream_of(h))
        return dx if need_x else None, dr if need_r else None, dw if need_w else None, None


def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                       eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual`` and ``y = h * rsqrt(mean(h^2) + eps) * weight`` in one pass over
    the last dimension; returns ``(y, h)``, ``y`` in x's dtype and ``h`` in the residual's
    (x's dtype, or fp32 for a residual stream kept in 32 bits).

    The norm is that of the rounded ``h``, so the result is that of the addition followed by
    ``FusedRMSNorm``; in the backward pass the gradient that arrives at ``h`` is added in 32
    bits before the one rounding of the inputs' gradient."""
    assert residual is not None, "without a residual there is nothing to add: call FusedRMSNorm"
    _check_add_norm(x, residual, weight)
    if _lib.wants_derivative(x, residual, weight):
        return _FusedAddRMSNormFn.apply(x, residual, weight, float(eps))
    return _add_norm(x, residual, weight.contiguous(), float(eps), False)[:2]


def fused_add_rms_norm_quant(x: torch.Tensor, residual: torch.Tensor | None,
                             weight: torch.Tensor, eps: float = 1e-6, block: int | None = None
                             ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """RMSNorm of ``h = x + residual`` (of ``x`` itself where residual is None) with its
    output in 8 bits: returns ``(q, scales, h)``, ``q`` float8_e4m3fn of x's shape with
    ``y ~ q * scales``.

    ``block=None`` gives one fp32 scale per row (scales [..., 1]), ``block=128`` one per 128
    columns (scales [..., ceil(cols / 128)]): max|y| / 448 over the group, at least 2^-126.  The
    32-bit ``y`` is quantised, so it is rounded once; quotients that are ties of e4m3 in exact
    arithmetic (those of 16-bit values often are) go by the last bit of that ``y``.  It is a
    forward for inference and for the 8-bit side of a product: it has no gradient, and asserts
    that none is asked for."""
    _check_add_norm(x, residual, weight)
    assert block in (None, 128), "block is None (a scale per row) or 128"
    assert not _lib.wants_derivative(x, weight, *(() if residual is None else (residual,))), \
        "fused_add_rms_norm_quant has no gradient: call it under torch.no_grad()"
    n_cols = x.shape[-1]
    n_rows = x.numel() // n_cols
    x2, xs = _lib.rows_of(x, n_cols)
    w = weight.contiguous()
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    groups = 1 if block is None else -(-n_cols // block)
    scales = x.new_empty((*x.shape[:-1], groups), dtype=torch.float32)
    r2, rs, h = None, 0, x
    if residual is not None:
        r2, rs = _lib.rows_of(residual, n_cols)
        h = residual.new_empty(x.shape)
    with _lib.on_device(x):
        _lib.call("fk_add_rmsnorm_quant", x2.data_ptr(), xs, _lib.ptr(r2), rs,
                  _lib.dtype_code(h.dtype), w.data_ptr(), _lib.dtype_code(w.dtype), q.data_ptr(),
                  scales.data_ptr(), None if r2 is None else h.data_ptr(), n_rows, n_cols,
                  block or 0, float(eps), _lib.dtype_code(x.dtype), _lib.stream_of(x))
    return q, scales, h


class FusedAddRMSNorm(FusedRMSNorm):
    """``FusedRMSNorm`` that takes the residual stream along: ``forward(x, residual)`` returns
    ``(norm(x + residual), x + residual)``; with residual None, ``(norm(x), x)``.  Same
    parameter and state_dict key."""

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        if residual is None:
            return super().forward(x), x
        return fused_add_rms_norm(x, residual, self.weight, self.eps)
