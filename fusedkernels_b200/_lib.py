"""ctypes binding of libfkb200.so, the C ABI declared in include/fkb200.h.

The library is loaded on first use.  If it has not been built, every op raises
RuntimeError: there is no CPU fallback for any op in this package.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import threading
from pathlib import Path

import torch
from torch.autograd import forward_ad

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libfkb200.so"

FK_F32, FK_F16, FK_BF16 = 0, 1, 2
_DTYPE_CODES = {torch.float32: FK_F32, torch.float16: FK_F16, torch.bfloat16: FK_BF16}

_vp, _i64, _i32, _f32, _sz = C.c_void_p, C.c_int64, C.c_int, C.c_float, C.c_size_t

# name -> argtypes (restype is int status unless listed in _RESTYPES)
SIGNATURES: dict[str, list] = {
    "fk_version": [],
    "fk_status_string": [_i32],
    "fk_last_error": [],
    "fk_swiglu_fwd": [_vp, _vp, _vp, _i64, _i32, _vp],
    "fk_swiglu_bwd": [_vp, _vp, _vp, _vp, _vp, _i64, _i32, _vp],
    "fk_rmsnorm_fwd": [_vp, _i64, _vp, _i32, _vp, _i64, _vp, _i64, _i64, _f32, _i32, _vp],
    "fk_rmsnorm_bwd_workspace_size": [_i64, _i64, C.POINTER(_sz)],
    "fk_rmsnorm_bwd": [_vp, _vp, _vp, _i32, _vp, _vp, _vp, _vp, _sz, _i64, _i64, _i32, _vp],
    "fk_rmsnorm_bwd_noalloc": [_vp, _vp, _vp, _i32, _vp, _vp, _vp, _i64, _i64, _i32, _vp],
    "fk_add_rmsnorm_fwd": [_vp, _i64, _vp, _i64, _i32, _vp, _i32, _vp, _vp, _vp, _i64, _i64, _f32,
                           _i32, _vp],
    "fk_add_rmsnorm_bwd_workspace_size": [_i64, _i64, C.POINTER(_sz)],
    "fk_add_rmsnorm_bwd": [_vp, _i64, _vp, _i64, _vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp,
                           _sz, _i64, _i64, _i32, _vp],
    "fk_add_rmsnorm_quant": [_vp, _i64, _vp, _i64, _i32, _vp, _i32, _vp, _vp, _vp, _i64, _i64,
                             _i64, _f32, _i32, _vp],
    "fk_grad_rescale": [_vp, _i64, _i64, _i64, _vp, _f32, _i32, _vp],
    "fk_moe_balance_workspace_size": [C.POINTER(_sz)],
    "fk_moe_balance": [_vp, _i64, _vp, _vp, _i64, _i32, _i32, _f32, _f32, _vp, _vp, _vp, _vp, _sz,
                       _i32, _vp],
    "fk_distill_workspace_size": [_i64, _i32, C.POINTER(_sz)],
    "fk_distill": [_vp, _i64, _vp, _i64, _vp, _vp, _i32, _i32, _vp, _i64, _i64, _i64, _f32, _f32,
                   _f32, _i32, _vp, _vp, _vp, _sz, _vp],
    "fk_router_fwd": [_vp, _i64, _i32, _i64, _i32, _i32, _vp, _vp, _vp],
    "fk_router_bwd": [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _vp],
    "fk_ce_fwd": [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _f32, _i32, _vp, _vp, _vp, _vp,
                  _vp],
    "fk_ce_bwd_scale": [_vp, _i64, _i64, _i64, _vp, _i32, _vp],
    "fk_moe_capacity": [_i64, _i32, _i32, C.POINTER(_i64), C.POINTER(_sz)],
    "fk_moe_route_meta": [_vp, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64,
                          _vp, _sz, _vp, _vp],
    "fk_moe_gather": [_vp, _i32, _vp, _i32, _vp, _i64, _vp, _i32, _vp],
    "fk_moe_gather_by_token": [_vp, _i32, _vp, _i64, _i32, _vp, _vp, _i64, _vp, _i32, _vp],
    "fk_moe_combine": [_vp, _i32, _vp, _vp, _i64, _i32, _vp, _i32, _vp],
    "fk_moe_combine_bwd": [_vp, _vp, _i32, _vp, _vp, _i32, _vp, _i64, _vp, _vp, _i32, _vp],
    "fk_moe_gemm_up": [_vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _i32, _vp, _vp],
    "fk_moe_gemm_down": [_vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _i32, _vp, _vp],
    "fk_moe_gemm_down_dgrad": [_vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _i32, _vp,
                               _vp],
    "fk_moe_gemm_up_dgrad": [_vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _i32, _vp, _vp],
    "fk_moe_gemm_wgrad": [_vp, _i32, _vp, _i32, _i64, _vp, _i32, _vp, _i32, _vp, _vp],
    "fk_moe_gemm_up_weighted": [_vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp,
                                _i32, _vp, _vp],
    "fk_moe_gemm_down_dgrad_weighted": [_vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp, _vp,
                                        _vp, _vp, _vp, _i32, _vp, _vp],
    "fk_moe_dw_from_parts": [_vp, _i32, _vp, _vp, _i64, _vp, _vp],
    "fk_tf32_split": [_vp, _i64, _vp, _vp, _vp],
    "fk_moe_gemm_up_typed": [_vp, _vp, _i64, _i32, _vp, _vp, _i32, _i32, _vp, _vp, _vp, _vp,
                             _i32, _vp, _vp],
    "fk_moe_gemm_down_typed": [_vp, _vp, _i64, _i32, _vp, _vp, _i32, _i32, _vp, _vp, _vp, _i32,
                               _vp, _vp],
    "fk_moe_gemm_down_dgrad_typed": [_vp, _vp, _i64, _i32, _vp, _vp, _i32, _i32, _vp, _vp, _vp,
                                     _vp, _i32, _vp, _vp],
    "fk_moe_gemm_up_dgrad_typed": [_vp, _vp, _i64, _i32, _vp, _vp, _i32, _i32, _vp, _vp, _vp,
                                   _i32, _vp, _vp],
    "fk_moe_gemm_wgrad_typed": [_vp, _vp, _i32, _vp, _vp, _i32, _i64, _vp, _i32, _vp, _i32, _vp,
                                _vp],
    "fk_moe_route_meta_skip": [_vp, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                               _i64, _vp, _sz, _vp, _vp],
    "fk_ep_plan_workspace_size": [_i64, _i32, C.POINTER(_sz)],
    "fk_ep_plan": [_vp, _vp, _i64, _i32, _vp, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                   _vp, _vp],
    "fk_ep_pack": [_vp, _i32, _vp, _i64, _vp, _i32, _vp],
    "fk_ep_unpack_sum": [_vp, _i32, _vp, _i64, _i32, _vp, _i32, _vp],
    "fk_ep_unpack_dw": [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _vp, _vp],
    "fk_ipc_alloc": [_sz, C.POINTER(_vp), _vp],
    "fk_ipc_open": [_vp, C.POINTER(_vp)],
    "fk_ipc_close": [_vp],
    "fk_ipc_free": [_vp],
    "fk_ep_peer_put_rows": [_vp, _i32, _vp, _i64, _i32, _i32, _vp, _vp, _i32, _vp, _vp, _vp, _vp,
                            _i32, _vp, _i32, _vp],
    "fk_ep_peer_combine_put": [_vp, _i32, _vp, _vp, _i64, _i32, _i32, _i32, _vp, _vp, _vp, _vp,
                               _i32, _vp, _i32, _vp],
    "fk_ep_peer_wait": [_vp, _i32, _i32, _vp, _i32, _vp, _vp],
    "fk_bitonic_sort_i32": [_vp, _i64, _i32, _i64, _vp, _i64, _vp],
    "fk_bitonic_sort_bounded_i32": [_vp, _i64, _i32, _i64, _i32, _vp, _vp],
    "fk_bitonic_merge_topk_i32": [_vp, _vp, _i64, _i32, _vp, _vp],
}
_RESTYPES = {"fk_status_string": C.c_char_p, "fk_last_error": C.c_char_p}

_lib = None
_lock = threading.Lock()


def load() -> C.CDLL:
    """Load libfkb200.so (once) and attach the declared signatures."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(
                    f"{LIB_PATH} is not built; run `python -m fusedkernels_b200._build` "
                    "(fusedkernels_b200 has no CPU fallback)")
            lib = C.CDLL(str(LIB_PATH))
            for name, args in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = _RESTYPES.get(name, C.c_int)
            _lib = lib
    return _lib


def check(status: int, name: str) -> None:
    if status != 0:
        lib = load()
        msg = lib.fk_last_error().decode(errors="replace")
        raise RuntimeError(f"{name} failed ({lib.fk_status_string(status).decode()}): {msg}")


def call(name: str, *args) -> None:
    """Call a status-returning entry point and raise RuntimeError on failure."""
    status = getattr(_lib or load(), name)(*args)
    if status:
        check(status, name)


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16")


def stream_of(t: torch.Tensor) -> int:
    """Handle of the current stream of ``t``'s device."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_ws_cache: dict = {}


def rmsnorm_bwd_workspace_bytes(rows: int, cols: int, device: torch.device) -> int:
    key = (rows, cols, device.index)
    v = _ws_cache.get(key)
    if v is None:
        out = C.c_size_t(0)
        with torch.cuda.device(device):
            check(load().fk_rmsnorm_bwd_workspace_size(rows, cols, C.byref(out)),
                  "fk_rmsnorm_bwd_workspace_size")
        v = _ws_cache[key] = out.value
    return v


def ep_plan_workspace_bytes(n_tokens: int, n_ranks: int) -> int:
    out = C.c_size_t(0)
    check(load().fk_ep_plan_workspace_size(n_tokens, n_ranks, C.byref(out)),
          "fk_ep_plan_workspace_size")
    return out.value


_cap_cache: dict = {}


def moe_capacity(n_tokens: int, k: int, n_experts: int) -> tuple[int, int]:
    """(max sorted rows, metadata workspace bytes) for a routing of this size."""
    key = (n_tokens, k, n_experts)
    v = _cap_cache.get(key)
    if v is None:
        rows = C.c_int64(0)
        ws = C.c_size_t(0)
        check(load().fk_moe_capacity(n_tokens, k, n_experts, C.byref(rows), C.byref(ws)),
              "fk_moe_capacity")
        v = _cap_cache[key] = (rows.value, ws.value)
    return v


_op_ws_cache: dict = {}


def workspace_bytes(name: str, device: torch.device, *sizes) -> int:
    """Bytes that the sizing entry point ``name`` gives for these sizes on ``device``."""
    key = (name, device.index, *sizes)
    v = _op_ws_cache.get(key)
    if v is None:
        if len(_op_ws_cache) >= 4096:  # batches of ever new lengths: start over
            _op_ws_cache.clear()
        out = C.c_size_t(0)
        with torch.cuda.device(device):
            check(getattr(load(), name)(*sizes, C.byref(out)), name)
        v = _op_ws_cache[key] = out.value
    return v


_NO_SWITCH = contextlib.nullcontext()


def on_device(t: torch.Tensor):
    """Context in which launches go to ``t``'s device (free where it is the current one)."""
    i = t.device.index
    return _NO_SWITCH if i == torch.cuda.current_device() else torch.cuda.device(i)


def rows_of(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """``t`` seen as rows of ``cols`` elements with unit stride, and the rows' stride in
    elements: a tensor to read from (t itself, a view or a copy)."""
    if t.is_contiguous():
        return t, cols
    t = t.reshape(-1, cols)
    if cols > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < cols:
        return t.contiguous(), cols
    return t, max(t.stride(0), cols)  # a tensor of one row may report any stride


def wants_derivative(*tensors) -> bool:
    """Whether autograd has to see an operator's call: some input requires a gradient, or carries
    a tangent of forward mode (which an autograd.Function without a jvp refuses)."""
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors) or \
        has_tangent(*tensors)


def has_tangent(*tensors) -> bool:
    if forward_ad._current_level < 0:  # outside every dual_level: none can
        return False
    return any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _NoSecondDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, _anchor, *grads):
        return tuple(None if g is None else g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("this operator has no second derivative: its backward pass is "
                           "once_differentiable")


def once_differentiable(fn):
    """For backward passes made of kernels: under create_graph the gradients come with a node
    that raises when they are differentiated, whether grad_output asks for it or not."""
    def backward(ctx, *grads):
        if not torch.is_grad_enabled():
            return fn(ctx, *grads)
        with torch.no_grad():
            out = fn(ctx, *grads)
        out = out if isinstance(out, tuple) else (out,)
        return _NoSecondDerivative.apply(torch.empty(0, requires_grad=True), *out)

    return backward


def hand_over_gradient(ctx, grad_output: torch.Tensor) -> torch.Tensor:
    """The gradient that a forward pass already computed (ctx.grad, for grad_output ==
    ctx.loss_scale), scaled in place where grad_output is another number: the device decides,
    without a host sync.  It is the caller's from here on, so it is given once."""
    grad = ctx.grad
    if grad is None:
        raise RuntimeError("the gradient of this loss was handed over in its first backward "
                           "pass: compute the loss again for another one")
    ctx.grad = None
    go = grad_output if grad_output.dtype == torch.float32 else grad_output.to(torch.float32)
    rows, cols = grad.shape
    with on_device(grad):
        call("fk_grad_rescale", grad.data_ptr(), max(grad.stride(0), cols), rows, cols,
             go.data_ptr(), ctx.loss_scale, _DTYPE_CODES[grad.dtype], stream_of(grad))
    return grad.detach()


def num_sms(device: torch.device | None = None) -> int:
    """Streaming multiprocessors of the current (or given) CUDA device: the grid of the
    persistent kernels, one CTA per SM."""
    dev = torch.cuda.current_device() if device is None else device
    return torch.cuda.get_device_properties(dev).multi_processor_count
