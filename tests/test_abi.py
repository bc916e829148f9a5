"""The C ABI library: loads without a GPU, exports every symbol include/fkb200.h declares,
and rejects bad arguments before touching the device (no compute calls here)."""
import ctypes
import re
from pathlib import Path

import pytest

from fusedkernels_b200 import _lib

HEADER = Path(__file__).resolve().parents[1] / "include" / "fkb200.h"


def declared_symbols():
    text = HEADER.read_text()
    return sorted(set(re.findall(r"FK_API\s+[\w\s\*]+?\b(fk_\w+)\s*\(", text)))


def test_header_declares_entry_points():
    syms = declared_symbols()
    assert "fk_router_fwd" in syms and "fk_ce_fwd" in syms and len(syms) >= 12


def test_library_exports_every_declared_symbol():
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    missing = [s for s in declared_symbols() if not hasattr(lib, s)]
    assert not missing, f"missing exports: {missing}"


def test_binding_covers_header():
    assert set(declared_symbols()) <= set(_lib.SIGNATURES)


def test_status_strings():
    lib = _lib.load()
    assert lib.fk_version() >= 100
    assert lib.fk_status_string(0) == b"ok"
    assert lib.fk_status_string(1) == b"invalid argument"


@pytest.mark.parametrize("k,E", [(0, 8), (9, 8)])
def test_router_rejects_bad_k(k, E):
    lib = _lib.load()
    st = lib.fk_router_fwd(None, E, 0, 4, E, k, None, None, None)
    assert st == 1 and b"k" in lib.fk_last_error()


def test_router_rejects_too_many_experts():
    lib = _lib.load()
    assert lib.fk_router_fwd(None, 512, 0, 4, 512, 2, None, None, None) == 2


def test_negative_sizes_and_bad_dtype_rejected():
    lib = _lib.load()
    assert lib.fk_swiglu_fwd(None, None, None, -1, 0, None) == 1
    assert lib.fk_swiglu_fwd(None, None, None, 0, 0, None) == 0  # empty: no-op
    assert lib.fk_rmsnorm_fwd(None, 8, None, 0, None, 8, None, -1, 8, 1e-6, 0, None) == 1
    assert lib.fk_ce_fwd(None, 4, None, 4, None, 2, 0, -100, 0.0, 0, None, None, None, None,
                         None) == 1
    with pytest.raises(RuntimeError, match="invalid argument"):
        _lib.call("fk_router_bwd", None, None, None, None, 4, 8, 9, None)


def test_ce_rejects_bad_smoothing():
    lib = _lib.load()
    one = ctypes.c_int(0)
    f = ctypes.c_float(0)
    st = lib.fk_ce_fwd(None, 4, None, 4, None, 0, 4, -100, 1.5, 0, None, ctypes.byref(f),
                       ctypes.byref(one), ctypes.byref(one), None)
    assert st == 1


def test_ep_planning_workspace_and_peer_argument_checks():
    """The expert-parallel entry points validate their arguments on the host (no device
    work happens for a rejected call)."""
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    assert lib.fk_ep_plan_workspace_size(1000, 8, ctypes.byref(n)) == 0
    assert n.value == 4 * 8 * 4  # ceil(1000 / 256) chunks x 8 ranks x int32
    assert lib.fk_ep_plan_workspace_size(10, 33, ctypes.byref(n)) == 1  # at most 32 ranks
    # n_ranks 0, my_rank out of range, phase out of range
    assert lib.fk_ep_peer_put_rows(None, 64, None, 4, 0, 0, None, None, 2, None, None, None,
                                   None, 0, None, 2, None) == 1
    assert lib.fk_ep_peer_put_rows(None, 64, None, 4, 2, 2, None, None, 2, None, None, None,
                                   None, 0, None, 2, None) == 1
    assert lib.fk_ep_peer_combine_put(None, 64, None, None, 4, 2, 0, 2, None, None, None, None,
                                      4, None, 2, None) == 1
    assert lib.fk_ep_peer_wait(None, 2, 0, None, 100, None, None) == 1
    assert lib.fk_ep_peer_wait(None, 0, 0, None, 100, None, None) == 1
    assert lib.fk_ipc_alloc(0, None, None) == 1
    assert lib.fk_ipc_open(None, None) == 1


def test_add_rmsnorm_argument_checks():
    """Refused on the host, before any device work."""
    lib = _lib.load()
    F32, F16, BF16 = 0, 1, 2

    def fwd(xs=8, rs=8, rd=BF16, wd=F32, rows=4, cols=8, dt=BF16):
        return lib.fk_add_rmsnorm_fwd(None, xs, None, rs, rd, None, wd, None, None, None, rows, cols,
                                      1e-6, dt, None)

    assert fwd() == 1 and b"null" in lib.fk_last_error()
    assert fwd(rows=0) == 0
    assert fwd(rows=-1) == 1 and fwd(cols=0) == 1 and fwd(xs=7) == 1 and fwd(rs=7) == 1
    assert fwd(rd=F16) == 1 and fwd(dt=7) == 1 and fwd(wd=7) == 1
    assert fwd(dt=F32, rd=BF16) == 1  # a residual narrower than x
    n = ctypes.c_size_t(0)
    assert lib.fk_add_rmsnorm_bwd_workspace_size(10, 8, None) == 1
    assert lib.fk_add_rmsnorm_bwd_workspace_size(10, 0, ctypes.byref(n)) == 1
    assert lib.fk_add_rmsnorm_bwd_workspace_size(10, 8, ctypes.byref(n)) == 0 and n.value > 0

    def bwd(ptr=1, dr=None, ws=None, size=0, rd=BF16, stride=8):
        return lib.fk_add_rmsnorm_bwd(ptr, stride, None, 0, ptr, rd, ptr, F32, ptr, ptr, dr, ptr, ws,
                                      size, 4, 8, BF16, None)

    assert bwd(ptr=None) == 1 and bwd(rd=F32) == 1 and bwd(stride=7) == 1
    assert bwd() == 4 and bwd(ws=8, size=1 << 30) == 4  # no workspace; one off its alignment

    def quant(block=0, r=None, h=None, rows=4):
        return lib.fk_add_rmsnorm_quant(1, 8, r, 8, BF16, 1, F32, 1, 1, h, rows, 8, block, 1e-6, BF16,
                                        None)

    assert quant(block=64) == 1 and quant(block=-1) == 1 and quant(r=1) == 1
    assert quant(rows=0) == 0


def test_balance_argument_checks():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    assert lib.fk_moe_balance_workspace_size(None) == 1
    assert lib.fk_moe_balance_workspace_size(ctypes.byref(n)) == 0 and n.value > 0

    def run(stride=8, rows=4, e=8, k=2, dt=0, ptr=16, ws=16, size=1 << 30, scale=1.0):
        return lib.fk_moe_balance(ptr, stride, ptr, None, rows, e, k, 0.0, scale, None, ptr, ptr, ws,
                                  size, dt, None)

    assert run(e=257, stride=257) == 2 and b"257" in lib.fk_last_error()
    assert run(rows=-1) == 1 and run(e=0) == 1 and run(stride=7) == 1 and run(dt=3) == 1
    assert run(rows=1 << 30, k=2) == 1  # slots are counted in 32 bits
    assert run(ptr=None) == 1 and run(scale=0.0) == 1 and run(scale=float("inf")) == 1
    assert run(ws=None) == 4 and run(ws=8) == 4 and run(size=16) == 4


def test_distill_argument_checks():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    assert lib.fk_distill_workspace_size(4, 2, None) == 1
    assert lib.fk_distill_workspace_size(4, 0, ctypes.byref(n)) == 1
    assert lib.fk_distill_workspace_size(4, 2, ctypes.byref(n)) == 0 and n.value > 0

    def run(ptr=16, stride=8, grad=None, gstride=0, k=2, rows=4, cols=8, t=1.0, hw=0.5, dt=0, tdt=0,
            ws=16, size=1 << 30, scale=1.0):
        return lib.fk_distill(ptr, stride, grad, gstride, ptr, ptr, tdt, k, None, rows, cols, -100, t,
                              hw, scale, dt, ptr, ptr, ws, size, None)

    assert run(k=1025) == 2 and b"1025" in lib.fk_last_error()
    assert run(k=0) == 1 and run(rows=-1) == 1 and run(cols=0) == 1 and run(stride=7) == 1
    assert run(cols=1 << 31, stride=1 << 31) == 1 and run(grad=16, gstride=7) == 1
    assert run(t=0.0) == 1 and run(t=float("inf")) == 1 and run(t=float("nan")) == 1
    assert run(scale=-1.0) == 1 and run(scale=float("nan")) == 1
    assert run(hw=1.5) == 1 and run(hw=float("nan")) == 1 and run(dt=3) == 1 and run(tdt=-1) == 1
    assert run(ptr=None) == 1
    assert run(ws=None) == 4 and run(ws=8) == 4 and run(size=16) == 4


def test_grad_rescale_argument_checks():
    lib = _lib.load()

    def run(ptr=16, stride=8, rows=4, cols=8, expected=1.0, dt=0):
        return lib.fk_grad_rescale(ptr, stride, rows, cols, ptr, expected, dt, None)

    assert run(ptr=None) == 1 and run(stride=7) == 1 and run(rows=-1) == 1 and run(dt=5) == 1
    assert run(expected=0.0) == 1 and run(expected=float("nan")) == 1
    assert run(rows=0) == 0 and run(cols=0) == 0
