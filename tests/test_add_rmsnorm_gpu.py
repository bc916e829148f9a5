"""Residual addition + RMSNorm (forward, backward, 8-bit output) against 64-bit arithmetic.

The bounds are those of operator_reference.add_norm plus one rounding to the output's type
(torch.finfo(t).eps / 2 of the value); h is the fp32 sum rounded once and has to be equal.
For the 8-bit output the scale has the bound of y, and q has to be what e4m3 rounding gives for
some quotient within that bound of the 64-bit one."""
import pytest
import torch

import fusedkernels_b200 as fk
from conftest import gen
from operator_reference import U, add_norm, assert_within, half_step, tiny

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
TYPES = [(FP, FP), (BF, BF), (HF, HF), (BF, FP), (HF, FP)]


def inputs(shape, dtype, res, wdtype, seed=0):
    G = gen(seed)
    x = torch.randn(*shape, generator=G).to(dtype)
    r = (2 * torch.randn(*shape, generator=G)).to(res)
    w = (1 + 0.1 * torch.randn(shape[-1], generator=G)).to(wdtype)
    dy = torch.randn(*shape, generator=G).to(dtype)
    dh = torch.randn(*shape, generator=G).to(res)
    return x, r, w, dy, dh


def rounded(pair, dtype):
    want, bound = pair
    return want, bound + half_step(dtype) * (want.abs() + bound) + tiny(dtype)


def check(x, r, w, dy, dh, xg, rg, wg):
    """Runs the op on the given CUDA leaves and compares everything with the CPU inputs."""
    y, h = fk.fused_add_rms_norm(xg, rg, wg, EPS)
    assert y.dtype == x.dtype and h.dtype == r.dtype and y.shape == x.shape
    outs, grads = zip(*[(o, g.cuda()) for o, g in ((y, dy), (h, dh)) if g is not None])
    gx, gr, gw = torch.autograd.grad(outs, (xg, rg, wg), grads)
    assert gx.dtype == x.dtype and gr.dtype == r.dtype and gw.dtype == w.dtype
    ref = add_norm(x, r, w, EPS, dy, dh)
    assert torch.equal(h.detach().cpu(), ref["h"][0])
    assert_within(y, *rounded(ref["y"], x.dtype), "y")
    assert_within(gx, *rounded(ref["g"], x.dtype), "dx")
    assert_within(gr, *rounded(ref["g"], r.dtype), "dr")
    assert_within(gw, *rounded(ref["dw"], w.dtype), "dw")
    return y, h, gx, gr, gw


def leaves(*ts):
    return [t.cuda().requires_grad_(True) for t in ts]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 7), (5, 64), (33, 100), (4, 9, 1000),
                                   (301, 1111), (700, 1024), (40, 2752), (17, 4096), (9, 8192),
                                   (333, 12288), (7, 16384), (3, 16392), (2, 40000)], ids=str)
def test_matches_64_bits(shape, types):
    x, r, w, dy, dh = inputs(shape, *types, FP, seed=len(shape) + shape[-1])
    check(x, r, w, dy, dh, *leaves(x, r, w))


@pytest.mark.parametrize("wdtype", [BF, HF, FP])
@pytest.mark.parametrize("cols", [4096, 999])
def test_weight_types(wdtype, cols):
    x, r, w, dy, dh = inputs((64, cols), BF, BF, wdtype, seed=3)
    check(x, r, w, dy, dh, *leaves(x, r, w))


@pytest.mark.parametrize("types", [(BF, BF), (BF, FP), (FP, FP)], ids=str)
def test_many_rows(types):
    """More rows than the grid holds at once; twice, with the same bits."""
    x, r, w, dy, dh = inputs((5000, 512), *types, FP, seed=4)
    a = check(x, r, w, dy, dh, *leaves(x, r, w))
    b = check(x, r, w, dy, dh, *leaves(x, r, w))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(10007, 33), (20005, 130), (9, 2001), (17, 7001)], ids=str)
def test_odd_widths(shape, types):
    """Widths that are not whole 16-byte packets: many short rows, long rows."""
    x, r, w, dy, dh = inputs(shape, *types, FP, seed=30 + shape[1])
    check(x, r, w, dy, dh, *leaves(x, r, w))
    check(x, r, w, dy, None, *leaves(x, r, w))
    for block in (None, 128):
        check_quant(x, r, w, block)


def test_one_output_used():
    x, r, w, dy, dh = inputs((30, 256), BF, FP, FP, seed=5)
    check(x, r, w, dy, None, *leaves(x, r, w))
    xg, rg, wg = leaves(x, r, w)
    _, h = fk.fused_add_rms_norm(xg, rg, wg, EPS)
    gx, gr, gw = torch.autograd.grad(h, (xg, rg, wg), dh.cuda())
    assert torch.equal(gr.cpu(), dh) and torch.equal(gx.cpu(), dh.to(BF))
    assert torch.count_nonzero(gw) == 0 and gw.dtype == FP


@pytest.mark.parametrize("which", range(3))
def test_one_input_needs_a_gradient(which):
    x, r, w, dy, dh = inputs((10, 128), FP, FP, FP, seed=6)
    ts = [t.cuda() for t in (x, r, w)]
    ts[which].requires_grad_(True)
    y, h = fk.fused_add_rms_norm(*ts, EPS)
    assert h.requires_grad == (which != 2) or which == 2
    (g,) = torch.autograd.grad(y, ts[which], dy.cuda())
    ref = add_norm(x, r, w, EPS, dy)
    assert_within(g, *rounded(ref["dw" if which == 2 else "g"], FP))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides_and_offsets(dtype):
    """Column slices, a transposed tensor, an expanded residual, rows off 16-byte boundaries and
    expanded gradients give what contiguous copies give."""
    G = gen(7)
    wide = torch.randn(40, 1100, generator=G).to(dtype)
    tall = torch.randn(512, 40, generator=G).to(dtype)
    one = torch.randn(1, 512, generator=G).to(dtype)
    w = 1 + 0.1 * torch.randn(512, generator=G)
    dy, dh = torch.randn(2, 40, 512, generator=G).to(dtype)
    wide_g, tall_g, one_g = wide.cuda(), tall.cuda(), one.cuda()
    for a, b in ((0, 512), (512, 1024), (3, 515), (580, 1092)):
        for r, rg in ((tall.t(), tall_g.t()), (one.expand(40, 512), one_g.expand(40, 512)),
                      (wide[:, 7:519], wide_g[:, 7:519])):
            check(wide[:, a:b], r, w, dy, dh, wide_g[:, a:b].detach().requires_grad_(True),
                  rg.detach().requires_grad_(True), w.cuda().requires_grad_(True))
    xg, rg, wg = leaves(wide[:, :512].contiguous(), tall.t().contiguous(), w)
    y, h = fk.fused_add_rms_norm(xg, rg, wg, EPS)
    (y.float().sum() + h.float().sum()).backward()
    ref = add_norm(wide[:, :512], tall.t(), w, EPS, torch.ones(40, 512), torch.ones(40, 512))
    assert_within(xg.grad, *rounded(ref["g"], dtype))
    assert_within(wg.grad, *rounded(ref["dw"], FP))


def test_same_tensor_twice_and_second_backward():
    x, _, w, dy, dh = inputs((20, 96), FP, FP, FP, seed=8)
    xg, wg = leaves(x, w)
    y, h = fk.fused_add_rms_norm(xg, xg, wg, EPS)
    ref = add_norm(x, x, w, EPS, dy, dh)
    for _ in range(2):
        gx, gw = torch.autograd.grad((y, h), (xg, wg), (dy.cuda(), dh.cuda()), retain_graph=True)
        want, bound = rounded(ref["g"], FP)
        assert_within(gx, 2 * want, 2 * bound + 2 * U * want.abs())
        assert_within(gw, *rounded(ref["dw"], FP))


def test_gradient_against_differences():
    """The kernels' own gradient against central differences of their forward in fp32: steps of
    2^-7 on values of order 1, whose third derivatives are of order 1 (error about 2^-14 / 6), plus
    the forward's roundings over the step: 2^-22 * sum|y| / 2^-7."""
    x, r, w, dy, dh = inputs((4, 24), FP, FP, FP, seed=9)
    xg, rg, wg = leaves(x, r, w)
    y, h = fk.fused_add_rms_norm(xg, rg, wg, EPS)
    grads = torch.autograd.grad((y, h), (xg, rg, wg), (dy.cuda(), dh.cuda()))

    def value(x, r, w):
        with torch.no_grad():
            y, h = fk.fused_add_rms_norm(x.cuda(), r.cuda(), w.cuda(), EPS)
        return (y.cpu().double() * dy).sum() + (h.cpu().double() * dh).sum()

    step = 2.0 ** -7
    for which, g in enumerate(grads):
        flat = [x, r, w][which].reshape(-1)
        for i in range(0, flat.numel(), 5):
            ends = []
            for sign in (1, -1):
                ts = [x.clone(), r.clone(), w.clone()]
                ts[which].reshape(-1)[i] += sign * step
                ends.append((value(*ts), ts[which].reshape(-1)[i].double()))
            diff = (ends[0][0] - ends[1][0]) / (ends[0][1] - ends[1][1])
            assert abs(float(diff) - float(g.reshape(-1)[i])) <= 5e-3


def test_not_finite_stays_in_its_row():
    x, r, w, dy, dh = inputs((6, 300), BF, BF, FP, seed=10)
    x[1, 5] = float("nan")
    r[3, 7] = float("inf")
    xg, rg, wg = leaves(x, r, w)
    y, h = fk.fused_add_rms_norm(xg, rg, wg, EPS)
    ref = add_norm(x, r, w, EPS)
    rows = [0, 2, 4, 5]
    want, bound = rounded(ref["y"], BF)
    assert_within(y[rows], want[rows], bound[rows])
    assert torch.isnan(y[1]).all() and torch.isnan(y[3, 7])
    assert torch.count_nonzero(y[3, :7]) == 0  # finite values over an infinite norm


def test_zero_rows_and_zero_row():
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", dtype=BF, requires_grad=True)
    y, h = fk.fused_add_rms_norm(x, x.detach(), w)
    (y.float().sum() + h.float().sum()).backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and torch.count_nonzero(w.grad) == 0
    x = torch.zeros(2, 64, device="cuda")
    y, h = fk.fused_add_rms_norm(x, x, w.detach())
    assert torch.count_nonzero(y) == 0


def test_other_stream_and_graph_replay():
    """A forward and backward captured once and replayed on new inputs, beside eager calls on
    another stream."""
    x, r, w, dy, dh = inputs((64, 520), BF, FP, FP, seed=11)
    xs, rs, ws = leaves(x, r, w)
    dys, dhs = dy.cuda(), dh.cuda()

    def step():
        y, h = fk.fused_add_rms_norm(xs, rs, ws, EPS)
        return (y, h) + torch.autograd.grad((y, h), (xs, rs, ws), (dys, dhs))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    x2, r2, _, dy2, dh2 = inputs((64, 520), BF, FP, FP, seed=12)
    with torch.no_grad():
        xs.copy_(x2.cuda())
        rs.copy_(r2.cuda())
        dys.copy_(dy2.cuda())
        dhs.copy_(dh2.cuda())
    graph.replay()
    torch.cuda.synchronize()
    ref = add_norm(x2, r2, w, EPS, dy2, dh2)
    for got, key, t in zip(outs, ("y", "h", "g", "g", "dw"), (BF, FP, BF, FP, FP)):
        want, bound = ref[key]
        assert_within(got, want, bound + half_step(t) * want.double().abs() * 1.01 + tiny(t), key)


def test_module_and_refusals():
    norm = fk.FusedAddRMSNorm(64, eps=1e-5).cuda()
    assert list(norm.state_dict()) == ["weight"]
    x = torch.randn(5, 64, device="cuda")
    y, h = norm(x, None)
    assert h is x and torch.equal(y, fk.FusedRMSNorm(64, eps=1e-5).cuda()(x))
    y, h = norm(x, x)
    assert torch.equal(h, x + x)
    w = norm.weight
    for bad in ((x, x[:4], w), (x, x[:, :1], w), (x, x.bfloat16(), w), (x.double(), x.double(), w),
                (x, x.cpu(), w), (x, x, w[:32]), (x.cpu(), x.cpu(), w), (x, x, w.cpu())):
        with pytest.raises(AssertionError):
            fk.fused_add_rms_norm(*bad)
    with pytest.raises(AssertionError, match="no gradient"):
        fk.fused_add_rms_norm_quant(x, x, w)
    with pytest.raises(AssertionError, match="block"), torch.no_grad():
        fk.fused_add_rms_norm_quant(x, x, w, block=64)


# ------------------------------------------------------------------ 8 bits --------------
def check_quant(x, r, w, block, xg=None, rg=None):
    xg = x.cuda() if xg is None else xg
    rg = (None if r is None else r.cuda()) if rg is None else rg
    with torch.no_grad():
        q, scales, h = fk.fused_add_rms_norm_quant(xg, rg, w.cuda(), EPS, block=block)
    ref = add_norm(x, r, w, EPS)
    assert torch.equal(h.cpu(), ref["h"][0])
    if r is None:
        assert h is xg
    y, bound = ref["y"]
    d = y.shape[-1]
    b = block or d
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    assert scales.shape == (*x.shape[:-1], -(-d // b)) and scales.dtype == FP
    parts = y.split(b, dim=-1)
    s64 = torch.stack([p.abs().amax(-1) for p in parts], -1).div(448).clamp(min=2.0 ** -126)
    f = (d / 256 + 48) * U
    assert_within(scales, s64, f * s64, "scales")
    quot = torch.cat([p / s64[..., i:i + 1] for i, p in enumerate(parts)], -1)
    e4m3 = lambda v: v.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()  # noqa: E731
    lo, hi = e4m3(quot * (1 - 4 * f)), e4m3(quot * (1 + 4 * f))
    got = q.cpu().double()
    assert ((got >= torch.minimum(lo, hi)) & (got <= torch.maximum(lo, hi))).all()
    return q, scales


@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 7), (70, 64), (33, 129), (2, 3, 1000),
                                   (301, 1111), (40, 2752), (64, 4096), (5, 8192), (2, 16400),
                                   (2, 40000)], ids=str)
def test_quant_matches_64_bits(shape, types, block):
    x, r, w, _, _ = inputs(shape, *types, FP, seed=20 + shape[-1])
    check_quant(x, r, w, block)
    if types[0] == types[1]:
        check_quant(x, None, w, block)


@pytest.mark.parametrize("block", [None, 128])
def test_quant_strides_weights_and_many_rows(block):
    x, r, w, _, _ = inputs((3000, 300), BF, BF, BF, seed=21)
    xg, rg = torch.zeros(3000, 333, device="cuda", dtype=BF), r.t().contiguous().cuda().t()
    xg[:, 5:305] = x.cuda()
    check_quant(x, r, w, block, xg[:, 5:305], rg)
    a, b = check_quant(x, r, w, block), check_quant(x, r, w, block)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("block", [None, 128])
def test_quant_edges(block):
    """A row of zeros, one huge value beside small ones, tiny rows (below eps), NaN, no rows."""
    G = gen(22)
    x = torch.randn(8, 384, generator=G)
    x[0] = 0
    x[1, 200] = 1e4
    x[2] *= 1e-30
    x[3, :128] = 0
    check_quant(x, torch.zeros_like(x), 1 + 0.1 * torch.randn(384, generator=G), block)
    x[4, 130] = float("nan")
    q, scales, _ = fk.fused_add_rms_norm_quant(x.cuda(), None, torch.ones(384, device="cuda"),
                                               block=block)
    assert torch.isnan(q[4].float()).all() and not torch.isnan(q[5].float()).any()
    assert torch.count_nonzero(q[0].float()) == 0 and (scales[0] == 2.0 ** -126).all()
    q, scales, h = fk.fused_add_rms_norm_quant(x[:0].cuda(), x[:0].cuda(),
                                               torch.ones(384, device="cuda"), block=block)
    assert q.shape == (0, 384) and scales.shape == (0, 3 if block else 1) and h.shape == (0, 384)


def test_quant_graph_replay():
    x, r, w, _, _ = inputs((16, 4096), BF, BF, FP, seed=23)
    xs, rs, ws = x.cuda(), r.cuda(), w.cuda()
    with torch.no_grad():
        want = fk.fused_add_rms_norm_quant(xs, rs, ws, block=128)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = fk.fused_add_rms_norm_quant(xs, rs, ws, block=128)
        for t in got:
            t.view(torch.uint8).zero_()
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# In fp32 the forward's y is the very y that is quantised: its row sum has the same terms in the
# same order.  So scales and bytes have to be those of the 32-bit divisions, bit for bit.
def divided(y, block):
    b = block or y.shape[-1]
    parts = y.split(b, dim=-1)
    scales = torch.stack([p.abs().amax(-1) for p in parts], -1).div(448).clamp(min=2.0 ** -126)
    q = torch.cat([p / scales[..., i:i + 1] for i, p in enumerate(parts)], -1)
    return q.clamp(-448, 448).to(torch.float8_e4m3fn), scales


def assert_divided(got, y, block):
    q, scales = divided(y.cpu(), block)
    assert torch.equal(got[1].cpu(), scales)
    assert torch.equal(got[0].cpu().view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("shape", [(700, 64), (64, 4096), (2048, 2048), (400, 1111), (9, 8192),
                                   (3, 16400)], ids=str)
def test_quant_is_a_division(shape, block):
    """Short rows to the longest, whole packets, single elements and element loops."""
    x, r, w, _, _ = inputs(shape, FP, FP, FP, seed=24)
    for row, size in enumerate((1e-26, 1e-30, 1e-34)[:shape[0]]):  # rows far below eps: tiny scales
        x[row] *= size
        r[row] *= size
    w[0], w[1], w[2] = 0.0, 1e30, 1e33  # zeros of both signs; large scales
    xg, rg, wg = x.cuda(), r.cuda(), w.cuda()
    with torch.no_grad():
        y, _ = fk.fused_add_rms_norm(xg, rg, wg, EPS)
        assert_divided(fk.fused_add_rms_norm_quant(xg, rg, wg, EPS, block=block), y, block)
        wg[:3] = 1.0
        y, _ = fk.fused_add_rms_norm(xg, rg, wg, EPS)
        assert_divided(fk.fused_add_rms_norm_quant(xg, rg, wg, EPS, block=block), y, block)


@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cols", [4096, 1111])
def test_quant_is_a_division_in_16_bits(cols, dtype, block):
    """Rows of +1 and -1: the sum of squares is exact in any order, so the 32-bit y of the same
    values in fp32 is known beside a 16-bit x."""
    G = gen(25)
    x = (torch.randint(0, 2, (500, cols), generator=G) * 2 - 1).to(dtype).cuda()
    w = (1 + 0.5 * torch.randn(cols, generator=G)).cuda()
    w[5] = 0.0
    with torch.no_grad():
        y, _ = fk.fused_add_rms_norm(x.float(), torch.zeros(500, cols, device="cuda"), w, EPS)
        for r in (None, torch.zeros_like(x), torch.zeros(500, cols, device="cuda")):
            assert_divided(fk.fused_add_rms_norm_quant(x, r, w, EPS, block=block), y, block)


def test_no_residual_is_refused():
    """(The module and the 8-bit form take None.)"""
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(AssertionError, match="residual"):
        fk.fused_add_rms_norm(x, None, w)


@pytest.mark.parametrize("types", [(FP, FP), (BF, BF), (BF, FP)], ids=str)
@pytest.mark.parametrize("cols", [64, 1000, 1111, 4096, 40000])
@pytest.mark.parametrize("size", [1e-12, 1e10, 1e14, 1e16])
def test_gradient_of_rows_of_any_size(size, cols, types):
    """s^3 leaves the normal range of fp32 at 1e13 and more, the gradient does not."""
    x, r, w, dy, _ = inputs((6, cols), *types, FP, seed=31)
    x, r = (x.double() * size).to(types[0]), (r.double() * size).to(types[1])
    check(x, r, w, dy, None, *leaves(x, r, w))
