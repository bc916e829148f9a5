"""Tensors of more than 2^31 elements: the last rows give the bits that the same rows give by
themselves (every row's result depends on the row alone, but for the mean's 1/n, which powers of
two keep exact)."""
import pytest
import torch

import fusedkernels_b200 as fk

pytestmark = pytest.mark.gpu


def room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
        pytest.skip("not enough free memory")


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols", [8192, 8191])
def test_add_norm(cols):
    rows = (1 << 31) // 8191 + 300
    room(45)
    G = torch.Generator("cuda").manual_seed(1)
    x, r, dy, dh = (torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=G)
                    for _ in range(4))
    w = torch.rand(cols, generator=G, device="cuda")
    last = slice(rows - 5, rows)

    def run(x, r, dy, dh):
        x, r = x.requires_grad_(True), r.requires_grad_(True)
        y, h = fk.fused_add_rms_norm(x, r, w)
        return (y, h) + torch.autograd.grad((y, h), (x, r), (dy, dh))

    want = run(*(t[last].clone() for t in (x, r, dy, dh)))
    got = run(x, r, dy, dh)
    assert all(torch.equal(a[last], b) for a, b in zip(got, want))
    del got, dy, dh
    with torch.no_grad():
        for block in (None, 128):
            want = fk.fused_add_rms_norm_quant(x[last].clone(), r[last].clone(), w, block=block)
            got = fk.fused_add_rms_norm_quant(x, r, w, block=block)
            assert all(torch.equal(a[last].float(), b.float()) for a, b in zip(got, want))


@pytest.mark.parametrize("experts", [160, 161])
def test_balance(experts):
    rows = 1 << 24  # 16.8 M tokens: 2.7e9 logits
    room(35)
    G = torch.Generator("cuda").manual_seed(2)
    x = torch.empty(rows, experts, device="cuda").normal_(generator=G).requires_grad_(True)
    idx = torch.arange(rows, device="cuda")[:, None] % experts  # an even load but for the rest
    loss, counts = fk.fused_moe_balance_loss(x, idx)
    (grad,) = torch.autograd.grad(loss, x)
    assert torch.equal(counts, torch.bincount(idx[:, 0], minlength=experts))
    tail = x[-7:].detach().double()
    f = counts.double() / rows
    p = torch.softmax(tail, 1)
    want = experts / rows * p * (f - (p * f).sum(1, keepdim=True))
    size = experts / rows * p * ((f - 1 / experts).abs() + (p * (f - 1 / experts).abs()).sum(1, keepdim=True))
    assert ((grad[-7:].double() - want).abs() <= 128 * 2.0 ** -24 * size + 1e-30).all()
    assert abs(float(loss.detach()) - 1.0) <= 1e-4


@pytest.mark.parametrize("vocab", [131072, 131071])
def test_distillation(vocab):
    rows = 1 << 15  # 4.3e9 logits
    room(40)
    G = torch.Generator("cuda").manual_seed(3)
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda").normal_(generator=G)
    idx = torch.randint(0, vocab, (rows, 4), generator=G, device="cuda")
    top = torch.randn(rows, 4, generator=G, device="cuda")
    targets = torch.randint(0, vocab, (rows,), generator=G, device="cuda")

    def run(x, idx, top, targets):
        x = x.requires_grad_(True)
        loss = fk.fused_distillation_loss(x, idx, top, targets)
        return loss.detach(), torch.autograd.grad(loss, x)[0]

    # 2^15 rows here, 8 there: 1/n differs by 2^12, exactly
    want = run(x[-8:].clone(), idx[-8:], top[-8:], targets[-8:])[1]
    loss, got = run(x, idx, top, targets)
    tail = got[-8:].float() * 2.0 ** 12
    # The row's slices (and so the order of its sum) may be others: one step of bf16.
    assert ((tail - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-30).all()
    assert torch.isfinite(loss)


def spots(rows, cols):
    """First rows, last rows, some between, and those beside every 2^31st element."""
    near = [k * (1 << 31) // cols + d for k in range(1, rows * cols // (1 << 31) + 1)
            for d in (-1, 0, 1)]
    some = torch.randint(0, rows, (200,), generator=torch.Generator().manual_seed(9)).tolist()
    at = [*range(5), *near, *some, *range(rows - 5, rows)]
    return torch.tensor(sorted({i for i in at if 0 <= i < rows}), device="cuda")


def leave_nan(*shapes_and_types):
    """Memory that the next allocations of these sizes are given holds NaN, so that what a kernel
    does not write is seen."""
    for shape, dtype in shapes_and_types:
        torch.full(shape, float("nan"), dtype=dtype, device="cuda")


@pytest.mark.parametrize("cols", [8192, 8191])
def test_add_norm_everywhere(cols):
    rows = (1 << 31) // 8191 + 300
    room(45)
    G = torch.Generator("cuda").manual_seed(4)
    x, r, dy, dh = (torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=G)
                    for _ in range(4))
    w = torch.rand(cols, generator=G, device="cuda")
    at = spots(rows, cols)
    leave_nan(*[((rows, cols), torch.bfloat16)] * 3)

    def run(x, r, dy, dh):
        x, r = x.requires_grad_(True), r.requires_grad_(True)
        y, h = fk.fused_add_rms_norm(x, r, w)
        return (y, h) + torch.autograd.grad((y, h), (x, r), (dy, dh))

    got = run(x, r, dy, dh)
    assert all(torch.isfinite(t).all() for t in got)
    want = run(*(t.detach()[at] for t in (x, r, dy, dh)))
    assert all(torch.equal(a[at], b) for a, b in zip(got, want))
    del got, dy, dh
    with torch.no_grad():
        for block in (None, 128):
            got = fk.fused_add_rms_norm_quant(x, r, w, block=block)
            want = fk.fused_add_rms_norm_quant(x[at], r[at], w, block=block)
            assert all(torch.equal(a[at].float(), b.float()) for a, b in zip(got, want))


@pytest.mark.parametrize("experts", [160, 161])
def test_balance_everywhere(experts):
    rows = 1 << 24
    room(45)
    G = torch.Generator("cuda").manual_seed(5)
    x = torch.empty(rows, experts, device="cuda").normal_(generator=G).requires_grad_(True)
    idx = torch.arange(rows, device="cuda")[:, None] % (experts - 1)  # one expert gets nothing
    leave_nan(((rows, experts), torch.float32))
    loss, counts = fk.fused_moe_balance_loss(x, idx)
    (grad,) = torch.autograd.grad(loss, x)
    assert torch.isfinite(grad).all()
    at = spots(rows, experts)
    p = torch.softmax(x.detach()[at].double(), 1)
    g = counts.double() / rows - 1 / experts
    want = experts / rows * p * (g - (p * g).sum(1, keepdim=True))
    size = experts / rows * p * (g.abs() + (p * g.abs()).sum(1, keepdim=True))
    assert ((grad[at].double() - want).abs() <= 128 * 2.0 ** -24 * size + 1e-30).all()


@pytest.mark.parametrize("vocab", [131072, 131071])
def test_distillation_everywhere(vocab):
    rows = 1 << 15
    room(40)
    G = torch.Generator("cuda").manual_seed(6)
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda").normal_(generator=G)
    idx = torch.randint(0, vocab, (rows, 4), generator=G, device="cuda")
    top = torch.randn(rows, 4, generator=G, device="cuda")
    targets = torch.randint(0, vocab, (rows,), generator=G, device="cuda")
    leave_nan(((rows, vocab), torch.bfloat16))

    def run(x, idx, top, targets):
        x = x.requires_grad_(True)
        loss = fk.fused_distillation_loss(x, idx, top, targets)
        return torch.autograd.grad(loss, x)[0]

    got = run(x, idx, top, targets)
    assert torch.isfinite(got).all()
    at = spots(rows, vocab)
    at = at[torch.linspace(0, len(at) - 1, 128, device="cuda").long()]  # 2^7 rows: 1/n 2^8 apart
    want = run(x.detach()[at], idx[at], top[at], targets[at]).float()
    # The row's slices (and so the order of its sum) may be others: one step of bf16.
    assert ((got[at].float() * 2.0 ** 8 - want).abs() <= 2.0 ** -7 * want.abs() + 1e-30).all()
