"""64-bit restatements of the training operators around the reference's ops (add + RMSNorm and
its 8-bit form, the router's balance loss, distillation), with the magnitudes that error bounds
are made of.  CPU tensors, plain PyTorch."""
import torch

U = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    """Relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Absolute error of one rounding among the subnormals (twice half a step)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound elementwise; NaN and infinities have to be the same."""
    got, want = got.detach().cpu().double(), want.double()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: finite in other places"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    over = (got - want).abs() - bound
    over[~fine] = -1.0
    if over.numel() and over.max() > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: {got.reshape(-1)[i].item()!r} for "
                             f"{want.reshape(-1)[i].item()!r}, off by more than "
                             f"{bound.reshape(-1)[i].item():.3g} ({int((over > 0).sum())} of "
                             f"{over.numel()})")


def add_norm(x, r, w, eps, dy=None, dh=None):
    """y, h and with dy the gradient g of both inputs and dw, each with its error bound:
    {name: (value, bound without the last rounding)}.  h is the rounded sum."""
    h = (x.float() + r.float()).to(r.dtype) if r is not None else x
    d = h.shape[-1]
    hd, wd = h.double(), w.double()
    s = torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + eps)
    # A row's sum: at most cols/256 additions by one thread, then 5 + 32 over the CTA; halved by
    # the root, then rsqrtf (2 ulp) and two products.
    f = (d / 256 + 40) * U
    y = hd * s * wd
    out = {"h": (h, 0.0), "y": (y, f * y.abs())}
    if dy is not None:
        dyd = dy.double()
        dhd = torch.zeros_like(hd) if dh is None else dh.double()
        a = s * wd * dyd
        c = s.pow(3) * (wd * dyd * hd).mean(-1, keepdim=True)
        c_abs = s.pow(3) * (wd * dyd * hd).abs().mean(-1, keepdim=True)
        out["g"] = (dhd + a - hd * c, 4 * f * (dhd.abs() + a.abs() + hd.abs() * c_abs))
        rows = hd.reshape(-1, d).shape[0]
        t = (dyd * hd * s).reshape(-1, d)
        out["dw"] = (t.sum(0), (rows / 148 + 100 + f / U) * U * t.abs().sum(0))
    return out


def balance(logits, idx, mask, z_coef, loss_scale=1.0):
    """loss, counts, gradient and the bounds of loss and gradient (without the rounding)."""
    x = logits.double()
    n_rows, e = x.shape
    keep = torch.ones(n_rows, dtype=torch.bool) if mask is None else mask
    used = keep[:, None] & (idx >= 0)
    counts = torch.bincount(idx[used], minlength=e)
    f = counts.double() / max(1, int(counts.sum()))
    n = max(1, int(keep.sum()))
    full = (x > -float("inf")).any(1) | x.isnan().any(1)
    p = torch.where(full[:, None], torch.softmax(x, 1), torch.zeros_like(x))
    lse = torch.where(full, torch.logsumexp(x, 1), torch.zeros(n_rows, dtype=torch.float64))
    p, lse = p * keep[:, None], lse * keep
    share = (p * f).sum(1)
    loss = (e * share.sum() + z_coef * (lse * lse).sum()) / n
    ce, cz = e * loss_scale / n, 2 * z_coef * loss_scale / n
    grad = p * (ce * (f - share[:, None]) + cz * lse[:, None])
    size = p * (ce * (f + share[:, None]) + cz * lse.abs()[:, None])
    finite = x[torch.isfinite(x)]
    far = float(finite.abs().max()) if finite.numel() else 0.0
    # exp: 2 ulp plus the rounding of its argument (2 far at most); sums of at most 256 terms in
    # a tree of depth 13; reciprocal, products and lse within 32 roundings.
    b = (64 + 4 * far) * U
    return loss, counts, grad, b * loss.abs(), b * size


def distill(logits, idx, top, targets, temperature=1.0, hard_weight=0.5, ignore_index=-100,
            loss_scale=1.0):
    """loss, gradient and the bounds of both (without the rounding)."""
    x = logits.double()
    n_rows, v = x.shape
    a = 0.0 if targets is None else hard_weight
    t = temperature
    used = idx >= 0
    scores = (top.double() / t).masked_fill(~used, -float("inf"))
    held = ((scores > -float("inf")) | scores.isnan()).any(1)
    valid = held if targets is None else targets != ignore_index
    n = max(1, int(valid.sum()))
    grad, size = torch.zeros_like(x), torch.zeros_like(x)
    loss = loss_size = torch.zeros((), dtype=torch.float64)
    for i in range(n_rows):
        if not valid[i]:
            continue
        ids = idx[i][used[i]]
        bad = (ids >= v).any() or (targets is not None and not 0 <= targets[i] < v)
        if bad:
            grad[i] = float("nan")
            loss = loss + float("nan")
            continue
        if held[i] and a < 1.0:
            p = torch.softmax(scores[i][used[i]], 0)
            lse = torch.logsumexp(x[i] / t, 0)
            pos = ~(p <= 0)
            logq = (x[i] / t)[ids] - lse
            row = (p[pos] * (p[pos].log() - logq[pos])).sum()
            loss = loss + (1 - a) * t * t * row
            loss_size = loss_size + (1 - a) * t * t * (
                (p[pos] * (p[pos].log().abs() + (x[i] / t)[ids][pos].abs())).sum() + lse.abs() + 1)
            q = torch.softmax(x[i] / t, 0)
            dense = torch.zeros(v, dtype=torch.float64).index_add_(0, ids, p)
            grad[i] += (1 - a) * t * (q - dense)
            size[i] += (1 - a) * t * (q + dense)
        if targets is not None and a > 0.0:
            y = int(targets[i])
            lse = torch.logsumexp(x[i], 0)
            loss = loss + a * (lse - x[i, y])
            loss_size = loss_size + a * (lse.abs() + x[i, y].abs() + 1)
            q = torch.softmax(x[i], 0)
            grad[i] += a * q
            grad[i, y] -= a
            size[i] += a * q
            size[i, y] += a
    finite = x[torch.isfinite(x)]
    far = float(finite.abs().max()) if finite.numel() else 0.0
    # A row's sum: at most v/256 additions by one thread, then a tree; each exponential has 4 ulp
    # and the rounding of its argument (up to 2 far / T, in units of log2 as well).
    b = (v / 256 + 4 * far / min(t, 1.0) + 64) * U
    return loss / n, grad * (loss_scale / n), b * loss_size / n, b * size * (loss_scale / n)
