"""Cases of four training operators: the residual addition with its RMS norm (forward and
backward), the same with an 8-bit output and scales, the router's balance loss with its
per-expert counts, and distillation from a teacher's top logits.

Each case runs in a plain form (elementary torch operations in 32 bits) or, where ``own`` is
true, through the framework's public functions.

    add_norm  h = round(x + r);  y = h * rsqrt(mean(h^2) + eps) * w;  gradients of x, r, w
    quant     y as above, scale = max(max|y| / 448, 2^-126) per row or per 128 columns,
              q = e4m3(y / scale)
    balance   f_e = share of the slots that go to expert e;  p = softmax(logits)
              loss = E/n sum_t sum_e f_e p_te + z/n sum_t lse_t^2, and its gradient
    distill   (1-a) T^2 KL(teacher's top entries || softmax(s/T)) + a CE(s, target), the mean
              over the counted rows, and its gradient

The gradients of the two losses are those of loss * scale, as a loss scaler in fp16 asks for.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


# ------------------------------------------------------------------ cases -------------------
def listed():
    return [
        # One decoding step of 16 sequences: forward only, where latency counts.
        dict(name="add_norm decode", op="add_norm", rows=16, cols=4096, dtype="bf16",
             res="bf16", weight="bf16", train=False),
        # The benchmark's RMSNorm batch (16384 tokens of width 4096), forward and backward.
        dict(name="add_norm train", op="add_norm", rows=16384, cols=4096, dtype="bf16",
             res="bf16", weight="fp32", train=True),
        # An odd width and row count, 16-bit activations over an fp32 residual stream.
        dict(name="add_norm odd", op="add_norm", rows=5003, cols=1111, dtype="bf16",
             res="fp32", weight="fp32", train=True),
        # A decoding step in front of an 8-bit product with one scale per token.
        dict(name="quant decode", op="quant", rows=64, cols=4096, dtype="bf16", res="bf16",
             weight="bf16", block=0),
        # A long prompt in front of an 8-bit product with a scale per 128 columns.
        dict(name="quant prefill", op="quant", rows=16384, cols=4096, dtype="bf16", res="bf16",
             weight="fp32", block=128),
        # First layer (no residual yet), ragged width: the last group of a row is short.
        dict(name="quant ragged", op="quant", rows=3001, cols=2752, dtype="fp16", res="none",
             weight="fp32", block=128),
        # The router benchmark's small size: one microbatch.
        dict(name="balance small", op="balance", rows=4096, experts=64, k=2, dtype="fp32",
             masked=False, z=0.0),
        # The router benchmark's large size.
        dict(name="balance large", op="balance", rows=131072, experts=128, k=8, dtype="fp32",
             masked=False, z=1e-3),
        # A padded batch, 16-bit logits, an odd number of experts.
        dict(name="balance padded", op="balance", rows=20011, experts=161, k=6, dtype="bf16",
             masked=True, z=1e-3),
        # A few rows of the small GPT's vocabulary: latency, and rows too few for the GPU.
        dict(name="distill small", op="distill", rows=32, vocab=32000, k=16, dtype="bf16",
             hard=False, temperature=1.0),
        # The cross-entropy benchmark's batch, teacher's top 64 mixed with the hard label.
        dict(name="distill large", op="distill", rows=8192, vocab=128256, k=64, dtype="bf16",
             hard=True, temperature=1.0),
        # An odd vocabulary in 32 bits at a raised temperature.
        dict(name="distill odd", op="distill", rows=2048, vocab=50257, k=100, dtype="fp32",
             hard=True, temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _aligned(rng, n, step):
    """Two of three widths are multiples of `step`, the others are left odd."""
    return max(step, n // step * step) if rng.random() < 0.67 else n


def draw(rng):
    op = rng.choice(["add_norm", "quant", "balance", "distill"])
    if op in ("add_norm", "quant"):
        cols = _aligned(rng, _log_int(rng, 64, 8192), 64)
        rows = _log_int(rng, 1, min(16384, 16384 * 4096 // cols))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case = dict(op=op, rows=rows, cols=cols, dtype=dtype, res=rng.choice([dtype, "fp32"]),
                    weight=rng.choice([dtype, "fp32"]))
        if op == "add_norm":
            case["train"] = rng.random() < 0.7
        else:
            case["block"] = rng.choice([0, 128])
            if rng.random() < 0.25:
                case["res"] = "none"
        return case
    if op == "balance":
        experts = _aligned(rng, _log_int(rng, 4, 256), 8)
        return dict(op=op, rows=_log_int(rng, 1, 131072), experts=experts,
                    k=rng.randint(1, min(8, experts)), dtype=rng.choice(["fp32", "bf16", "fp16"]),
                    masked=rng.random() < 0.5, z=rng.choice([0.0, 1e-3]))
    vocab = _aligned(rng, _log_int(rng, 1000, 128256), 64)
    return dict(op=op, rows=_log_int(rng, 1, 8192), vocab=vocab, k=_log_int(rng, 1, 256),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]) if vocab < 64000 else "bf16",
                hard=rng.random() < 0.5, temperature=rng.choice([1.0, 1.0, 2.0, 1.5]))


# ------------------------------------------------------------------ inputs ------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"add_norm": _prepare_norm, "quant": _prepare_norm, "balance": _prepare_balance,
            "distill": _prepare_distill}[case["op"]]
    state = make(case, g)
    state["case"] = case
    return state


def _loss_scale(case):
    """fp16 training scales its losses so that gradients do not vanish: about the number of
    rows here, which undoes the mean's division."""
    return 2.0 ** int(math.log2(case["rows"])) if case["dtype"] == "fp16" else 1.0


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_norm(case, g):
    n, d = case["rows"], case["cols"]
    dt = DTYPES[case["dtype"]]
    state = dict(
        x=_randn(g, n, d).to(dt),
        r=None if case["res"] == "none" else (2.0 * _randn(g, n, d)).to(DTYPES[case["res"]]),
        w=(1.0 + 0.1 * _randn(g, d)).to(DTYPES[case["weight"]]))
    if case.get("train"):
        state["dy"] = _randn(g, n, d).to(dt)
        state["dh"] = _randn(g, n, d).to(DTYPES[case["res"]])
        for name in "xrw":
            state[name].requires_grad_(True)
    return state


def _prepare_balance(case, g):
    n, e, k = case["rows"], case["experts"], case["k"]
    logits = _randn(g, n, e) + 0.5 * _randn(g, e)  # some experts are preferred
    logits = logits.to(DTYPES[case["dtype"]])
    idx = logits.float().topk(k, dim=1).indices
    mask = None
    if case["masked"]:  # the padding of a batch of unequal sequences: about a fifth
        mask = torch.rand(n, generator=g, device="cuda") < 0.8
    scale = torch.tensor(_loss_scale(case), device="cuda")
    return dict(logits=logits.requires_grad_(True), idx=idx, mask=mask, scale=scale)


def _prepare_distill(case, g):
    n, v = case["rows"], case["vocab"]
    k = min(case["k"], v)
    dt = DTYPES[case["dtype"]]
    logits = torch.empty(n, v, dtype=dt, device="cuda")
    idx = torch.empty(n, k, dtype=torch.int64, device="cuda")
    top = torch.empty(n, k, dtype=dt, device="cuda")
    for a in range(0, n, 1024):  # the teacher agrees with the student in part
        s = 2.5 * _randn(g, min(1024, n - a), v)
        logits[a:a + 1024] = s.to(dt)
        vals, idx[a:a + 1024] = (0.8 * s + 1.5 * _randn(g, s.shape[0], v)).topk(k, dim=1)
        top[a:a + 1024] = vals.to(dt)
    used = torch.randint(max(1, k // 2), k + 1, (n, 1), generator=g, device="cuda")
    idx.masked_fill_(torch.arange(k, device="cuda")[None] >= used, -1)  # fewer kept: top-p
    targets = None
    dropped = torch.rand(n, generator=g, device="cuda") < 0.05
    if case["hard"]:
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        targets.masked_fill_(dropped, -100)
    elif n > 1:
        idx.masked_fill_(dropped[:, None], -1)  # rows without a teacher
    scale = torch.tensor(_loss_scale(case), device="cuda")
    return dict(logits=logits.requires_grad_(True), idx=idx, top=top, targets=targets,
                scale=scale)


# ------------------------------------------------------------------ one pass ----------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"add_norm": _own_norm, "quant": _own_quant, "balance": _own_balance,
                "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"add_norm": _plain_norm, "quant": _plain_quant, "balance": _plain_balance,
                "distill": _plain_distill}[op](state)


def _own_norm(s):
    from fusedkernels_b200 import fused_add_rms_norm
    if not s["case"]["train"]:
        with torch.no_grad():
            return fused_add_rms_norm(s["x"], s["r"], s["w"], EPS)
    y, h = fused_add_rms_norm(s["x"], s["r"], s["w"], EPS)
    grads = torch.autograd.grad((y, h), (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
    return y, h, *grads


def _own_quant(s):
    from fusedkernels_b200 import fused_add_rms_norm_quant
    out = fused_add_rms_norm_quant(s["x"], s["r"], s["w"], EPS, block=s["case"]["block"] or None)
    return out if s["r"] is not None else out[:2]


def _own_balance(s):
    from fusedkernels_b200 import fused_moe_balance_loss
    loss, counts = fused_moe_balance_loss(s["logits"], s["idx"], token_mask=s["mask"],
                                          z_coef=s["case"]["z"],
                                          loss_scale=_loss_scale(s["case"]))
    (grad,) = torch.autograd.grad(loss, s["logits"], s["scale"])
    return loss, counts, grad


def _own_distill(s):
    from fusedkernels_b200 import fused_distillation_loss
    loss = fused_distillation_loss(s["logits"], s["idx"], s["top"], targets=s["targets"],
                                   temperature=s["case"]["temperature"], hard_weight=0.5,
                                   loss_scale=_loss_scale(s["case"]))
    (grad,) = torch.autograd.grad(loss, s["logits"], s["scale"])
    return loss, grad


def _plain_sum_norm(s):
    x = s["x"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(s["r"].dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    return h, hf, rstd


def _plain_norm(s):
    h, hf, rstd = _plain_sum_norm(s)
    wf = s["w"].float()
    y = (hf * rstd * wf).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y, h
    dy = s["dy"].float()
    wdy = dy * wf
    c = (wdy * hf).mean(1, keepdim=True) * rstd * rstd * rstd
    g = s["dh"].float() + wdy * rstd - hf * c
    dw = (dy * hf * rstd).sum(0)
    return y, h, g.to(s["x"].dtype), g.to(s["r"].dtype), dw.to(s["w"].dtype)


def _plain_quant(s):
    h, hf, rstd = _plain_sum_norm(s)
    y = hf * rstd * s["w"].float()
    n, d = y.shape
    b = s["case"]["block"] or d
    groups = -(-d // b)
    yg = torch.zeros(n, groups * b, device=y.device)
    yg[:, :d] = y
    yg = yg.view(n, groups, b)
    scale = (yg.abs().amax(2) / E4M3_MAX).clamp(min=MIN_SCALE)
    q = (yg / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(n, groups * b)[:, :d]
    q = q.to(torch.float8_e4m3fn)
    return (q, scale, h) if s["r"] is not None else (q, scale)


def _plain_balance(s):
    logits, idx, mask = s["logits"].float(), s["idx"], s["mask"]
    n_rows, experts = logits.shape
    valid = torch.ones(n_rows, dtype=torch.bool, device=logits.device) if mask is None else mask
    counts = torch.zeros(experts, dtype=torch.int64, device=logits.device)
    counts.index_add_(0, idx.reshape(-1), valid[:, None].expand_as(idx).reshape(-1).long())
    f = counts.float() / counts.sum().clamp(min=1)
    n = valid.sum().clamp(min=1).float()
    m = logits.amax(1, keepdim=True)
    e = torch.exp(logits - m)
    z = e.sum(1, keepdim=True)
    p = e / z
    lse = m + torch.log(z)
    share = (p * f).sum(1, keepdim=True)
    zc = s["case"]["z"]
    rows = torch.where(valid[:, None], experts * share + zc * lse * lse, torch.zeros_like(share))
    loss = (rows.double().sum() / n).float()
    grad = p * (experts * (f - share) + 2.0 * zc * lse) / n * s["scale"]
    grad = torch.where(valid[:, None], grad, torch.zeros_like(grad))
    return loss, counts, grad.to(s["logits"].dtype)


def _plain_softmax(x):
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    return e.div_(z), m + torch.log(z)


def _plain_distill(s):
    case = s["case"]
    t = case["temperature"]
    logits, idx, targets = s["logits"], s["idx"], s["targets"]
    a = 0.5 if targets is not None else 0.0
    used = idx >= 0
    some = used.any(1, keepdim=True)
    valid = some[:, 0] if targets is None else targets != -100
    n = valid.sum().clamp(min=1).float()
    teacher = torch.where(used, s["top"].float() / t, torch.full_like(idx, -1, dtype=torch.float32))
    teacher = teacher.masked_fill(~used, -1e30)
    m = teacher.amax(1, keepdim=True)
    e = torch.where(used, torch.exp(teacher - m), torch.zeros_like(teacher))
    z = e.sum(1, keepdim=True).clamp(min=1e-30)
    p, logp = e / z, teacher - m - torch.log(z)
    at = idx.clamp(min=0)
    x = logits.float()
    picked = x.gather(1, at) / t
    q, lse = _plain_softmax(x / t)
    kl = torch.where(used, p * (logp - picked + lse), torch.zeros_like(p)).sum(1)
    rows = (1.0 - a) * t * t * kl
    grad = q.mul_(torch.where(some, 1.0, 0.0))
    grad.scatter_add_(1, at, -torch.where(used, p, torch.zeros_like(p)))
    grad.mul_((1.0 - a) * t)
    if targets is not None:
        y = targets.clamp(min=0)[:, None]
        hit = x.gather(1, y)[:, 0]
        q1, lse1 = _plain_softmax(x)
        rows = rows + a * (lse1[:, 0] - hit)
        grad.add_(q1, alpha=a)
        grad.scatter_add_(1, y, torch.full_like(y, -a, dtype=torch.float32))
    rows = torch.where(valid, rows, torch.zeros_like(rows))
    grad.mul_(s["scale"] / n).masked_fill_(~valid[:, None], 0.0)
    return (rows.double().sum() / n).float(), grad.to(logits.dtype)


# ------------------------------------------------------------------ floors ------------------
def work(case):
    """Bytes and operations of one pass: every input read and every output written once."""
    size = {"fp32": 4, "fp16": 2, "bf16": 2, "none": 0}
    es = size[case["dtype"]]
    if case["op"] in ("add_norm", "quant"):
        n, d = case["rows"], case["cols"]
        rs, ws = size[case["res"]], size[case["weight"]]
        if case["op"] == "quant":
            groups = -(-d // (case["block"] or d))
            return {"bytes": n * d * (es + 2 * rs + 1) + 4 * n * groups + d * ws,
                    "flops": 7.0 * n * d}
        moved = n * d * (2 * es + 2 * rs) + d * ws
        if not case["train"]:
            return {"bytes": moved, "flops": 5.0 * n * d}
        # dy, dh in; the gradient out, once if both inputs have one type
        back = n * d * (es + rs + (es if es == rs else es + rs)) + d * ws
        return {"bytes": moved + back, "flops": 15.0 * n * d}
    if case["op"] == "balance":
        n, e = case["rows"], case["experts"]
        return {"bytes": 2 * n * e * es + 8 * n * case["k"] + 8 * e + (n if case["masked"] else 0),
                "flops": 10.0 * n * e}
    n, v, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
    two = 2.0 if case["hard"] and case["temperature"] != 1.0 else 1.0
    return {"bytes": 2 * n * v * es + n * k * (8 + es) + (8 * n if case["hard"] else 0),
            "flops": 8.0 * n * v * two}


# ------------------------------------------------------------------ 64 bits -----------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"add_norm": _exact_norm, "quant": _exact_quant, "balance": _exact_balance,
                "distill": _exact_distill}[case["op"]](state)


def _exact_normed(s):
    h = s["x"].detach()
    if s["r"] is not None:
        h = torch.add(h.double(), s["r"].double()).to(s["r"].dtype)  # the stream's own rounding
    d = h.shape[1]
    length = torch.linalg.vector_norm(h.double(), dim=1, keepdim=True).square() / d + EPS
    unit = h.double() / length.sqrt()
    return h, length.sqrt(), unit


def _exact_norm(s):
    h, root, unit = _exact_normed(s)
    w = s["w"].double()
    y = torch.mul(unit, w)
    if not s["case"]["train"]:
        return y, h.double()
    up = s["dy"].double() * w  # gradient of the unit rows, projected off the rows themselves
    along = torch.einsum("nd,nd->n", up, unit)[:, None] / h.shape[1]
    g = s["dh"].double() + (up - unit * along) / root
    dw = torch.einsum("nd,nd->d", s["dy"].double(), unit)
    return y, h.double(), g, g, dw


def _exact_quant(s):
    h, _, unit = _exact_normed(s)
    y = unit * s["w"].double()
    b = s["case"]["block"] or y.shape[1]
    parts = y.split(b, dim=1)
    scale = torch.stack([p.abs().max(dim=1).values for p in parts], 1) / E4M3_MAX
    scale = torch.clamp_min(scale, MIN_SCALE)
    q = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], 1)
    return (q, scale, h.double()) if s["r"] is not None else (q, scale)


def _exact_balance(s):
    x = s["logits"].detach().double()
    n_rows, experts = x.shape
    keep = slice(None) if s["mask"] is None else s["mask"]
    kept, slots = x[keep], s["idx"][keep].reshape(-1)
    counts = torch.bincount(slots, minlength=experts)
    f = counts.double() / max(1, slots.numel())
    n = max(1, kept.shape[0])
    logp = torch.log_softmax(kept, 1)
    lse = torch.logsumexp(kept, 1)
    p = logp.exp()
    z = s["case"]["z"]
    loss = experts * torch.dot(f, p.sum(0)) / n + z * lse.square().sum() / n
    up = experts * f  # d loss / d p, times n
    inner = p * (up[None] - torch.mv(p, up)[:, None]) + 2.0 * z * lse[:, None] * p
    grad = torch.zeros_like(x)
    grad[keep] = inner * (_loss_scale(s["case"]) / n)
    return loss, counts, grad


def _exact_distill(s):
    t = s["case"]["temperature"]
    logits, idx, targets = s["logits"].detach(), s["idx"], s["targets"]
    n_rows, v = logits.shape
    a = 0.0 if targets is None else 0.5
    valid = (idx >= 0).any(1) if targets is None else targets.ne(-100)
    n = max(1, int(valid.sum()))
    grad = torch.zeros(n_rows, v, dtype=torch.float64, device=logits.device)
    loss = torch.zeros((), dtype=torch.float64, device=logits.device)
    for at in range(0, n_rows, 1024):
        rows = valid[at:at + 1024].nonzero()[:, 0] + at
        x, slots = logits[rows].double(), idx[rows]
        held = slots.ge(0).any(1)
        scores = (s["top"][rows].double() / t).masked_fill(slots < 0, -math.inf)
        scores[~held] = 0.0
        dense = torch.zeros_like(x)
        probs = torch.softmax(scores, 1).masked_fill(slots < 0, 0.0)
        dense.scatter_add_(1, slots.clamp(min=0), probs)
        logq = torch.log_softmax(x / t, 1)
        entropy = torch.special.xlogy(probs, probs).sum(1)
        kl = entropy - (dense * logq).sum(1)
        loss += (1.0 - a) * t * t * kl[held].sum()
        part = (logq.exp() * held[:, None] - dense) * ((1.0 - a) * t)
        if targets is not None:
            y = targets[rows]
            logq = torch.log_softmax(x, 1)
            loss -= a * logq.gather(1, y[:, None]).sum()
            hard = logq.exp()
            hard[torch.arange(len(rows), device=y.device), y] -= 1.0
            part += a * hard
        grad[rows] = part * (_loss_scale(s["case"]) / n)
    return loss / n, grad
