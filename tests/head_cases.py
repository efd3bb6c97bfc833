"""Inputs, a plain 64-bit form and derived tolerances for the head's losses (cross entropy and distillation through
the head), shared by the CPU and the GPU tests. torch in float64, on whatever device the inputs are."""
import torch

from presk_b200 import abi

TORCH = {abi.BF16: torch.bfloat16, abi.F16: torch.float16, abi.F32: torch.float32}
CODE = {v: k for k, v in TORCH.items()}
#: half a step of a type, relative to the value
HALF = {abi.BF16: 2.0**-8, abi.F16: 2.0**-11, abi.F32: 2.0**-24}
#: the least step of a type (subnormal spacing): half of it is the error near zero
LEAST = {abi.BF16: 0.0, abi.F16: 2.0**-24, abi.F32: 0.0}


def make(outer, vocab, model, dtype, top=0, tau=1.0, vocab_major=False, ignored=0.2, seed=0, device="cpu", spread=2.0, teacher=None, pad=0):
    """Rows that lean towards their label, a head, targets of which `ignored` have none. `pad`: elements between x's rows."""
    g = torch.Generator().manual_seed(seed)
    dt = TORCH[dtype]
    rows = 1
    for n in outer:
        rows *= n
    w = torch.randn(vocab, model, generator=g) * (spread / model**0.5)
    label = torch.randint(0, vocab, (rows,), generator=g)
    x = torch.randn(rows, model + pad, generator=g)
    if rows:
        x[:, :model] += 1.5 * w[label]
    gone = torch.rand(rows, generator=g) < ignored
    s = dict(outer=tuple(outer), vocab=vocab, model=model, dtype=dtype, top=top, tau=tau, vocab_major=vocab_major)
    s["x"] = x.to(dt).reshape(*outer, model + pad)[..., :model] if not pad else x.to(dt).to(device).reshape(*outer, model + pad)[..., :model]
    s["w"] = (w if vocab_major else w.t().contiguous()).to(dt)
    s["ct"] = torch.rand(rows, generator=g).reshape(outer) / max(1, rows) + 0.25 / max(1, rows)
    if not top:
        s["labels"] = torch.where(gone, torch.full_like(label, -1), label).reshape(outer)
    else:
        ids = torch.stack([torch.randperm(vocab, generator=g)[:top] if top <= vocab else torch.randint(0, vocab, (top,), generator=g) for _ in range(rows)]) if rows else torch.zeros(0, top, dtype=torch.int64)
        if rows and top > 1:
            ids[::3, top - 1] = ids[::3, 0]  # a class named twice
            ids[1::4, top // 2:] = -1  # a shorter list
        ids[gone] = -1
        t = 2.0 * torch.randn(rows, top, generator=g)
        if rows > 2 and top > 1:
            t[2, 1] = -float("inf")
        s["ids"], s["teacher"] = ids.reshape(*outer, top), t.to(TORCH[teacher or abi.F32]).reshape(*outer, top)
    for k, v in s.items():
        if isinstance(v, torch.Tensor):
            s[k] = v.to(device)
    return s


def targets(s):
    """(distribution [rows, vocab], its entropy, whether a row has a target), in 64 bits."""
    rows, v = s["ct"].numel(), s["vocab"]
    q = torch.zeros(rows, v, dtype=torch.float64, device=s["w"].device)
    if not s["top"]:
        y = s["labels"].reshape(-1)
        q.scatter_add_(1, y.clamp(min=0)[:, None], (y >= 0).double()[:, None])
        return q, torch.zeros(rows, dtype=torch.float64, device=q.device), y >= 0
    ids, t = s["ids"].reshape(rows, -1), s["teacher"].double().reshape(rows, -1) / s["tau"]
    t = torch.where(ids < 0, -float("inf"), t)
    has = (t > -float("inf")).any(1)
    t = t - torch.where(has, t.amax(1), 0.0)[:, None]  # first: at the types' lowest values a log-sum-exp has no digits after the point left
    logp = torch.where(has[:, None], t - torch.logsumexp(torch.where(has[:, None], t, 0.0), 1, keepdim=True), -float("inf"))
    p = logp.exp()
    q.scatter_add_(1, ids.clamp(min=0), p)
    return q, -torch.where(p > 0, p * logp, 0.0).sum(1), has


def plain(s, lse_in=None):
    """loss, lse, dx, dw and bounds of a kernel's error for each (see `bounds`)."""
    rows, dt, tau = s["ct"].numel(), s["dtype"], s["tau"]
    x = s["x"].reshape(rows, s["model"]).double()
    w = s["w"].double() if s["vocab_major"] else s["w"].double().t()
    q, entropy, has = targets(s)
    x = torch.where(has[:, None], x, 0.0)
    z = x @ w.t() / tau
    lse = torch.logsumexp(z, 1)
    loss = torch.where(has, (q * (lse[:, None] - z)).sum(1) - entropy, 0.0)
    lse = torch.where(has, lse, 0.0)
    ct = torch.where(has, s["ct"].reshape(-1).double(), 0.0) / tau
    e = torch.where(has[:, None], torch.exp(z - lse[:, None]), 0.0)
    g = (e - q) * ct[:, None]
    # A logit's error. An accumulator holds up to 512 products of the summed axis: 32 matrix instructions of 16
    # (24 for the planes of f32) that each add by truncation, below 2^-23 of a partial sum, itself at most
    # the sum of |x w|; those partial sums are then added rounded to nearest.
    absum = x.abs() @ w.abs().t() / tau
    chunks = (s["model"] + 63) // 64
    el = absum * (32 * 2.0**-23 + (chunks + 4) * 2.0**-24) + 1e-30
    small = 2.0**-39  # of the greatest element: half binary16's least step, when the greatest is scaled to 2^14 or more
    if dt == abi.F32 and x.numel():
        # two binary16 planes: each operand to 2^-23 (its second plane's half step), lo·lo left out, below 2^-22
        el = el + absum * 2.0**-21 + small * (x.abs().amax(1, keepdim=True) * w.abs().sum(1)[None] + w.abs().amax() * x.abs().sum(1, keepdim=True)) / tau
    el_row = el.amax(1) if rows and s["vocab"] else torch.zeros(rows, dtype=torch.float64, device=x.device)
    # the exponentials' sum: 2^-22 a term (the hardware's), 34 additions a thread and as many as there are parts; the
    # exponent's product and differences round once each
    ez = 2.0**-22 + (40 + s["vocab"] // 128) * 2.0**-24 + z.abs().amax(1) * 2.0**-23
    b_lse = el_row + ez + lse.abs() * 2.0**-23
    # the loss adds logits weighted by p, and the teacher's own sum: p to 2^-21 (expf, a division), |ln p| up to the list's spread
    spread = (q.sum(1) * (z.abs().amax(1) + 40)) * (2.0**-21 if s["top"] else 0.0)
    b_loss = b_lse + el_row + (z.abs().amax(1) + lse.abs()) * 2.0**-22 + spread
    b_lse, b_loss = (torch.where(has, b, 0.0) for b in (b_lse, b_loss))
    # gradients: g's own error (e from a logit and a log-sum-exp that are off by b_lse and el; p), its rounding to the
    # operands' type, then a sum of products by truncation (as above, chunks of 256) and the result's rounding
    eg = ct.abs()[:, None] * (e * (el + b_lse[:, None] + ez[:, None]) + q * 2.0**-20) + g.abs() * (HALF[dt] + 2.0**-22)
    if dt != abi.F32 or not x.numel():
        planes = 0.0
    else:
        planes = 2.0**-21  # of a product, as above
    if x.numel():
        eg = eg + torch.where(has[:, None], ct.abs().amax() * 2 * small, 0.0)  # g in binary16 is scaled by the greatest ct
    dx, dw = g @ w, g.t() @ x
    # one accumulator throughout: truncation below 2^-23 of a partial sum an instruction of 16
    acc = (max(s["vocab"], 2 * rows) // 16 + 8) * 2.0**-23 + planes
    low = small * (g.abs().sum(1, keepdim=True) * w.abs().amax() if x.numel() else 0.0)  # copies of w and x in binary16
    # of x where a row's ct is 2^-k of the greatest: its copy is scaled by 2^(k/2) less (k counts powers of two: at most
    # one more than the quotient's)
    less = torch.sqrt(2 * ct.abs().amax() / ct.abs().clamp(min=1e-300)) if x.numel() else ct
    less = torch.where(ct == 0, 1.0, less)
    low_w = small * ((g.abs() * (1 + 2 * less)[:, None]).sum(0)[:, None] * x.abs().amax() if x.numel() else 0.0)
    b_dx = eg @ w.abs() + acc * (g.abs() @ w.abs()) + low + dx.abs() * HALF[dt] * 1.01 + LEAST[dt]
    b_dw = eg.t() @ x.abs() + acc * (g.abs().t() @ x.abs()) + low_w + dw.abs() * HALF[dt] * 1.01 + LEAST[dt]
    if not s["vocab_major"]:
        dw, b_dw = dw.t(), b_dw.t()
    shape = s["ct"].shape
    out = {"loss": loss.reshape(shape), "lse": lse.reshape(shape), "dx": dx.reshape(*shape, s["model"]), "dw": dw}
    tol = {"loss": b_loss.reshape(shape), "lse": b_lse.reshape(shape), "dx": b_dx.reshape(*shape, s["model"]), "dw": b_dw}
    return out, tol


def launches(s, loss_dtype=abi.F32, ct_dtype=abi.F32, **more):
    """The two launches of a case, and the order of their inputs."""
    import presk_b200
    kw = dict(outer=s["outer"], vocab=s["vocab"], model=s["model"], dtype=s["dtype"], x_strides=s["x"].stride(), vocab_major=s["vocab_major"], top=s["top"], temperature=s["tau"])
    if s["top"]:
        kw["teacher_dtype"] = CODE[s["teacher"].dtype]
    kw.update(more)
    return presk_b200.head_loss_launch(loss_dtype=loss_dtype, **kw), presk_b200.head_loss_vjp_launch(ct_dtype=ct_dtype, **kw)


def given(s):
    return [s["x"], s["w"]] + ([s["ids"], s["teacher"]] if s["top"] else [s["labels"]])
