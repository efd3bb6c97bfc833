"""The head's losses where the Llama program uses them: `loss`, `loss_grad`, `distill`, `distill_grad` under the declared
order `loss: pieces`, on the CPU oracle and on the GPU, against a float64 statement of the model."""
import numpy as np
import pytest
import torch

import models
from presk_b200 import Host, PreskError

PIECES = {"kind": "device", "loss": "pieces"}


def llama_hidden(t, c, ids):
    """The decoder of examples/coverage/llama.psk up to its last norm, in the type of the tensors of `t`."""
    D, H, L = c["D"], c["H"], c["L"]
    G = c.get("G", H)
    HD, P = D // H, H // G
    B, T = ids.shape
    x = t["tok"][torch.tensor(ids)]
    rms = lambda g, x: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * g
    phi = torch.arange(T, dtype=torch.float64)[:, None] * torch.exp(-2.0 * torch.arange(HD // 2, dtype=torch.float64) / HD * np.log(1e4))[None, :]
    cs, sn = torch.cos(phi), torch.sin(phi)

    def rope(x):
        x0, x1 = x[..., : HD // 2], x[..., HD // 2:]
        return torch.cat([x0 * cs - x1 * sn, x1 * cs + x0 * sn], -1)

    mask = torch.tril(torch.ones((T, T), dtype=torch.bool))
    for l in range(L):
        h = rms(t["blocks.n1.γ"][l], x)
        q = rope((h @ t["blocks.attn.wq"][l]).reshape(B, T, G, P, HD).permute(0, 2, 3, 1, 4))
        k = rope((h @ t["blocks.attn.wk"][l]).reshape(B, T, G, HD).permute(0, 2, 1, 3))
        v = (h @ t["blocks.attn.wv"][l]).reshape(B, T, G, HD)
        a = torch.softmax((torch.einsum("bgpsh,bgth->bgpst", q, k) / np.sqrt(HD)).masked_fill(~mask, -np.inf), -1)
        x = x + torch.einsum("bgpst,btgh->bsgph", a, v).reshape(B, T, D) @ t["blocks.attn.wo"][l]
        h = rms(t["blocks.n2.γ"][l], x)
        g = h @ t["blocks.ff.gate.w"][l]
        x = x + ((g * torch.sigmoid(g)) * (h @ t["blocks.ff.up.w"][l])) @ t["blocks.ff.down.w"][l]
    return rms(t["norm.γ"], x)


def autograd(p, c, ids, y=None, classes=None, teacher=None, tau=1.0):
    t = {k: torch.tensor(np.asarray(v, np.float64), requires_grad=True) for k, v in p.items()}
    logits = llama_hidden(t, c, ids) @ t["head"]
    logq = torch.log_softmax(logits / tau, -1)
    if y is not None:
        y = torch.tensor(y)
        row = -torch.gather(logq, -1, y.clamp(min=0)[..., None])[..., 0] * (y >= 0)
    else:
        classes, teacher = torch.tensor(classes), torch.tensor(np.asarray(teacher, np.float64)) / tau
        has = (classes >= 0).any(-1, keepdim=True)
        logp = torch.log_softmax(torch.where(has, teacher.masked_fill(classes < 0, -np.inf), torch.zeros_like(teacher)), -1)
        p_ = torch.where((classes >= 0) & has, logp.exp(), torch.zeros_like(teacher))
        row = (torch.where(p_ > 0, p_ * logp, torch.zeros_like(p_)) - p_ * torch.gather(logq, -1, classes.clamp(min=0))).sum(-1)
    loss = row.mean()
    loss.backward()
    return float(loss.detach()), {k: v.grad.numpy() for k, v in t.items()}


def inputs(c, seed, b, t, top=4):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, c["V"], size=(b, t), dtype=np.int64)
    y = rng.integers(0, c["V"], size=(b, t), dtype=np.int64)
    classes = np.stack([np.stack([rng.permutation(c["V"])[:top] for _ in range(t)]) for _ in range(b)]).astype(np.int64)
    teacher = (2 * rng.standard_normal((b, t, top))).astype(np.float32)
    classes[0, 1, 2:] = -1
    classes[b - 1, 0] = -1
    y[0, 2] = -1  # a padded position
    return ids, y, classes, teacher


def within(h, want, atol):
    for k, w in want.items():
        got = h.result(k, w.shape)
        assert np.isfinite(got).all(), k
        assert np.abs(got - w).max() <= atol * np.abs(w).max(), (k, np.abs(got - w).max() / np.abs(w).max())


def check_f32(executor, c, b, t, atol):
    p = models.llama_params(c, seed=4, std=0.2)
    ids, y, classes, teacher = inputs(c, 3, b, t)
    h = models.give(Host(executor, {"default": "f32", "order": PIECES}).prepare("llama", TEMP=2, **c), p)
    h.set_logging(True)
    loss, grads = autograd(p, c, ids, y)
    assert float(h.call("loss", [ids, y], ())) == pytest.approx(loss, rel=2e-6)
    assert "head_xent[pieces]" in h.launch_log() and "cross_entropy" not in h.launch_log()
    h.call("loss_grad", [ids, y], p["tok"].shape)
    log = h.launch_log()
    assert "head_xent[pieces]" in log and "head_xent_vjp[pieces]" in log and "cross_entropy_vjp" not in log
    within(h, grads, atol)
    loss, grads = autograd(p, c, ids, classes=classes, teacher=teacher, tau=2.0)
    assert float(h.call("distill", [ids, classes, teacher], ())) == pytest.approx(loss, rel=4e-6)
    h.call("distill_grad", [ids, classes, teacher], p["tok"].shape)
    assert "head_distill_vjp[pieces]" in h.launch_log()
    within(h, grads, atol)


def test_pieces_on_the_oracle(oracle):
    # the tolerances of the same program's gradient with the logits stored (tests/test_llama_grad_cpu.py)
    check_f32(oracle.vtable(), dict(V=50, D=32, H=4, G=2, FF=48, L=3), 2, 12, 3e-5)


@pytest.mark.gpu
def test_pieces_on_the_gpu(cuda):
    check_f32(cuda, dict(V=50, D=32, H=4, G=2, FF=48, L=3), 2, 12, 3e-5)
    check_f32(cuda, dict(V=515, D=64, H=4, G=2, FF=96, L=2), 3, 50, 3e-5)


def test_what_pieces_leaves_as_it_was(oracle):
    """Without the word, and where the launch is declined (e8m15 operands), the launch list and the bits are the old ones."""
    c = models.LLAMA_TINY
    p = models.llama_params(c, seed=4, std=0.2)
    rng = np.random.default_rng(3)
    ids, y = (rng.integers(0, c["V"], size=(2, 12), dtype=np.int64) for _ in range(2))
    runs = []
    for default, order in (("e8m15", {"kind": "device"}), ("e8m15", PIECES)):
        h = models.give(Host(oracle.vtable(), {"default": default, "order": order}).prepare("llama", **c), p)
        h.set_logging(True)
        out = h.call("loss", [ids, y], ())
        h.call("loss_grad", [ids, y], p["tok"].shape)
        runs.append((float(out), h.launch_log(), [h.result(k, np.shape(v)) for k, v in p.items()]))
    assert runs[0][0] == runs[1][0] and runs[0][1] == runs[1][1]
    for a, b in zip(runs[0][2], runs[1][2]):
        assert np.array_equal(a, b)


def test_calibration_keeps_the_launches_apart(oracle):
    """The logits' site has an envelope only where it is stored."""
    c = models.LLAMA_TINY
    p = models.llama_params(c, seed=4, std=0.2)
    rng = np.random.default_rng(3)
    ids, y = (rng.integers(0, c["V"], size=(2, 12), dtype=np.int64) for _ in range(2))
    h = models.give(Host(oracle.vtable(), {"default": "f32", "order": PIECES}).prepare("llama", **c), p)
    h.set_calibrating(True)
    h.call("loss", [ids, y], ())
    assert "Llama.apply/%11" in h.envelope()


def test_refused_realizations(oracle):
    for order, words in (({"kind": "sequential", "loss": "pieces"}, "part of the order `device`"), ({"kind": "device", "loss": "tiles"}, "logits, pieces")):
        with pytest.raises(PreskError, match=words):
            Host(oracle.vtable(), {"default": "f32", "order": order})
    c = models.LLAMA_TINY
    p = models.llama_params(c)
    h = models.give(Host(oracle.vtable(), "f32").prepare("llama", **c), p)
    ids, y, classes, teacher = inputs(c, 3, 2, 6)
    for entry in ("distill", "distill_grad"):
        with pytest.raises(PreskError, match="pieces of the vocabulary"):
            h.call(entry, [ids, classes, teacher], p["tok"].shape if "grad" in entry else ())
    h = models.give(Host(oracle.vtable(), {"default": "f32", "order": PIECES}).prepare("llama", **c), p)
    with pytest.raises(PreskError, match="takes 3 inputs"):
        h.call("distill", [ids, classes], ())
    with pytest.raises(PreskError, match="teacher's classes"):
        h.call("distill", [ids, classes, teacher[..., :2]], ())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_training_run_in_pieces(cuda, dtype):
    """The benchmark's storage types at a size whose products reach the tensor cores: the loss agrees with the one
    through stored f32 logits, every leaf of the gradient within that program's own tolerance of its sequential form
    (tests/test_gpu_models.py), and the optimizer takes it; then distillation on the same host."""
    c = dict(V=515, D=256, H=2, G=2, FF=512, L=2)
    p = models.llama_params(c, seed=5, std=0.05)
    ids, y, classes, teacher = inputs(c, 9, 2, 128, top=8)
    y = np.abs(y)
    rz = {"default": dtype, "params": {k: dtype for k in p}, "storage": {"Llama.apply/%11": "f32", "loss/%5": "f32", "loss/%6": "f32", "distill/loss": "f32", "distill/mean": "f32"},
          "functions": {"adamw.step": "f32", "adamw.lr": "f32"}}
    logits = models.give(Host(cuda, dict(rz, order={"kind": "device"})).prepare("llama", **c), p)
    h = models.give(Host(cuda, dict(rz, order=PIECES)).prepare("llama", TEMP=2, **c), p).adamw(lr=1e-2, weight_decay=0.1, grad_clip=1.0)
    a, b = float(logits.call("loss", [ids, y], ())), float(h.call("loss", [ids, y], ()))
    # the same hidden states; f32 logits of truncated sums (4e-6) in one, of sums rounded in parts in the other
    assert b == pytest.approx(a, rel=1e-5)
    logits.call("loss_grad", [ids, y], p["tok"].shape)
    want = {k: logits.result(k, np.shape(v)) for k, v in p.items()}
    for t in (1, 2):
        h.call("loss_grad", [ids, y], p["tok"].shape)
        if t == 1:
            within(h, want, 0.06)
        h.adamw_step(t, 2)
    h.call("distill_grad", [ids, classes, teacher], p["tok"].shape)
    assert all(np.isfinite(h.result(k, np.shape(v))).all() for k, v in p.items())
    assert np.isfinite(float(h.call("distill", [ids, classes, teacher], ())))


@pytest.mark.gpu
def test_pieces_behind_merged_launches_and_integer_weights(cuda):
    """The benchmark's prefill realization with its loss in pieces; int8 heads are declined, and run as before."""
    c = dict(V=512, D=256, H=2, G=2, FF=512, L=2)
    p = models.llama_params(c)
    rng = np.random.default_rng(0)
    ids, y = (rng.integers(0, c["V"], size=(2, 128), dtype=np.int64) for _ in range(2))
    base = {"default": "bf16", "params": {k: "bf16" for k in p}, "storage": {"Llama.apply/%11": "f32", "loss/%5": "f32", "loss/%6": "f32", "RMSNorm.apply/%3": "f32", "RMSNorm.apply/%7": "f32"}}
    order = {"kind": "device", "attention": "online", "launches": "merged"}
    got = []
    for rz in (dict(base, order=order), dict(base, order=dict(order, loss="pieces"))):
        h = models.give(Host(cuda, rz).prepare("llama", **c), p)
        h.set_logging(True)
        got.append(float(h.call("loss", [ids, y], ())))
        assert ("head_xent[pieces]" in h.launch_log()) == ("loss" in rz["order"])
    assert got[1] == pytest.approx(got[0], rel=1e-5)
    quant = dict(base, order=dict(order, loss="pieces"), quant={"head": {"bits": 8, "over": 0}})
    h = models.give(Host(cuda, quant).prepare("llama", **c), p)
    h.set_logging(True)
    h.call("loss", [ids, y], ())
    assert "cross_entropy" in h.launch_log() and "head_xent[pieces]" not in h.launch_log()
