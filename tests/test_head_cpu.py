"""The head's losses on the CPU: the oracle's restatement against an independent 64-bit form and against differences,
and the refusals of a launch that is not one (no GPU: the check is compiled for the host)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import head_cases as hc
from presk_b200 import abi, head_loss_launch, head_loss_vjp_launch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def check():
    src, out = os.path.join(ROOT, "tests", "support", "head_shape.cpp"), os.path.join(ROOT, "tests", "support", "_head_shape.so")
    deps = [src, os.path.join(ROOT, "presk_b200", "csrc", "psk_head_shape.h"), os.path.join(ROOT, "include", "presk_cuda.h")]
    if not os.path.exists(out) or os.path.getmtime(out) < max(os.path.getmtime(d) for d in deps):
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", src, "-o", out], check=True)
    lib = C.CDLL(out)

    def f(l):
        err = C.create_string_buffer(512)
        rc = lib.head_shape_check(C.byref(l), err, C.c_size_t(512))
        return rc, err.value.decode()
    return f


class _Array:
    """A torch tensor as the oracle wrapper wants it (numpy has no bfloat16): only its address is read."""

    def __init__(self, t):
        self.t = t
        self.ctypes = self

    @property
    def data(self):
        return self.t.data_ptr()


def run_oracle(oracle, s):
    fwd, bwd = hc.launches(s)
    loss, lse = torch.full(s["outer"], 7.0), torch.full(s["outer"], 7.0)
    dx, dw = torch.full((*s["outer"], s["model"]), 7.0).to(s["x"].dtype), torch.full_like(s["w"], 7.0)
    oracle.run(fwd, [_Array(t) for t in hc.given(s) + [lse, loss]])
    oracle.run(bwd, [_Array(t) for t in hc.given(s) + [s["ct"], lse, dw, dx]])
    return {"loss": loss, "lse": lse, "dx": dx, "dw": dw}


CASES = [
    dict(outer=(3, 4), vocab=37, model=12, dtype=abi.F32),
    dict(outer=(5,), vocab=64, model=8, dtype=abi.BF16, vocab_major=True),
    dict(outer=(2, 3), vocab=19, model=7, dtype=abi.F16),
    dict(outer=(7,), vocab=40, model=9, dtype=abi.F32, top=6, tau=2.0),
    dict(outer=(2, 4), vocab=33, model=16, dtype=abi.BF16, top=5, tau=0.7, vocab_major=True, teacher=abi.BF16),
    dict(outer=(1,), vocab=1, model=1, dtype=abi.F32, ignored=0.0),
    dict(outer=(0, 3), vocab=5, model=4, dtype=abi.F32),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c['outer']}x{c['vocab']}x{c['model']}-{c.get('top', 0)}")
def test_the_oracle_agrees_with_the_formulas(oracle, case):
    s = hc.make(**case)
    got = run_oracle(oracle, s)
    want, _ = hc.plain(s)
    for k in want:
        # the oracle rounds once at the store, and its backward reads the f32 log-sum-exp
        tol = want[k].abs() * (hc.HALF[s["dtype"]] * 1.01 if k in ("dx", "dw") else 2.0**-23) + 2.0**-21
        assert ((got[k].double() - want[k]).abs() <= tol).all(), k


@pytest.mark.parametrize("top,tau", [(0, 1.0), (4, 1.7)])
def test_the_formulas_gradients_are_the_losses_differences(top, tau):
    s = hc.make((4,), 11, 6, abi.F32, top=top, tau=tau, ignored=0.25, seed=3)
    want, _ = hc.plain(s)
    step = 2.0**-10

    def total(t):
        return (hc.plain(t)[0]["loss"] * s["ct"].double()).sum()

    for name, key in (("x", "dx"), ("w", "dw")):
        flat = s[name].reshape(-1)
        for i in range(0, flat.numel(), 5):
            up, down = dict(s), dict(s)
            for t, sign in ((up, 1.0), (down, -1.0)):
                m = s[name].double().clone().reshape(-1)
                m[i] += sign * step
                t[name] = m.reshape(s[name].shape)  # 64-bit: `plain` reads any type
            diff = (total(up) - total(down)) / (2 * step)
            # central differences leave step² times a third derivative, here below 2 (|x|, |w| up to 4, ct up to 1/2)
            assert abs(diff - want[key].reshape(-1)[i]) <= 2 * step**2, (name, i)


def test_a_label_the_vocabulary_does_not_have(oracle):
    s = hc.make((3,), 8, 4, abi.F32, ignored=0.0)
    s["labels"][1] = 8
    with pytest.raises(RuntimeError, match="7001"):
        run_oracle(oracle, s)


def strided(l, which, axis, value):
    (l.out if which == "out" else l.inputs[which]).stride[axis] = value
    return l


def typed(l, which, dtype):
    (l.out if which == "out" else l.inputs[which]).dtype = dtype
    return l


def changed(l, **kw):
    for k, v in kw.items():
        if k == "tau":
            l.fparam[0] = v
        elif k.startswith("dim"):
            l.dims[int(k[3:])] = v
        else:
            setattr(l, k, v)
    return l


def fwd(**kw):
    return head_loss_launch((2, 3), 16, 8, abi.BF16, **kw)


def bwd(**kw):
    return head_loss_vjp_launch((2, 3), 16, 8, abi.BF16, **kw)


REFUSED = {
    "sequential order": (lambda: changed(fwd(), order=abi.ORDER_SEQUENTIAL), abi.E7005, "declared order"),
    "f64": (lambda: typed(typed(fwd(), 0, abi.F64), 1, abi.F64), abi.E7005, "one type"),
    "two types": (lambda: typed(fwd(), 1, abi.F16), abi.E7005, "one type"),
    "int8 head": (lambda: typed(fwd(), 1, abi.I8), abi.E7005, "one type"),
    "e8m15": (lambda: typed(typed(fwd(), 0, abi.E8M15), 1, abi.E8M15), abi.E7005, "one type"),
    "labels that are reals": (lambda: typed(fwd(), 2, abi.F32), abi.E7001, "indices"),
    "an empty vocabulary": (lambda: changed(fwd(), dim2=0), abi.E7001, "head of"),
    "an empty model": (lambda: changed(fwd(), dim3=0), abi.E7001, "head of"),
    "a negative length": (lambda: changed(fwd(), dim0=-1), abi.E7001, "negative length"),
    "too many rows": (lambda: changed(fwd(), dim0=1 << 40, dim1=1 << 40), abi.E7001, "more rows"),
    "a negative stride": (lambda: strided(fwd(), 0, 1, -8), abi.E7001, "negative stride"),
    "x over the classes": (lambda: strided(fwd(), 0, 2, 1), abi.E7001, "does not have"),
    "a head a row": (lambda: strided(fwd(), 1, 0, 128), abi.E7001, "does not have"),
    "a loss over one row": (lambda: strided(fwd(), "out", 1, 0), abi.E7005, "broadcast"),
    "dx of a broadcast x": (lambda: strided(bwd(), "out", 0, 0), abi.E7005, "broadcast"),
    "dw of a broadcast head": (lambda: strided(bwd(), 5, 2, 0), abi.E7005, "broadcast"),
    "dx in f32 of bf16": (lambda: typed(bwd(), "out", abi.F32), abi.E7005, "operands' type"),
    "dw in f32 of bf16": (lambda: typed(bwd(), 5, abi.F32), abi.E7005, "operands' type"),
    "lse in bf16": (lambda: typed(bwd(), 4, abi.BF16), abi.E7001, "log-sum-exp"),
    "no ct": (lambda: changed(bwd(), n_inputs=3), abi.E7001, "ct, lse"),
    "too many inputs": (lambda: changed(fwd(), n_inputs=5), abi.E7001, "labels"),
    "no temperature": (lambda: changed(fwd(top=4), tau=0.0), abi.E7001, "temperature"),
    "a temperature that is no number": (lambda: changed(fwd(top=4), tau=float("nan")), abi.E7001, "temperature"),
    "no entries": (lambda: changed(fwd(top=4), dim4=0), abi.E7001, "entries"),
    "too many entries": (lambda: changed(fwd(top=4), dim4=1025), abi.E7005, "1024"),
    "a teacher of indices": (lambda: typed(fwd(top=4), 3, abi.I64), abi.E7005, "teacher"),
    "an affine x": (lambda: changed_operand(fwd(), 0), abi.E7005, "one type"),
}


def changed_operand(l, i):
    l.inputs[i].affine = 1
    return l


@pytest.mark.parametrize("name", REFUSED)
def test_refusals(check, name):
    make, code, words = REFUSED[name]
    rc, msg = check(make())
    assert rc == code and words in msg, (rc, msg)


def test_what_is_not_refused(check):
    for l in (fwd(), fwd(lse=False), fwd(top=1024), bwd(), bwd(dw=False), bwd(top=3, temperature=4.0), head_loss_launch((0,), 1, 1, abi.F32), head_loss_vjp_launch(5, 3, 2, abi.F16, vocab_major=True),
              strided(bwd(), 3, 0, 0), strided(fwd(), 0, 0, 0)):  # a cotangent, or an x, of broadcast rows
        assert check(l) == (abi.OK, "")
