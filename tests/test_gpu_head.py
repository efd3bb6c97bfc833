"""The head's losses on the GPU (PSK_OP_HEAD_XENT, PSK_OP_HEAD_DISTILL and their gradients) against a plain form in 64
bits, with bounds of error derived in head_cases.py; layouts, types, rows without a target, refusals."""
import numpy as np
import pytest
import torch

import head_cases as hc
from presk_b200 import PreskError, abi

pytestmark = pytest.mark.gpu

GUARD = 64  # elements around every result that must stay as they are


class Fenced:
    """A result buffer with guard elements on both sides, every one the same number before the call."""

    def __init__(self, shape, dtype, offset=0):
        n = 1
        for d in shape:
            n *= d
        self.flat = torch.full((n + 2 * GUARD + offset,), 7.0, dtype=dtype, device="cuda")
        self.lo, self.n = GUARD + offset, n
        self.t = self.flat[self.lo:self.lo + n].reshape(shape)

    def check(self):
        assert (self.flat[:self.lo] == 7.0).all() and (self.flat[self.lo + self.n:] == 7.0).all(), "written outside the result"
        return self.t


def run(cuda, s, loss_dtype=abi.F32, step=True, offset=0, **more):
    fwd, bwd = hc.launches(s, loss_dtype=loss_dtype, **more)
    lse = Fenced(s["outer"], torch.float32)
    loss = Fenced(s["outer"], hc.TORCH[loss_dtype])
    out = {"loss": loss, "lse": lse}
    torch.cuda.synchronize()
    cuda.run(fwd, [t.data_ptr() for t in hc.given(s) + [lse.t, loss.t]])
    if step:
        out["dx"], out["dw"] = Fenced((*s["outer"], s["model"]), s["x"].dtype, offset), Fenced(s["w"].shape, s["w"].dtype, offset)
        cuda.run(bwd, [t.data_ptr() for t in hc.given(s) + [s["ct"], lse.t, out["dw"].t, out["dx"].t]])
    cuda.sync()
    return {k: f.check() for k, f in out.items()}


def compare(got, want, tol, keys=None):
    for k in keys or got:
        off = (got[k].double() - want[k]).abs()
        bad = ~(off <= tol[k])
        assert not bad.any(), (k, int(bad.sum()), float(off[bad].max() if bad.any() else 0), float((off / tol[k].clamp(min=1e-300)).nan_to_num(1e9).max()))


CASES = [
    # one of everything; a tile exactly; one more than a tile either way
    dict(outer=(1,), vocab=1, model=1, dtype=abi.BF16, ignored=0.0),
    dict(outer=(1,), vocab=2, model=3, dtype=abi.F32, ignored=0.0),
    dict(outer=(128,), vocab=256, model=64, dtype=abi.BF16),
    dict(outer=(129,), vocab=257, model=65, dtype=abi.BF16),
    dict(outer=(127,), vocab=255, model=63, dtype=abi.F16),
    dict(outer=(3, 5), vocab=1000, model=72, dtype=abi.BF16, vocab_major=True),
    dict(outer=(2, 3, 7), vocab=513, model=200, dtype=abi.F16, vocab_major=True),
    dict(outer=(64,), vocab=640, model=320, dtype=abi.BF16),  # the most rows whose g keeps its remainder
    dict(outer=(65,), vocab=640, model=320, dtype=abi.BF16),
    dict(outer=(300,), vocab=2000, model=1000, dtype=abi.BF16),
    dict(outer=(40,), vocab=300, model=2049, dtype=abi.F16),
    dict(outer=(33,), vocab=384, model=136, dtype=abi.F32),
    dict(outer=(200,), vocab=777, model=257, dtype=abi.F32, vocab_major=True),
    dict(outer=(700,), vocab=130, model=40, dtype=abi.BF16),
    # many rows (g in binary16, x and w copied into it), and enough tiles of dw for the products of 256 rows
    dict(outer=(257,), vocab=640, model=320, dtype=abi.BF16),
    dict(outer=(300,), vocab=10000, model=2048, dtype=abi.BF16),
    dict(outer=(301,), vocab=10001, model=2052, dtype=abi.BF16, vocab_major=True),
    dict(outer=(290,), vocab=9999, model=2051, dtype=abi.F16),
    dict(outer=(5000,), vocab=520, model=4100, dtype=abi.BF16, top=5, tau=2.0),
    # few rows under a large head: g's remainder as rows of dx's own tile
    dict(outer=(10,), vocab=17000, model=1000, dtype=abi.BF16),
    dict(outer=(64,), vocab=17001, model=1001, dtype=abi.F16, vocab_major=True, top=3),
    dict(outer=(65,), vocab=17000, model=1000, dtype=abi.BF16),
    # every row without a target; none
    dict(outer=(17,), vocab=100, model=32, dtype=abi.BF16, ignored=1.1),
    dict(outer=(17,), vocab=100, model=32, dtype=abi.F32, ignored=1.1, top=3),
    dict(outer=(31,), vocab=4096, model=256, dtype=abi.BF16, top=64, tau=2.0),
    dict(outer=(2, 70), vocab=1001, model=96, dtype=abi.BF16, top=7, tau=0.5, vocab_major=True, teacher=abi.BF16),
    dict(outer=(129,), vocab=515, model=130, dtype=abi.F16, top=33, tau=1.5, teacher=abi.F16),
    dict(outer=(50,), vocab=300, model=70, dtype=abi.F32, top=20, tau=3.0),
    dict(outer=(5,), vocab=1100, model=64, dtype=abi.BF16, top=1024),  # the longest list, most of a small vocabulary
    dict(outer=(9,), vocab=6, model=16, dtype=abi.BF16, top=10),  # more entries than classes: named again and again
    dict(outer=(1,), vocab=32000, model=128, dtype=abi.BF16, top=1, ignored=0.0),
]


def name(c):
    return "-".join([str(c["outer"]), str(c["vocab"]), str(c["model"]), abi.DTYPE_NAMES[c["dtype"]], f"top{c.get('top', 0)}", "vm" if c.get("vocab_major") else "mv"]).replace(" ", "")


@pytest.mark.parametrize("case", CASES, ids=name)
def test_loss_and_gradients(cuda, case):
    s = hc.make(device="cuda", **case)
    want, tol = hc.plain(s)
    compare(run(cuda, s), want, tol)


@pytest.mark.parametrize("dtype", [abi.BF16, abi.F16, abi.F32])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_strides_and_alignments(cuda, dtype, pad, offset):
    """Rows of x apart, results that begin at any element, a head whose rows do not begin on 16-byte boundaries."""
    s = hc.make((4, 33), 401, 88, dtype, pad=pad, device="cuda", top=5 if pad == 5 else 0, tau=1.3 if pad == 5 else 1.0)
    if offset:
        for k in ("x", "w"):
            flat = torch.zeros(s[k].numel() + offset, dtype=s[k].dtype, device="cuda")
            flat[offset:] = s[k].reshape(-1)
            s[k] = flat[offset:].reshape(s[k].shape)
    want, tol = hc.plain(s)
    compare(run(cuda, s, offset=offset), want, tol)


def test_an_axis_of_rows_that_x_does_not_walk_densely(cuda):
    """Next-token rows: all but the last position of every sequence (x read through [batch, seq + 1, model]), dx the same way."""
    s = hc.make((3, 20), 300, 64, abi.BF16, device="cuda")
    full = torch.full((3, 21, 64), float("nan"), dtype=torch.bfloat16, device="cuda")  # what lies between must not matter
    full[:, :20] = s["x"]
    s["x"] = full[:, :20]
    want, tol = hc.plain(s)
    _, bwd = hc.launches(s)
    got = run(cuda, s)
    compare(got, want, tol)
    for a, st in zip((0, 1, 3), (21 * 64, 64, 1)):
        bwd.out.stride[a] = st
    dfull = torch.full((3, 21, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    cuda.run(bwd, [t.data_ptr() for t in hc.given(s) + [s["ct"], got["lse"], got["dw"], dfull]])
    cuda.sync()
    assert (dfull[:, 20] == 7.0).all()
    assert torch.equal(dfull[:, :20], got["dx"])


def test_strange_strides(cuda):
    """x with its model axis apart, a head with both axes apart, a broadcast cotangent, a permuted dw."""
    s = hc.make((2, 9), 50, 24, abi.BF16, device="cuda")
    xt = torch.empty(24, 2, 9, dtype=torch.bfloat16, device="cuda")
    xt.copy_(s["x"].permute(2, 0, 1))
    big = torch.zeros(48, 100, dtype=torch.bfloat16, device="cuda")
    big[::2, ::2] = s["w"]
    s["ct"] = torch.full((2, 9), 0.125, device="cuda")
    want, tol = hc.plain(s)
    fwd, bwd = hc.launches(s)
    for l in (fwd, bwd):
        for a, st in zip((0, 1, 3), (9, 1, 18)):
            l.inputs[0].stride[a] = st
        for a, st in zip((2, 3), (2, 200)):
            l.inputs[1].stride[a] = st
    bwd.inputs[3].stride[0] = bwd.inputs[3].stride[1] = 0
    for a, st in zip((2, 3), (24, 1)):  # dw as [vocab, model] although w is not
        bwd.inputs[5].stride[a] = st
    loss, lse = Fenced((2, 9), torch.float32), Fenced((2, 9), torch.float32)
    dx, dw, one = Fenced((2, 9, 24), torch.bfloat16), Fenced((50, 24), torch.bfloat16), torch.full((1,), 0.125, device="cuda")
    torch.cuda.synchronize()
    cuda.run(fwd, [t.data_ptr() for t in (xt, big, s["labels"], lse.t, loss.t)])
    cuda.run(bwd, [t.data_ptr() for t in (xt, big, s["labels"], one, lse.t, dw.t, dx.t)])
    cuda.sync()
    compare({"loss": loss.check(), "lse": lse.check(), "dx": dx.check(), "dw": dw.check().t()}, want, tol)


@pytest.mark.parametrize("dtype", [abi.BF16, abi.F16, abi.F32])
@pytest.mark.parametrize("top", [0, 6])
def test_what_a_row_without_a_target_holds_reaches_nothing(cuda, dtype, top):
    s = hc.make((150,), 300, 64, dtype, device="cuda", top=top, ignored=0.3)
    want, tol = hc.plain(s)
    gone = (s["labels"] < 0) if not top else (s["ids"] < 0).all(-1)
    assert gone.any() and not gone.all()
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").to(s["x"].dtype)
    s["x"][gone] = bad[torch.arange(int(gone.sum()), device="cuda") % 3][:, None]
    s["ct"] = torch.where(gone, float("nan"), s["ct"])
    if top:
        s["teacher"][gone] = float("nan")
    got = run(cuda, s)
    compare(got, want, tol)
    for k in ("loss", "lse", "dx"):
        assert (got[k][gone] == 0).all(), k


def test_entries_of_minus_infinity_and_a_list_of_nothing_else(cuda):
    s = hc.make((40,), 200, 32, abi.BF16, device="cuda", top=8, ignored=0.0)
    s["teacher"][::2, ::2] = -float("inf")
    s["teacher"][3] = -float("inf")  # a row whose classes are there and whose logits are not
    s["ids"][5, :7] = -1
    s["teacher"][7] = -3.0e38  # the type's lowest values are values: a uniform list
    want, tol = hc.plain(s)
    got = run(cuda, s)
    compare(got, want, tol)
    assert got["loss"][3] == 0 and (got["dx"][3] == 0).all()


def test_a_nan_in_a_row_with_a_target_stays_in_it(cuda):
    s = hc.make((70,), 300, 64, abi.BF16, device="cuda", ignored=0.0)
    want, tol = hc.plain(s)
    s["x"][11, 3] = float("nan")
    got = run(cuda, s)
    rest = torch.arange(70, device="cuda") != 11
    assert torch.isnan(got["loss"][11]) and torch.isnan(got["dx"][11]).all() and torch.isnan(got["dw"]).all()
    for k in ("loss", "lse", "dx"):
        assert ((got[k][rest].double() - want[k][rest]).abs() <= tol[k][rest]).all(), k


def test_far_logits(cuda):
    """Logits of hundreds: the maximum is taken out before the exponential; a certain row has a gradient near zero."""
    for dtype in (abi.BF16, abi.F32):
        s = hc.make((140,), 500, 64, dtype, device="cuda", spread=60.0, ignored=0.0)
        want, tol = hc.plain(s)
        got = run(cuda, s)
        assert all(torch.isfinite(t.double()).all() for t in got.values())
        compare(got, want, tol)


def test_f16_gradients_below_the_types_least_number(cuda):
    """Under a mean over many rows most of g lies below binary16's subnormals; dx and dw do not."""
    s = hc.make((256,), 8192, 32, abi.F16, device="cuda", spread=0.5, ignored=0.0)
    s["ct"] = s["ct"] * 256 / 16384
    want, tol = hc.plain(s)
    got = run(cuda, s)
    compare(got, want, tol)
    s["ct"] = s["ct"] * 16384 * 64
    want, tol = hc.plain(s)
    compare(run(cuda, s), want, tol)
    far = got["dw"].double() - want["dw"] / (16384 * 64)
    assert float(far.norm() / (want["dw"] / (16384 * 64)).norm()) < 0.05  # outputs below 2^-14 have few bits left themselves


@pytest.mark.parametrize("loss_dtype", [abi.F32, abi.BF16, abi.F16])
def test_the_loss_in_other_types(cuda, loss_dtype):
    s = hc.make((77,), 300, 64, abi.BF16, device="cuda")
    want, tol = hc.plain(s)
    tol["loss"] = tol["loss"] + want["loss"].abs() * hc.HALF[loss_dtype] * 1.01
    compare(run(cuda, s, loss_dtype=loss_dtype, step=False), want, tol)


def test_cotangents_in_other_types(cuda):
    s = hc.make((77,), 300, 64, abi.BF16, device="cuda")
    s["ct"] = s["ct"].to(torch.bfloat16).float()
    got = run(cuda, s)
    _, bwd = hc.launches(s, ct_dtype=abi.BF16)
    ct, dx, dw = s["ct"].to(torch.bfloat16), torch.empty_like(got["dx"]), torch.empty_like(got["dw"])
    torch.cuda.synchronize()
    cuda.run(bwd, [t.data_ptr() for t in hc.given(s) + [ct, got["lse"], dw, dx]])
    cuda.sync()
    assert torch.equal(dx, got["dx"]) and torch.equal(dw, got["dw"])


def test_without_the_second_results(cuda):
    s = hc.make((77,), 300, 64, abi.BF16, device="cuda")
    got = run(cuda, s)
    fwd, bwd = hc.launches(s)
    fwd.n_inputs, bwd.n_inputs = 3, 5
    loss, dx = Fenced((77,), torch.float32), Fenced((77, 64), torch.bfloat16)
    torch.cuda.synchronize()
    cuda.run(fwd, [t.data_ptr() for t in hc.given(s) + [loss.t]])
    cuda.run(bwd, [t.data_ptr() for t in hc.given(s) + [s["ct"], got["lse"], dx.t]])
    cuda.sync()
    assert torch.equal(loss.check(), got["loss"]) and torch.equal(dx.check(), got["dx"])


@pytest.mark.parametrize("dtype,rows,vocab,model,vocab_major", [(abi.BF16, 16500, 26000, 64, False), (abi.F32, 8200, 25000, 32, True), (abi.F16, 20001, 20500, 40, True)])
def test_several_pieces_of_the_vocabulary(cuda, dtype, rows, vocab, model, vocab_major):
    """More than 768 MB of g: the vocabulary goes in pieces, and dx is summed over them."""
    s = hc.make((rows,), vocab, model, dtype, device="cuda", vocab_major=vocab_major)
    want, tol = hc.plain(s)
    compare(run(cuda, s), want, tol)


def test_no_rows(cuda):
    s = hc.make((0, 4), 100, 32, abi.BF16, device="cuda")
    got = run(cuda, s)
    assert (got["dw"] == 0).all() and got["loss"].numel() == 0


def test_the_same_call_gives_the_same_bits(cuda):
    s = hc.make((200,), 3000, 512, abi.BF16, device="cuda", top=16, tau=2.0)
    a = run(cuda, s)
    other = hc.make((150,), 2500, 256, abi.BF16, device="cuda", seed=9)
    run(cuda, other)
    b = run(cuda, s)
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_precision_of_long_sums(cuda):
    """A model of 8192 with products of one sign: sums by truncation alone would be 3e-5 too small."""
    s = hc.make((64,), 300, 8192, abi.BF16, device="cuda", ignored=0.0)
    s["x"], s["w"] = s["x"].abs(), s["w"].abs()
    want, tol = hc.plain(s)
    got = run(cuda, s)
    compare(got, want, tol)
    assert float((got["lse"].double() - want["lse"]).norm() / want["lse"].norm()) < 2e-6


@pytest.mark.parametrize("rows", [1, 3, 60, 200, 400])
@pytest.mark.parametrize("top", [0, 4])
def test_gradients_are_as_exact_as_their_type(cuda, rows, top):
    """bf16 results: g's own rounding must not show beside the result's (its half step is 2^-8, 2^-9.2 on average)."""
    s = hc.make((rows,), 3000, 256, abi.BF16, device="cuda", top=top, ignored=0.0, seed=rows)
    want, _ = hc.plain(s)
    got = run(cuda, s)
    for k in ("dx", "dw"):
        off = float((got[k].double() - want[k]).norm() / want[k].norm())
        best = float((want[k].to(torch.bfloat16).double() - want[k]).norm() / want[k].norm())
        assert off <= 1.1 * best, (k, off, best)


def test_rows_of_other_magnitudes(cuda):
    """f32 operands are split about a row's own greatest element: a row of 1e18 takes nothing from its neighbours' logits."""
    s = hc.make((140,), 300, 64, abi.F32, device="cuda", ignored=0.0)
    want, tol = hc.plain(s)
    s["x"][7] *= 1e18
    s["x"][9] *= 1e-18
    got = run(cuda, s, step=False)
    rest = torch.tensor([i not in (7, 9) for i in range(140)], device="cuda")
    for k in ("loss", "lse"):
        assert ((got[k][rest].double() - want[k][rest]).abs() <= tol[k][rest]).all(), k
    w9, t9 = hc.plain(s)
    assert (got["lse"][9].double() - w9["lse"][9]).abs() <= t9["lse"][9]
    big = w9["lse"][7]
    assert (got["lse"][7].double() - big).abs() <= t9["lse"][7]


@pytest.mark.parametrize("dtype,rows", [(abi.F32, 20), (abi.F32, 300), (abi.BF16, 300), (abi.BF16, 20)])
def test_rows_of_other_weights(cuda, dtype, rows):
    """A power of two, up to 2^30, taken from a row's cotangent is taken from its gradient: what g loses at the bottom of
    binary16 is 2^-39 of the greatest ct's, of a row at 2^-30 of that 2^(30/2 - 39), and one power for the halving."""
    s = hc.make((rows,), 700, 96, dtype, device="cuda", ignored=0.0)
    got = run(cuda, s)
    less = torch.exp2(-(torch.arange(rows, device="cuda") % 30).float())
    s["ct"] = s["ct"] * less
    want, tol = hc.plain(s)
    again = run(cuda, s)
    compare(again, want, tol)
    w = s["w"].double().abs().sum(1)[None]  # two runs: each g to 2^-23 of the row's ct, each result to its half step
    close = 2 * 2.0**-23 * s["ct"].double()[:, None] * w + 2.02 * hc.HALF[dtype] * want["dx"].abs()
    off = (again["dx"].double() - got["dx"].double() * less[:, None].double()).abs()
    rounds = 2.0**-20 * s["ct"].double()[:, None] * w  # g itself, and the sums (as in head_cases), the same in both but for the scale
    assert (off <= close + rounds).all(), float((off / (close + rounds)).max())


@pytest.mark.parametrize("dtype,rows", [(abi.F32, 20), (abi.F32, 300), (abi.BF16, 300), (abi.BF16, 20), (abi.F16, 300)])
@pytest.mark.parametrize("top", [0, 3])
def test_rows_of_no_weight(cuda, dtype, rows, top):
    """A cotangent of zero: the row's gradient is zero, and nothing of it is in dw."""
    s = hc.make((rows,), 700, 96, dtype, device="cuda", ignored=0.1, top=top)
    s["ct"][::3] = 0.0
    s["x"][::3] *= 100.0
    want, tol = hc.plain(s)
    got = run(cuda, s)
    compare(got, want, tol)
    assert (got["dx"][::3] == 0).all()
    s["ct"].zero_()
    got = run(cuda, s)
    assert (got["dx"] == 0).all() and (got["dw"] == 0).all()


def test_gradients_summed_over_a_large_vocabulary(cuda):
    """dx of 131072 products of one sign (x = 0: g is 2^-17, exactly, beside the labels' class, whose weight is 0). Added by
    truncation alone it is 4.5e-4 too small on average. Its rounding to binary16, at most 2^-11, is zero on average over
    2048 outputs to 2^-11 / sqrt(3 x 2048) = 6e-6, four times which and 1.4e-5 of truncation are below 5e-5."""
    rows, vocab, model = 2304, 131072, 2048  # tiles for one wave: the sums are not split
    gen = torch.Generator(device="cuda").manual_seed(3)
    s = hc.make((rows,), 64, model, abi.F16, device="cuda", ignored=0.0)
    s["x"].zero_()
    s["vocab"], s["w"] = vocab, torch.rand(model, vocab, generator=gen, device="cuda").add_(1.0).to(torch.float16)
    s["labels"].zero_()
    s["w"][:, 0] = 0
    s["ct"] = torch.ones_like(s["ct"])
    got = run(cuda, s)
    want = s["w"].double().sum(1) / vocab
    off = (got["dx"].double() / want - 1)
    assert float(off.abs().max()) <= 2 ** -11 + 1.4e-5 + 2 ** -20
    assert abs(float(off[0].mean())) < 5e-5, float(off[0].mean())


def normals(rows, cols, scale, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for lo in range(0, rows, 1 << 16):
        t[lo:lo + (1 << 16)] = torch.randn(min(1 << 16, rows - lo), cols, generator=g, device="cuda") * scale
    return t


@pytest.mark.parametrize("rows,vocab", [(4, 600_001), (600_001, 200)])
def test_offsets_beyond_32_bits(cuda, rows, vocab):
    """x or the head of 2.5e9 elements (4.9 GB, its gradient as much): the last of them against 64 bits."""
    model = 4096
    s = dict(outer=(rows,), vocab=vocab, model=model, dtype=abi.BF16, top=0, tau=1.0, vocab_major=True)
    s["x"], s["w"] = normals(rows, model, 1.0, 1), normals(vocab, model, 2.0 / model**0.5, 2)
    s["labels"] = vocab - 1 - torch.arange(rows, device="cuda") % min(vocab, 150)
    s["ct"] = torch.full((rows,), 1.0 / rows, device="cuda")
    loss, lse = Fenced((rows,), torch.float32), Fenced((rows,), torch.float32)
    dx, dw = Fenced((rows, model), torch.bfloat16), Fenced((vocab, model), torch.bfloat16)
    fwd, bwd = hc.launches(s)
    torch.cuda.synchronize()
    cuda.run(fwd, [t.data_ptr() for t in hc.given(s) + [lse.t, loss.t]])
    cuda.run(bwd, [t.data_ptr() for t in hc.given(s) + [s["ct"], lse.t, dw.t, dx.t]])
    cuda.sync()
    last = slice(max(0, rows - 100), rows)
    x, step = s["x"][last].double(), 20_000
    z = torch.cat([x @ s["w"][lo:lo + step].double().t() for lo in range(0, vocab, step)], 1)
    want = torch.logsumexp(z, 1)
    # a logit of 4096 products: accumulators of 512 (32 additions by truncation of sums below 100), eight of them added
    assert ((lse.check()[last].double() - want).abs() <= 100 * 40 * 2.0**-23).all()
    assert ((loss.check()[last].double() - (want - z.gather(1, s["labels"][last][:, None])[:, 0])).abs() <= 2 * 100 * 40 * 2.0**-23).all()
    g = torch.exp(z - want[:, None])
    g[torch.arange(len(x), device="cuda"), s["labels"][last]] -= 1.0
    g /= rows
    want_dx = sum(g[:, lo:lo + step] @ s["w"][lo:lo + step].double() for lo in range(0, vocab, step))
    off = (dx.check()[last].double() - want_dx).norm() / want_dx.norm()
    assert float(off) <= 2.0**-8  # the result's half step at most everywhere
    end = slice(max(0, vocab - 100), vocab)
    want_dw = torch.zeros(100, model, dtype=torch.float64, device="cuda")
    for lo in range(0, rows, step):  # every row's part of the last classes
        xb, y = s["x"][lo:lo + step].double(), s["labels"][lo:lo + step]
        if rows > 100:
            zb = xb @ s["w"].double().t()
            gb = torch.exp(zb - torch.logsumexp(zb, 1, keepdim=True))[:, end]
        else:
            gb = torch.exp(z - want[:, None])[:, end]
        hit = y - end.start
        gb[torch.arange(len(y), device="cuda")[hit >= 0], hit[hit >= 0]] -= 1.0
        want_dw += gb.t() @ xb / rows
    off = (dw.check()[end].double() - want_dw).norm() / want_dw.norm()
    assert float(off) <= 2.0**-8


def test_a_class_the_vocabulary_does_not_have(cuda):
    for top in (0, 4):
        s = hc.make((10,), 100, 32, abi.BF16, device="cuda", top=top, ignored=0.0)
        (s["ids"] if top else s["labels"]).reshape(-1)[2] = 100
        with pytest.raises(PreskError, match="index outside its bound"):
            run(cuda, s)
        cuda.sync()  # reported once


def test_refusals_leave_the_executor_usable(cuda):
    s = hc.make((10,), 100, 32, abi.BF16, device="cuda")
    fwd, _ = hc.launches(s)
    fwd.order = abi.ORDER_SEQUENTIAL
    loss = torch.zeros(10, device="cuda")
    with pytest.raises(PreskError, match="declared order"):
        cuda.run(fwd, [t.data_ptr() for t in hc.given(s) + [loss, loss]])
    want, tol = hc.plain(s)
    compare(run(cuda, s), want, tol)


def test_not_while_the_stream_is_captured(cuda):
    s = hc.make((10,), 100, 32, abi.BF16, device="cuda")
    fwd, _ = hc.launches(s)
    loss, lse = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    tab = [t.data_ptr() for t in hc.given(s) + [lse, loss]]
    torch.cuda.synchronize()
    stream = torch.cuda.ExternalStream(cuda.stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            with pytest.raises(PreskError, match="captured"):
                cuda.run(fwd, tab)
        finally:
            graph.capture_end()
    cuda.run(fwd, tab)
    cuda.sync()


def test_the_workspace_goes_back_to_the_pool(cuda):
    s = hc.make((100,), 1000, 64, abi.BF16, device="cuda")
    run(cuda, s)
    live, _ = cuda.memory()
    for _ in range(3):
        run(cuda, s)
    assert cuda.memory()[0] == live
