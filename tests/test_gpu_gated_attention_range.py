"""float16 training of gated_attention over its range: what stands between the gate and the gradients may lie far below and above float16's numbers."""
import pytest
import torch

import gated_attention_exact as X

pytestmark = pytest.mark.gpu
F16 = torch.float16
HALF = 2.0 ** -25                              # half of float16's smallest step: what the rounding of a result below 2^-14 is off by


def _close(got, want, names):
    """the norm of the error over the entries within the type; an entry beyond its largest number (65520 and more round to infinity) is the infinity of its sign.
    An entry sum_j a_j b_jc whose factors a_j (a row's dO, weights or score gradients) were rounded is off by u / sqrt(3) of sqrt(sum_j a_j^2 b_jc^2), which is the root mean
    square of its row whatever the entry itself came to: the small entries of a row whose large ones are infinite keep an error of the row's size.  So the bound is
    u of the norm of all entries, those beyond the type among them."""
    u = X.U[F16]
    for n in names:
        a, b = got[n].double(), want[n]
        fits, beyond = b.abs() < 65504 * (1 - 4 * u), b.abs() > 65520 * (1 + 4 * u)
        assert torch.equal(a[beyond], b[beyond].sign() * float("inf")) and bool(a[fits].isfinite().all()), n
        lim = 1.05 * u * float(b.norm()) + HALF * b.numel() ** 0.5
        a, b = a[fits], b[fits]
        assert float((a - b).norm()) <= lim, (n, X.off(a, b), lim / float(b.norm()))


@pytest.mark.parametrize("dv", [64, 320])
@pytest.mark.parametrize("kind", ["relu2", "softmax"])
def test_small_gates_and_gradients(kind, dv):
    """dout near 2^-13 behind gates near 2^-8: their products lie below float16's normal numbers, the gradients do not"""
    t = X.inputs(1, F16, 2, 600, 600, 2, 1, 64, dv, True, 16, 64, std={"dout": 2.0 ** -13, "gate": 2.0 ** -8, "v": 2.0 ** 7 if kind == "softmax" else 4.0, "k": 32.0, "q": 2.0 ** -3})
    for causal in (False, True):
        got, want = X.run(t, kind, causal), X.attention(t, kind, causal)
        _close(got, want, ("out", "dq", "dk", "dv", "dgate"))
        assert X.off(got["dtable"], want["dtable"]) <= 1e-3
        assert float(want["dq"].abs().mean()) > 2.0 ** -14


@pytest.mark.parametrize("kind", ["relu2", "softmax"])
def test_products_beyond_the_largest_number(kind):
    """dout * gate above 65504, weights and values small enough that the gradients are within the type, all but a few entries of dv"""
    t = X.inputs(2, F16, 2, 400, 400, 2, 2, 64, 72, True, 16, 64, std={"dout": 2.0 ** 9, "gate": 2.0 ** 9, "v": 2.0 ** -9, "k": 2.0 ** -3, "q": 2.0 ** -3})
    scale = 0.125
    if kind == "relu2":
        t["table"] *= 2.0 ** -3
    else:
        t["gate"][:, 4:] *= 2.0 ** -9           # (a few such rows: a key's gradient is their sum)
    got, want = X.run(t, kind, False, scale=scale), X.attention(t, kind, False, scale=scale)
    assert float((t["dout"].double() * t["gate"].double()).abs().max()) > 65504
    _close(got, want, ("out", "dq", "dk", "dv", "dgate"))
    assert X.off(got["dtable"], want["dtable"]) <= 1e-3


@pytest.mark.parametrize("kind", ["relu2", "softmax"])
def test_rows_of_different_size(kind):
    """half of the rows 2^-12 behind the others, in turn and after them: keys that only small rows see get their gradients in full"""
    for later in (False, True):
        t = X.inputs(3, F16, 1, 640, 640, 1, 1, 64, 64, True, 0, std={"dout": 0.5, "v": 4.0, "k": 2.0})
        if later:
            t["gate"][:, 320:] *= 2.0 ** -12
        else:
            t["gate"][:, ::2] *= 2.0 ** -12
        got, want = X.run(t, kind, True), X.attention(t, kind, True)
        _close(got, want, ("out", "dq", "dk", "dv", "dgate"))
        if later:
            _close({n: got[n][:, 320:] for n in got}, {n: want[n][:, 320:] for n in want}, ("dq", "dk", "dv"))


def test_rows_of_zeros_and_a_row_that_is_not_a_number():
    t = X.inputs(4, F16, 1, 70, 90, 1, 1, 64, 64, True, 0)
    t["gate"][:, 10:20] = 0
    for kind in ("relu2", "softmax"):
        got, want = X.run(t, kind), X.attention(t, kind)
        _close(got, want, ("out", "dq", "dk", "dv", "dgate"))
        assert not got["dq"][:, 10:20].any()
        bad = {**t, "dout": t["dout"].clone()}
        bad["dout"][0, 33, 0, 5] = float("inf")
        dq = X.run(bad, kind)["dq"]
        assert not dq[0, 33].isfinite().all() and torch.equal(dq[0, :33], got["dq"][0, :33]) and torch.equal(dq[0, 34:], got["dq"][0, 34:])


def test_values_before_the_gate_beyond_the_largest_number():
    """relu^2 weights of hundreds: o above 65504 behind gates that bring it back; the gate's gradient is dout * o"""
    for B, Lq, Lk, dv in ((2, 300, 300, 64), (2, 17, 40, 512), (1, 4, 2000, 72)):
        t = X.inputs(6, F16, B, Lq, Lk, 1, 1, 64, dv, True, 0, std={"q": 8.0, "k": 8.0, "gate": 2.0 ** -9, "dout": 2.0 ** -11, "v": 4.0})
        got, want = X.run(t, "relu2"), X.attention(t, "relu2")
        assert float((want["dgate"].abs() / t["dout"].double().abs().clamp(min=1e-30)).max()) > 65504
        _close(got, want, ("out", "dgate", "dv"))


@pytest.mark.parametrize("first", [320, 333])
@pytest.mark.parametrize("kind", ["relu2", "softmax"])
def test_keys_that_only_small_rows_see(kind, first):
    """causal: from row ``first`` on dout * gate lies 2^-24 behind the rows before it, so the keys from there on have nothing but small rows; their gradients are as
    exact as the others', whatever larger rows are worked on beside them"""
    t = X.inputs(7, F16, 1, 640, 640, 1, 1, 64, 64, True, 0, std={"dout": 2.0 ** 9, "gate": 2.0 ** 8, "v": 2.0 ** -2, "q": 0.5, "k": 0.5})
    t["gate"][:, first:] *= 2.0 ** -12
    t["dout"][:, first:] *= 2.0 ** -12
    got, want = X.run(t, kind, True), X.attention(t, kind, True)
    _close({n: got[n][:, first:] for n in got}, {n: want[n][:, first:] for n in want}, ("dq", "dk", "dv", "dgate"))
    _close(got, want, ("dq", "dk", "dv", "dgate"))
