"""The gradient of gated_attention's position bias where its sums cancel: every pair's score gradient enters it unrounded, behind a gate too."""
import pytest
import torch

import gated_attention_exact as X

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
# A pair's score gradient holds float32 sums of dk and dv products (off by about sqrt(n) 2^-24 of their root mean square, 34 * 2^-24 for 1152 of them) and a sum over up to
# 2^22 pairs of a bucket adds sqrt(2^22) 2^-24 of the root of the sum of squares at most: together below 2^-12.5.  A softmax's far entry is what little the near ones
# leave of a row's sum, sqrt(n / 2 D) times smaller than its terms: up to 8 times that at these sizes, 1e-3 with the other entries of the norm beside it.
TABLE = {"relu2": 2.0 ** -12.5, "softmax": 1e-3}


def _all_close(t, kind, causal, **kw):
    got, want = X.run(t, kind, causal, **kw), X.attention(t, kind, causal, **kw)
    far = {n: X.off(got[n], want[n]) for n in want}
    u = X.U[t["q"].dtype]
    for n, e in far.items():
        assert e <= (TABLE[kind] if n == "dtable" else 1.05 * u), (n, far)


@pytest.mark.parametrize("seed", [0, 1, 2, 3])
@pytest.mark.parametrize("D", [16, 128, 1100])
@pytest.mark.parametrize("kind", ["relu2", "softmax"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_bias_gradient_behind_a_gate(dtype, kind, D, seed):
    """dout * gate rounded to the type is off the same way for all keys of a row: it would not average out over a bucket's pairs"""
    _all_close(X.inputs(seed, dtype, 4, 1024, 1024, 1, 1, 128, 1024, True, 32, D, std={"dout": 0.02}), kind, True)


@pytest.mark.parametrize("kind", ["relu2", "softmax"])
@pytest.mark.parametrize("shape", [(2, 1000, 1000, 4, 2, 64, 64), (3, 515, 515, 2, 2, 96, 104), (2, 600, 600, 2, 1, 72, 200), (1, 40, 700, 2, 2, 128, 264), (64, 17, 17, 1, 1, 128, 512), (40, 30, 60, 1, 1, 64, 128)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_bias_gradient_behind_a_gate_at_every_width(dtype, shape, kind):
    _all_close(X.inputs(5, dtype, *shape, True, 32, 64, std={"dout": 0.02}), kind, False)


def test_bias_gradient_of_long_sequences_and_a_16_bit_table():
    for kind in ("relu2", "softmax"):
        t = X.inputs(7, BF16, 1, 4096, 4096, 1, 1, 128, 1024, True, 32, 128, BF16, std={"dout": 0.02})
        got, want = X.run(t, kind, True), X.attention(t, kind, True)
        assert X.off(got["dtable"], want["dtable"]) <= X.U[BF16] * 0.75 + TABLE[kind]          # (one rounding, evenly spread over the 32 entries' mantissas)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("L, dv", [(1000, 64), (700, 320), (24, 64), (2000, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_softmax_bias_gradient_where_one_entry_holds_nearly_all_keys(dtype, L, dv, gate):
    """A softmax row's score gradients sum to zero, so the entry that all distances but one share is what that one leaves, sqrt(L) times smaller than its terms.  The map
    reaches beyond the sequence: no distance lies behind its ends.  (What remains: float32 sums of L terms against one of them.)"""
    D = L + 3
    t = X.inputs(11, dtype, 2, L, L, 2, 1, 64, dv, gate, 4, D, std={"dout": 0.1})
    t["buckets"] = torch.ones(2 * D + 1, dtype=torch.int32, device="cuda")
    t["buckets"][D] = 0
    t["table"] = t["table"][:2].contiguous()
    for causal in (False, True):
        got, want = X.run(t, "softmax", causal)["dtable"], X.attention(t, "softmax", causal)["dtable"]
        assert X.off(got, want) <= TABLE["softmax"], (causal, got.tolist(), want.tolist())
