"""Norm of the error of every output and gradient of gated_attention, at lengths where the element bounds of gated_attention_reference.py have grown past the values."""
import pytest
import torch

import gated_attention_exact as X

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# 16-bit: the roundings that gated_attention_exact.py counts, and 5 % for the float32 sums between them.  float32: a sum of n <= 1100 terms is off by about sqrt(n) 2^-24 of their
# root mean square; a gradient passes at most five such sums in a row (S, the row's statistics, dW, delta, its own), 5 * 33 * 2^-24 < 2^-16.  The bias gradient: TABLE of its own test.
LIMIT = {F32: 2.0 ** -16, F16: 1.05 * X.U[F16], BF16: 1.05 * X.U[BF16]}


@pytest.mark.parametrize("gate, table", [(False, False), (True, False), (False, True), (True, True)], ids=["plain", "gate", "table", "both"])
@pytest.mark.parametrize("kind", ["relu2", "softmax"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_error_norms(dtype, kind, gate, table):
    for shape, causal, lens, start in (((2, 1000, 1000, 4, 2, 64, 64), True, None, 0), ((2, 515, 771, 2, 1, 128, 128), False, [771, 300], 0), ((1, 900, 1100, 1, 1, 128, 520), True, None, 200),
                                       ((3, 257, 1030, 2, 2, 80, 40), True, [1030, 513, 700], 300)):
        t = X.inputs(9, dtype, *shape, gate, 32 if table else 0, 100, std={"dout": 0.05})
        n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
        got, want = X.run(t, kind, causal, n, start), X.attention(t, kind, causal, n, start)
        far = {k: X.off(got[k], want[k]) for k in want}
        for k, e in far.items():
            assert e <= (1e-3 if k == "dtable" else LIMIT[dtype]), (shape, k, far)
