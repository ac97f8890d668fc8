"""gated_attention where the bias is far larger than the scores: a softmax's weights, forward and backward, depend on differences alone."""
import pytest
import torch

import gated_attention_exact as X

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _case(dtype, Lq, Lk, values, seed=1, table_dtype=F32):
    """q = 0: the scores are the bias alone.  Distances up to 1 see values[0], up to 40 values[1], all others values[2]"""
    t = X.inputs(seed, dtype, 2, Lq, Lk, 2, 1, 64, 72, True, 3 * 2, 64, table_dtype, std={"dout": 0.1})
    D = 64
    away = torch.arange(-D, D + 1).abs()
    t["buckets"] = torch.where(away <= 1, 0, torch.where(away <= 40, 1, 2)).to(torch.int32).cuda()
    t["table"] = torch.tensor(values, dtype=torch.float32).to(table_dtype)[:, None].repeat(1, 2).cuda()
    t["q"].zero_()
    return t


def _close(t, start=0, causal=False):
    got, want = X.run(t, "softmax", causal, start=start), X.attention(t, "softmax", causal, start=start)
    u = X.U[t["q"].dtype]
    for n in want:
        # 16-bit: as everywhere.  float32: weights of 2^x are off by a few units of 2^-24 for each of x's few bits before the point, sums of up to 2000 terms by 2^-18 of their size
        lim = (1.05 * u + 2.0 ** -16) * float(want[n].norm()) + (2.0 ** -25 * want[n].numel() ** 0.5 if t["q"].dtype == F16 else 0.0) + 2.0 ** -18 * (n == "dtable") * float(want["dq"].numel()) ** 0.5
        assert bool(got[n].isfinite().all()) and float((got[n].double() - want[n]).norm()) <= lim, (n, X.off(got[n], want[n]))


@pytest.mark.parametrize("value", [-1e4, -1e7, -1e9, -3e38, 1e9])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_rows_whose_keys_all_carry_a_large_bias(dtype, value):
    """every key of a row at the same large value weighs the same, in the backward pass too (queries that stand apart from all keys, and rows that see other keys as well)"""
    for Lq, Lk in ((50, 300), (3, 1500), (30, 30)):
        _close(_case(dtype, Lq, Lk, [0.5, 0.25, value]), start=-500)
        _close(_case(dtype, Lq, Lk, [0.5, 0.25, value]))
        _close(_case(dtype, Lq, Lk, [value, value, value]))
    if dtype != F32:
        low = float(torch.finfo(dtype).min)
        _close(_case(dtype, 50, 300, [0.5, low, low], table_dtype=dtype), start=-500)
        _close(_case(dtype, 50, 300, [0.5, low, low], table_dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_order_of_the_largest_finite_biases(dtype):
    """biases next to float32's largest numbers keep their order and stay finite: the larger one takes the row, equal ones share it"""
    for values in ([-2.5e38, -2.3e38, -2.3e38], [-2.3e38, -2.5e38, -3.3e38], [-2.3e38] * 3, [2.3e38, 2.5e38, 3.3e38], [3.3e38, 2.5e38, 1e38], [-1.1e38, -0.9e38, -3.4e38], [2.2e38] * 3):
        t = _case(dtype, 50, 300, values)
        _close(t)
        _close(t, start=-500)
        _close(_case(dtype, 3, 1500, values), start=700)
