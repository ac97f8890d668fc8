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


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_distances_and_positions_at_their_ends(dtype):
    """one query over many keys, keys all ahead of or all behind the queries, one distance for all, the widest map, a single tile of keys under many queries"""
    for Lq, Lk, D, start in ((1, 3000, 2048, 2999), (1, 3000, 1, 0), (200, 20, 40, -150), (150, 900, 0, 0), (70, 1100, 2048, -4000), (70, 1100, 300, 5000), (130, 500, 33, 200)):
        t = X.inputs(13, dtype, 2, Lq, Lk, 2, 1, 64, 72, True, 8, max(D, 1), std={"dout": 0.1})
        if D == 0:
            t["buckets"] = t["buckets"][1:2].contiguous()
        for kind in ("relu2", "softmax"):
            for causal in (False, True):
                got, want = X.run(t, kind, causal, start=start), X.attention(t, kind, causal, start=start)
                # a bias gradient that is zero by nature (one entry for all of a softmax's distances) keeps float32 sums of its terms: W |dW| adds to |dO| sqrt(dv) a row
                size = float((t["dout"].double() * t["gate"].double()).square().sum(-1).sqrt().square().sum().sqrt()) * 72 ** 0.5
                for n in want:
                    if n == "dtable":
                        lim = 1e-3 * float(want[n].norm()) + 2.0 ** -18 * size
                    else:
                        lim = LIMIT[dtype] * float(want[n].norm()) + (2.0 ** -25 if dtype == F16 else 2.0 ** -24 * 2.0 ** -16) * want[n].numel() ** 0.5 + (2.0 ** -18 * size if Lq == 1 or kind == "softmax" else 0.0)
                    assert bool(got[n].isfinite().all()) and float((got[n].double() - want[n]).norm()) <= lim, (Lq, Lk, D, start, kind, causal, n, X.off(got[n], want[n]))


def test_softmax_training_captured_and_replayed():
    """forward and backward with a gate and a table, both 16-bit types in one graph, replayed with new inputs between eager calls"""
    from tracklab_amd import attention as A
    sets = [X.inputs(21, dt, 3, 150, 150, 2, 1, 64, 72, True, 16, 20) for dt in (F16, BF16)]
    lens = torch.tensor([150, 7, 90], dtype=torch.int32, device="cuda")
    leaves = [[t[n].detach().requires_grad_() for n in ("q", "k", "v", "gate", "table")] for t in sets]

    def step():
        res = []
        for t, x in zip(sets, leaves):
            out = A.gated_attention(*x[:4], kind="softmax", bias=x[4], buckets=t["buckets"], causal=True, lens=lens)
            res += [out.detach(), *torch.autograd.grad(out, x, t["dout"])]
        return res

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(4):
        g = torch.Generator().manual_seed(turn)
        with torch.no_grad():
            for x in (*leaves[0], *leaves[1], *(t["dout"] for t in sets)):
                x.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
            lens.copy_(torch.randint(0, 151, (3,), generator=g, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
        torch.cuda.synchronize()
