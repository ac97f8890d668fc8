"""gated_attention and norm_gate_residual on the GPU against their 64-bit definition (tests/gated_attention_reference.py, which derives the bounds):
types, head layouts, lengths from one row up, odd widths, strides, masks that leave rows empty, gradients, splits, streams, graphs."""
import math

import pytest
import torch

import gated_attention_reference as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _A():
    from tracklab_amd import attention
    return attention


def _rand(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype).cuda()


def _inputs(seed, dtype, B, Lq, Lk, H, Hk, dk, dv, gate=True, buckets=8, D=6, table_dtype=None):
    g = torch.Generator().manual_seed(seed)
    t = dict(q=_rand(g, B, Lq, H, dk, dtype=dtype), k=_rand(g, B, Lk, Hk, dk, dtype=dtype), v=_rand(g, B, Lk, Hk, dv, dtype=dtype),
             gate=_rand(g, B, Lq, H, dv, dtype=dtype) if gate else None,
             table=_rand(g, buckets, H, dtype=table_dtype or dtype, std=0.5) if buckets else None,
             buckets=torch.randint(0, buckets, (2 * D + 1,), generator=g, dtype=torch.int32).cuda() if buckets else None,
             dout=_rand(g, B, Lq, H, dv, dtype=dtype, std=0.1))
    return t


def _within(got, val, bnd, what=""):
    got = got.detach().double().cpu()
    assert got.shape == val.shape, (what, got.shape, val.shape)
    over = (got - val).abs() - bnd
    assert bool((over <= 0).all()), f"{what}: off by up to {float((got - val).abs().max()):.3e}, {float(over.max()):.3e} beyond its bound, at {int((over > 0).sum())} of {over.numel()}"


def _run(t, kind, causal=False, lens=None, start=0, scale=None, train=True):
    A = _A()
    leaves = {n: t[n].detach().requires_grad_(train) for n in ("q", "k", "v", "gate", "table") if t[n] is not None}
    out = A.gated_attention(leaves["q"], leaves["k"], leaves["v"], leaves.get("gate"), kind=kind, scale=scale, bias=leaves.get("table"), buckets=t["buckets"], causal=causal,
                            lens=lens, q_start=start)
    got = {"out": out}
    if train:
        got.update({"d" + n: gr for n, gr in zip(leaves, torch.autograd.grad(out, list(leaves.values()), t["dout"]))})
    return got


def _check(t, kind, causal=False, lens=None, start=0, scale=None, train=True):
    got = _run(t, kind, causal, lens, start, scale, train)
    sc = t["q"].shape[-1] ** -0.5 if scale is None else scale
    val, bnd = R.attention(t["q"], t["k"], t["v"], t["gate"], t["table"], t["buckets"], lens, start, kind, causal, sc, t["dout"] if train else None)
    assert set(got) == set(val)
    for n in val:
        _within(got[n], val[n], bnd[n], n)
    return got


SHAPES = [  # B, Lq, Lk, H, Hk, dk, dv
    (1, 1, 1, 1, 1, 8, 8),
    (2, 2, 2, 2, 1, 16, 24),
    (3, 17, 17, 1, 1, 128, 512),
    (2, 16, 33, 4, 2, 64, 64),
    (1, 33, 31, 3, 3, 40, 104),
    (2, 65, 64, 2, 2, 64, 136),
    (1, 130, 129, 4, 1, 128, 128),
    (1, 257, 200, 2, 1, 72, 264),
    (1, 40, 300, 1, 1, 128, 520),
    (2, 5, 70, 6, 1, 32, 16),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["relu2", "softmax"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_attention_and_its_gradients(dtype, kind, shape):
    B, Lq, Lk = shape[:3]
    t = _inputs(1, dtype, *shape)
    _check(t, kind)
    # causal, lengths among them none and more than there is room, positions before and after the keys
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32)
    lens[0] = [0, Lk + 5, Lk, -3][sum(shape) % 4]
    start = torch.randint(-Lq, Lk, (B,), generator=g, dtype=torch.int32)
    _check(t, kind, causal=True, lens=lens.cuda(), start=start.cuda())
    _check(t, kind, causal=True, start=Lk - Lq)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("gate, buckets, table", [(False, 0, None), (True, 0, None), (False, 5, None), (True, 5, F32)])
def test_without_gate_or_bias_and_a_float32_table(dtype, gate, buckets, table):
    for kind in ("relu2", "softmax"):
        _check(_inputs(5, dtype, 2, 37, 50, 4, 2, 64, 72, gate, buckets, 9, table), kind, causal=kind == "softmax")


@pytest.mark.parametrize("D, buckets", [(0, 1), (1, 3), (20, 41), (300, 32), (2048, 7)])
def test_distances_of_the_bias(D, buckets):
    """one entry, fewer distances than a tile, more than the sequence; buckets beyond the table are clipped"""
    t = _inputs(6, BF16, 1, 70, 150, 2, 2, 64, 64, True, buckets, D)
    t["buckets"][0], t["buckets"][-1] = -4, buckets + 9
    _check(t, "softmax")
    _check(t, "relu2", causal=True, start=80)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dv, causal", [(64, False), (64, True), (320, False)])
def test_shared_distances_of_a_softmax_take_up_no_rounding(dtype, dv, causal):
    """A row's score gradients sum to zero.  With values between two neighbours of the type o is rounded the same way in every row, by up to half a step: a
    delta from that o would leave eps / 4 of sum W |dW| in the entries beyond +-D.  Bound: dW and S are float32 sums of dv and dk products (relative error
    below (dv + dk) 2^-24 < 2^-15), a weight's exponent of a few units takes S's error a few times, and sums over 700 keys add 2^-17: 2^-13 of sum W (|dW| +
    |delta|), which is below eps / 4 for both types' eps / 4 (2^-12 and 2^-9)."""
    L, D = 700, 16
    t = _inputs(35, dtype, 2, L, L, 1, 1, 64, dv, False, 2 * D + 1, D, F32)
    t["buckets"] = torch.arange(2 * D + 1, dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(36)
    t["v"] = (1 + torch.finfo(dtype).eps * (torch.rand(t["v"].shape, generator=g) < 0.75)).to(dtype).cuda()
    t["dout"] = torch.ones_like(t["dout"])
    got = _run(t, "softmax", causal)["dtable"].double().cpu()[:, 0]
    q, k, v, tab = (t[n].double().cpu() for n in ("q", "k", "v", "table"))
    away = torch.arange(L) - torch.arange(L)[:, None]
    want, size = torch.zeros(2 * D + 1, dtype=torch.float64), torch.zeros(2 * D + 1, dtype=torch.float64)
    for b in range(2):
        s = q[b, :, 0] @ k[b, :, 0].T / 8 + tab[:, 0][away.clamp(-D, D) + D]
        w = torch.softmax(torch.where(away > 0, -math.inf, s) if causal else s, -1)
        dw = v[b, :, 0].sum(-1).expand(L, L)
        delta = (w * dw).sum(-1, keepdim=True)
        want.index_add_(0, (away.clamp(-D, D) + D).reshape(-1), (w * (dw - delta)).reshape(-1))
        size.index_add_(0, (away.clamp(-D, D) + D).reshape(-1), (w * (dw + delta)).reshape(-1))
    for e in (0, 2 * D):
        assert float((got - want)[e].abs()) <= float(size[e]) * 2.0 ** -13, (e, float(got[e]), float(want[e]), float(size[e]))


@pytest.mark.parametrize("dk, dv", [(20, 13), (5, 3), (100, 33), (127, 257)])
def test_widths_that_are_no_multiple_of_16_bytes(dk, dv):
    for dtype in (F32, F16):
        _check(_inputs(7, dtype, 2, 19, 23, 2, 1, dk, dv), "softmax")


def test_what_stands_beside_float32_rows_of_half_a_fragment():
    """12 and 20 columns of float32, which 32-byte reads would pass: the columns next to them hold NaN"""
    for dk, dv, Lq, Lk in ((12, 20, 19, 23), (20, 12, 3, 40), (4, 4, 70, 1)):
        t = _inputs(30, F32, 2, Lq, Lk, 2, 1, dk, dv)
        for n, d in (("q", dk), ("k", dk), ("v", dv), ("gate", dv)):
            wide = torch.full((*t[n].shape[:3], d + 4), float("nan"), device="cuda")
            wide[..., :d] = t[n]
            t[n] = wide[..., :d]
        for kind in ("relu2", "softmax"):
            _check(t, kind)


def test_the_c_entry_ignores_the_row_strides_of_one_row():
    import ctypes as C
    A = _A()
    L = A._bound()
    t = _inputs(31, BF16, 2, 1, 1, 2, 1, 64, 72, True, 0)
    want = A.gated_attention(t["q"], t["k"], t["v"], t["gate"])
    a = A.GauArgs()
    a.dtype, a.kind, a.batch, a.len_q, a.len_k, a.heads, a.kv_heads, a.dim_k, a.dim_v, a.scale = 2, 0, 2, 1, 1, 2, 1, 64, 72, 0.125
    a.q_stride[:], a.k_stride[:], a.v_stride[:], a.gate_stride[:] = (128, 0, 64), (64, 0, 64), (72, 0, 72), (144, 0, 72)
    a.q, a.k, a.v, a.gate = (t[n].data_ptr() for n in ("q", "k", "v", "gate"))
    out = torch.zeros_like(want)
    assert L.tlk_gau_attention_fwd(C.byref(a), out.data_ptr(), None, None, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    assert want.any() and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
def test_the_widest_bias_with_the_widest_values(dtype):
    """2048 distances a side beside 256 and 300 columns of dv: float32 tiles leave less LDS for the waves' sums"""
    for dv in (256, 300):
        _check(_inputs(32, dtype, 1, 70, 150, 2, 2, 128, dv, True, 7, 2048), "softmax")


@pytest.mark.parametrize("kind", ["relu2", "softmax"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_few_tiles_of_rows_over_many_keys(dtype, kind):
    """more rows than one tile, too few to fill the card: the keys are split; lengths that end inside a split, on its border and at zero"""
    lens = torch.tensor([1500, 512, 0, 257], dtype=torch.int32).cuda()
    for Lq, H, Hk, dv in ((40, 2, 1, 64), (130, 1, 1, 72)):
        t = _inputs(33, dtype, 4, Lq, 1500, H, Hk, 64, dv, True, 16, 64)
        _check(t, kind, causal=True, lens=lens, start=lens - Lq, train=False)
        _check(t, kind, lens=lens)
    _check(_inputs(34, dtype, 1, 150, 1300, 1, 1, 128, 264, True, 16, 64), kind, causal=True, start=1150)


@pytest.mark.parametrize("kind", ["relu2", "softmax"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_few_rows_over_many_keys(dtype, kind):
    """a cache that is split over workgroups, heads sharing keys answered together; lengths that end inside a split, on its border, and at zero"""
    lens = torch.tensor([3001, 2048, 0, 1, 257, 4096], dtype=torch.int32).cuda()
    for Lq, H, Hk, dv in ((1, 8, 2, 128), (3, 7, 1, 64), (1, 1, 1, 520), (17, 2, 1, 64)):
        t = _inputs(8, dtype, 6, Lq, 4096, H, Hk, 64, dv, True, 16, 64)
        _check(t, kind, causal=True, lens=lens, start=lens - Lq, train=False)
        _check(t, kind, lens=lens, train=False)
    t = _inputs(9, dtype, 1, 2, 3000, 2, 1, 128, 64, True, 16, 64)
    _check(t, kind, causal=True, start=2998)                    # trained through the splits: the joined log-sum-exp feeds the backward pass


def test_keys_behind_the_length_are_not_read():
    A = _A()
    for dtype, kind in ((F16, "relu2"), (BF16, "softmax"), (F32, "softmax")):
        t = _inputs(10, dtype, 3, 40, 77, 2, 2, 64, 64)
        lens = torch.tensor([0, 33, 76], dtype=torch.int32).cuda()
        clean = _check(t, kind, lens=lens)
        for b, n in enumerate(lens.tolist()):
            t["k"][b, n:] = math.nan
            t["v"][b, n:] = math.inf
        dirty = _run(t, kind, lens=lens)
        for n in clean:
            assert torch.equal(clean[n], dirty[n]), n
        assert not clean["out"][0].any() and not clean["dv"][1, 33:].any() and not clean["dk"][0].any()
        # the lengths may be changed between calls without anything else (the first sequence holds nothing but NaN by now)
        lens.fill_(5)
        assert torch.equal(_run(t, kind, lens=lens, train=False)["out"][1:], _run({**t, "k": t["k"][:, :5], "v": t["v"][:, :5]}, kind, train=False)["out"][1:])


def test_bias_entries_that_forbid():
    """-inf and the lowest finite value as bias: forbidden distances; rows of nothing else give zeros (-inf) or the mean of the keys (finite)"""
    for dtype in (F32, F16, BF16):
        t = _inputs(11, dtype, 1, 30, 30, 1, 1, 64, 64, False, 3, 4)
        t["buckets"][:] = torch.tensor([0, 0, 0, 1, 1, 1, 2, 2, 2], dtype=torch.int32)
        t["table"][0] = -math.inf
        t["table"][2] = torch.finfo(dtype).min
        out = _run(t, "softmax", train=False)["out"]
        q, k, v = (t[n][0, :, 0].double().cpu() for n in ("q", "k", "v"))
        s = q @ k.t() / 8
        away = torch.arange(30)[None] - torch.arange(30)[:, None]
        want = torch.softmax(s.masked_fill(away.abs() > 1, -math.inf), -1) @ v       # distances 2 and more lie in the lowest-value bucket, -2 and less in -inf's
        # bounds as in the reference for these weights: two roundings of the type, float32 scores
        bound = 3 * R.U[dtype] * v.abs().max() + 1e-4
        ok = torch.ones(30, dtype=torch.bool)
        s2 = (s + t["table"][1].double().cpu()).masked_fill(away.abs() > 1, -math.inf)
        want = torch.softmax(s2, -1) @ v
        assert float((out[0, :, 0].double().cpu() - want)[ok].abs().max()) <= bound
        t["table"].fill_(-math.inf)
        assert not _run(t, "softmax", train=False)["out"].any()
        got = _run(t, "softmax")
        assert not got["dq"].any() and not got["dv"].any()
        t["table"].fill_(torch.finfo(dtype).min)
        if dtype != F16:                                        # the scores vanish next to it: every key weighs the same
            mean = v.mean(0).expand(30, 64)
            assert float((_run(t, "softmax", train=False)["out"][0, :, 0].double().cpu() - mean).abs().max()) <= bound
        t["table"].fill_(-1e4)
        assert not _run(t, "relu2", train=False)["out"].any()


def test_not_a_number_is_not_swallowed():
    for kind in ("relu2", "softmax"):
        for dtype in (F32, F16, BF16):
            t = _inputs(12, dtype, 1, 20, 20, 1, 1, 64, 64)
            t["q"][0, 3, 0, 5] = math.nan
            out = _run(t, kind, train=False)["out"]
            assert out[0, 3].isnan().all() and not out[0, 4:].isnan().any() and not out[0, :3].isnan().any()
            t["q"][0, 3, 0, 5] = 0
            t["v"][0, 7, 0, 9] = math.nan
            assert _run(t, kind, train=False)["out"][0, :, 0, 9].isnan().all()


def test_float16_weights_beyond_its_range():
    """relu^2 weights above 65504 and below float16's smallest normal number: a power of two per row carries them"""
    t = _inputs(13, F16, 1, 50, 90, 1, 1, 64, 64, True, 0)
    t["v"] *= 2.0 ** -9
    t["dout"] *= 2.0 ** -6
    t["k"][:, 60:] *= 24.0                                      # the row's largest scores come late: sums so far are rescaled
    got = _check(t, "relu2", scale=4.0)
    assert got["out"].isfinite().all()
    s = (t["q"][0, :, 0].float() @ t["k"][0, :, 0].float().t() * 4).relu()
    assert s.max() > 300
    t = _inputs(14, F16, 1, 50, 90, 1, 1, 64, 64, True, 0)
    t["v"] *= 2.0 ** 13
    _check(t, "relu2", scale=2.0 ** -12, train=False)
    t["v"] *= 2.0 ** -10
    t["dout"] *= 2.0 ** 4
    _check(t, "relu2", scale=2.0 ** -8)


def test_strides_views_and_alignment():
    """slices of one projection, a (B, H, L, d) layout, rows that start at odd addresses, broadcast gates, no head dimension: the same values"""
    A = _A()
    for dtype in (F32, F16, BF16):
        t = _inputs(15, dtype, 2, 21, 21, 2, 2, 64, 64, True, 8, 6)
        want = _run(t, "softmax", train=False)["out"]
        call = lambda q, k, v, gate: A.gated_attention(q, k, v, gate, kind="softmax", bias=t["table"], buckets=t["buckets"])      # noqa: E731
        wide = torch.cat([t["gate"], t["v"], t["q"], t["k"]], -1)
        u, v, q, k = wide.split(64, -1)
        assert torch.equal(call(q, k, v, u), want)
        bh = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (t["q"], t["k"], t["v"], t["gate"])]
        assert torch.equal(call(*bh), want)
        odd = [torch.empty(x.numel() + 3, dtype=dtype, device="cuda")[3:].view(x.shape).copy_(x) for x in (t["q"], t["k"], t["v"], t["gate"])]
        assert odd[0].data_ptr() % 16 and torch.equal(call(*odd), want)
        last = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (t["q"], t["k"], t["v"], t["gate"])]
        assert last[0].stride(-1) != 1 and torch.equal(call(*last), want)
        one = [x[:, :, :1] for x in (t["q"], t["k"], t["v"], t["gate"])]
        flat = A.gated_attention(*(x.squeeze(2) for x in one), kind="softmax", bias=t["table"][:, :1], buckets=t["buckets"])
        assert torch.equal(flat, call_one(A, one, t).squeeze(2)) and flat.dim() == 3
    # gradients of broadcast inputs: the gate of one token for all, keys shared by expanding
    t = _inputs(16, F32, 2, 9, 9, 4, 4, 32, 32)
    gate, k = t["gate"][:, :1].clone().requires_grad_(), t["k"][:, :, :1].clone().requires_grad_()
    out = A.gated_attention(t["q"], k.expand(-1, -1, 4, -1), t["v"], gate.expand(-1, 9, -1, -1), kind="softmax")
    dg, dk = torch.autograd.grad(out, [gate, k], t["dout"])
    full = _run({**t, "k": k.detach().expand(-1, -1, 4, -1), "gate": gate.detach().expand(-1, 9, -1, -1), "table": None, "buckets": None}, "softmax")
    assert torch.allclose(dg, full["dgate"].sum(1, keepdim=True), rtol=1e-5, atol=1e-6) and torch.allclose(dk, full["dk"].sum(2, keepdim=True), rtol=1e-5, atol=1e-6)
    # an expanded gradient (a sum's) and a gradient of one input alone
    q = t["q"].clone().requires_grad_()
    A.gated_attention(q, t["k"], t["v"], kind="softmax").sum().backward()
    ones = _run({**t, "gate": None, "table": None, "buckets": None, "dout": torch.ones_like(t["dout"])}, "softmax")
    assert torch.equal(q.grad, ones["dq"])


def call_one(A, one, t):
    return A.gated_attention(*one, kind="softmax", bias=t["table"][:, :1].contiguous(), buckets=t["buckets"])


def test_empty_calls():
    A = _A()
    for kind in ("relu2", "softmax"):
        t = _inputs(17, F16, 2, 5, 7, 2, 1, 64, 64)
        no_q = _run({**t, "q": t["q"][:, :0], "gate": t["gate"][:, :0], "dout": t["dout"][:, :0]}, kind)
        assert no_q["out"].shape == (2, 0, 2, 64) and not no_q["dk"].any() and not no_q["dv"].any() and not no_q["dtable"].any()
        no_k = _run({**t, "k": t["k"][:, :0], "v": t["v"][:, :0]}, kind)
        assert not no_k["out"].any() and not no_k["dq"].any() and not no_k["dgate"].any() and not no_k["dtable"].any() and no_k["dk"].shape == (2, 0, 1, 64)
        no_b = _run({n: x[:0] if n not in ("table", "buckets") else x for n, x in t.items()}, kind)
        assert no_b["out"].shape == (0, 5, 2, 64) and not no_b["dtable"].any()


def test_offsets_beyond_32_bits():
    """keys whose rows lie more than 2^31 elements behind the first: only those are non-zero, the answer is theirs alone"""
    A = _A()
    n = (1 << 24) + 333
    k = torch.zeros(1, n, 1, 128, dtype=F16, device="cuda")
    v = torch.zeros(1, n, 1, 128, dtype=F16, device="cuda")
    g = torch.Generator().manual_seed(18)
    tail = 40
    k[:, -tail:], v[:, -tail:] = _rand(g, 1, tail, 1, 128, dtype=F16), _rand(g, 1, tail, 1, 128, dtype=F16)
    q = _rand(g, 1, 1, 1, 128, dtype=F16)
    out = A.gated_attention(q, k, v, kind="relu2", causal=True, q_start=n - 1)
    val, bnd = R.attention(q, k[:, -tail:], v[:, -tail:], None, None, None, None, tail - 1, "relu2", True, 128 ** -0.5)
    _within(out, val["out"], bnd["out"])
    del k, v
    torch.cuda.empty_cache()


def test_equal_bits_on_every_run():
    for dtype in (F16, BF16, F32):
        t = _inputs(19, dtype, 2, 150, 150, 4, 2, 64, 136, True, 16, 32)
        for kind in ("relu2", "softmax"):
            a, b = _run(t, kind, causal=True), _run(t, kind, causal=True)
            assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("kind", ["relu2", "softmax"])
def test_gradients_against_differences(kind):
    """float32 gradients along a random direction against central differences of the 64-bit definition"""
    t = _inputs(20, F32, 2, 23, 29, 2, 1, 24, 40, True, 6, 5)
    got = _run(t, kind, causal=True, start=6)
    g = torch.Generator().manual_seed(21)
    names = ("q", "k", "v", "gate", "table")
    base = {n: t[n].double().cpu() for n in names}
    R.U[torch.float64] = 2.0 ** -53

    def f(x):
        val, _ = R.attention(x["q"], x["k"], x["v"], x["gate"], x["table"], t["buckets"], None, 6, kind, True, 24 ** -0.5)
        return float((val["out"] * t["dout"].double().cpu()).sum())

    for n in names:
        step = torch.randn(base[n].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        diff = (f({**base, n: base[n] + h * step}) - f({**base, n: base[n] - h * step})) / (2 * h)
        along = float((got["d" + n].double().cpu() * step).sum())
        size = float((got["d" + n].double().cpu() * step).abs().sum())
        # float32 gradients: a few hundred summed products each, 2^-24 of their magnitudes; the difference quotient: h^2 and 2^-53 / h, both below 1e-8 here
        assert abs(diff - along) <= 1e-4 * size + 1e-7, n


def test_another_stream_and_overlapping_calls():
    """calls on two streams at once use workspaces of their own and give what they give alone"""
    A = _A()
    t1, t2 = _inputs(22, BF16, 4, 1, 5000, 8, 2, 128, 128), _inputs(23, BF16, 4, 1, 5000, 8, 2, 128, 128)
    want = [_run(t, "softmax", train=False)["out"] for t in (t1, t2)]
    w1, w2 = _run(t1, "softmax"), _run(t2, "softmax")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, (s, t) in enumerate(zip(streams, (t1, t2))):
            with torch.cuda.stream(s):
                got[i].append(_run(t, "softmax", train=False)["out"])
                got[i].append(_run(t, "softmax"))
    torch.cuda.synchronize()
    for i, w in enumerate((w1, w2)):
        assert all(torch.equal(o, want[i]) for o in got[i][::2])
        assert all(torch.equal(o[n], w[n]) for o in got[i][1::2] for n in w)


def test_captured_and_replayed():
    """forward (split keys) and backward captured into graphs, two of them alive at once, replayed with new inputs between eager calls"""
    A = _A()
    graphs = []
    for seed, dtype in ((24, F16), (25, BF16)):
        t = _inputs(seed, dtype, 3, 20, 20, 2, 1, 64, 264, True, 8, 6)
        cache = _inputs(seed + 2, dtype, 3, 1, 3000, 4, 2, 64, 64, False, 8, 6)
        lens = torch.tensor([3000, 1500, 7], dtype=torch.int32).cuda()
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "gate", "table")]

        def both(t=t, cache=cache, lens=lens, leaves=leaves):
            out = A.gated_attention(*leaves[:4], kind="relu2", bias=leaves[4], buckets=t["buckets"])
            grads = torch.autograd.grad(out, leaves, t["dout"])
            with torch.no_grad():
                one = A.gated_attention(cache["q"], cache["k"], cache["v"], kind="softmax", bias=cache["table"], buckets=cache["buckets"], causal=True, lens=lens, q_start=lens - 1)
            return [out.detach(), one, *grads]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        graphs.append((graph, outs, both, t, cache, lens, leaves))
    for turn in range(4):
        for graph, outs, both, t, cache, lens, leaves in graphs:
            g = torch.Generator().manual_seed(100 + turn)
            with torch.no_grad():
                for x in (*leaves, t["dout"], cache["q"], cache["k"]):
                    x.copy_(torch.randn(x.shape, generator=g).mul_(0.3).to(x.dtype))
                lens.copy_(torch.randint(1, 3001, (3,), generator=g, dtype=torch.int32))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs, both, *_ in graphs:
            kept = [o.clone() for o in outs]
            assert all(torch.equal(a, b) for a, b in zip(kept, both()))
            torch.cuda.synchronize()


def test_refusals_on_the_gpu():
    from tracklab_amd._lib import TlkError
    A = _A()
    t = _inputs(26, F16, 2, 5, 7, 4, 2, 64, 64)
    q, k, v, gate, table, buckets = (t[n] for n in ("q", "k", "v", "gate", "table", "buckets"))
    lens = torch.tensor([1, 2], dtype=torch.int32).cuda()
    for args, kw in (((q, k, v.float()), {}), ((q, k[:1], v), {}), ((q[:, :, :3], k, v), {}), ((q, k, v, gate[:, :4]), {}), ((q, k, v), dict(bias=table)),
                     ((q, k, v), dict(bias=table[:, :3], buckets=buckets)), ((q, k, v), dict(bias=table, buckets=buckets[:-1])), ((q, k, v), dict(bias=table, buckets=buckets.long())),
                     ((q, k, v), dict(lens=lens.long())), ((q, k, v), dict(lens=lens.cpu())), ((q, k, v), dict(lens=lens[:1])), ((q, k, v), dict(q_start=lens.float())),
                     ((torch.cat([q, q, q], -1), torch.cat([k, k, k], -1), v), {}), ((q, k.cpu(), v), {})):
        with pytest.raises(TlkError):
            A.gated_attention(*args, **kw)
    h = q[:, :, 0]
    w = torch.ones(64, dtype=F16).cuda()
    for args, kw in (((h, h.float()), {}), ((h, h[:1]), {}), ((h,), dict(res_scale=w)), ((h,), dict(norm="rms")), ((h,), dict(weight=w)), ((h,), dict(norm="rms", weight=w[:3])),
                     ((h,), dict(norm="rms", weight=w, bias=w)), ((h,), dict(norm="scale", weight=w)), ((h,), dict(gate=h[:, :3])), ((h,), dict(gate=w[:5])), ((h,), dict(norm="batch", weight=w)),
                     ((torch.zeros(2, 8200, dtype=F16).cuda(),), {}), ((h,), dict(next_norm="layer")), ((h,), dict(norm="rms", weight=w, eps=-1.0))):
        with pytest.raises(TlkError):
            A.norm_gate_residual(*args, **kw)


# ------------------------------------------------------------------------------------------------------------------------------ joint

JOINTS = [  # shape, norm, gate, residual, res_scale, next
    ((2, 17, 256), "scale", "vector", True, True, "scale"),
    ((3, 1, 8), "rms", "full", True, False, "rms"),
    ((1, 1, 1), "layer", None, False, False, "scale"),
    ((4, 33, 264), "layer", "batch", True, True, "layer"),
    ((5, 7, 1000), "rms", "full", True, True, None),
    ((2, 3, 5, 100), None, "batch", True, True, "rms"),
    ((70, 513), "layer", "vector", True, True, "rms"),
    ((6, 2048), "scale", "full", False, False, None),
    ((9, 3333), "rms", None, True, True, "scale"),
    ((130, 4096), "rms", "full", True, True, "rms"),
    ((3, 8192), "layer", "vector", True, True, "layer"),
    ((2, 8191), "rms", "full", True, True, "layer"),
    ((300, 64), None, "full", False, False, None),
]


def _joint_inputs(seed, dtype, shape, norm, gate, residual, res_scale, after):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]

    def weights(kind):
        if kind is None:
            return None, None
        w = _rand(g, 1 if kind == "scale" else d, dtype=dtype, std=0.2, mean=1.0)
        return w, _rand(g, d, dtype=dtype, std=0.2) if kind == "layer" else None

    gates = {None: None, "vector": (d,), "full": shape, "batch": shape[:1] + (1,) * (len(shape) - 2) + (d,)}[gate]
    t = dict(h=_rand(g, *shape, dtype=dtype), x=_rand(g, *shape, dtype=dtype) if residual else None, gate=_rand(g, *gates, dtype=dtype, mean=0.3) if gates else None,
             rs=_rand(g, d, dtype=dtype, std=0.2, mean=1.0) if res_scale else None)
    t["w"], t["b"] = weights(norm)
    t["w2"], t["b2"] = weights(after)
    t["dy"], t["dz"] = _rand(g, *shape, dtype=dtype), _rand(g, *shape, dtype=dtype)
    return t


def _joint_run(t, norm, after, dtype=None, use=("y", "z")):
    A = _A()
    names = [n for n in ("h", "x", "gate", "rs", "w", "b", "w2", "b2") if t[n] is not None]
    leaf = {n: (t[n].detach().requires_grad_() if n in names else None) for n in ("h", "x", "gate", "rs", "w", "b", "w2", "b2")}
    got = A.norm_gate_residual(leaf["h"], leaf["x"], norm=norm, weight=leaf["w"], bias=leaf["b"], gate=leaf["gate"], res_scale=leaf["rs"], next_norm=after, next_weight=leaf["w2"],
                               next_bias=leaf["b2"])
    out = {"y": got[0], "z": got[1]} if after else {"y": got}
    pick = [n for n in out if n in use]
    grads = torch.autograd.grad([out[n] for n in pick], [leaf[n] for n in names], [t["d" + n] for n in pick], allow_unused=True)
    out.update({"d" + n: gr for n, gr in zip(names, grads)})
    return out


def _joint_reference(t, norm, after, use=("y", "z")):
    names = [n for n in ("h", "x", "gate", "rs", "w", "b", "w2", "b2") if t[n] is not None]
    leaf = {n: (t[n].detach().double().requires_grad_() if n in names else None) for n in ("h", "x", "gate", "rs", "w", "b", "w2", "b2")}
    y, z = R.joint(leaf["h"], leaf["x"], leaf["gate"], leaf["rs"], norm, leaf["w"], leaf["b"], after, leaf["w2"], leaf["b2"])
    out = {"y": y, "z": z} if after else {"y": y}
    pick = [n for n in out if n in use]
    grads = torch.autograd.grad([out[n] for n in pick], [leaf[n] for n in names], [t["d" + n].double() for n in pick], allow_unused=True)
    out.update({"d" + n: gr for n, gr in zip(names, grads)})
    return out


def _cancelled(t, norm, after, use):
    """What rounding leaves where a norm's gradient cancels: it is a sum of up to three terms no larger than |t| / norm (t: the gradient at the norm's result times its weight), each
    the product of a few rounded factors and of a mean of d products (64 * 2^-24, as below), so 256 * 2^-24 of the largest term; on its way to a parameter it is multiplied
    by that parameter's factor and summed over the rows."""
    big = lambda x: 1.0 if x is None else float(x.detach().double().abs().max())      # noqa: E731
    d, rows = t["h"].shape[-1], t["h"].numel() // t["h"].shape[-1]

    def inverse(kind, v):
        if kind is None:
            return 1.0
        v = v.detach().double()
        v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        q = v.pow(2).mean(-1).sqrt()
        return float((1 / (q.clamp(min=1e-5) if kind == "scale" else (q * q + 1e-5).sqrt())).max())

    f = {n: (None if x is None else x.double()) for n, x in t.items()}
    y, _ = R.joint(f["h"], f["x"], f["gate"], f["rs"], norm, f["w"], f["b"], None, None, None)
    n1, _ = R.joint(f["h"], None, None, None, norm, f["w"], f["b"], None, None, None)
    inv1, inv2 = inverse(norm, t["h"]), inverse(after, y)
    step = 256 * 2.0 ** -24
    up = (big(t["dy"]) if "y" in use else 0.0) + (big(t["dz"]) * big(t["w2"]) * inv2 if after and "z" in use else 0.0)
    e, gate = step * up, big(t["gate"])
    shared = 1 if t["gate"] is None or t["gate"].shape == t["h"].shape else rows
    hat = d ** 0.5                                               # no normalised value is larger
    return {"dx": e * big(t["rs"]), "drs": rows * e * big(t["x"]), "dgate": shared * e * big(n1), "db": rows * e * gate, "dw": rows * e * gate * hat * (d if norm == "scale" else 1),
            "dh": e * gate * big(t["w"]) * inv1 * 2}


def _joint_close(got, want, dtype, rows, what="", floor=None):
    """Outputs are rounded once: half a step u of the value.  Everything before is float32: each value passes at most two norms, whose sums of d terms are
    off by (log-depth sums of at most 32 in a row) 64 * 2^-24 of their magnitudes, and a norm's gradient subtracts terms as large as the row's largest (``floor``: what that leaves
    where they cancel); a column sum adds at most rows / 256 + 256 values in a row, its terms cancelling: relative to the largest entry of the tensor."""
    u = R.U[dtype]
    for n in want:
        if want[n] is None:
            assert got[n] is None or not got[n].any(), n
            continue
        a, b = got[n].detach().double().cpu(), want[n].detach().double().cpu()
        big = float(b.abs().max())
        per_row = n in ("y", "z", "dh", "dx") or a.dim() > 1
        size = b.abs().amax(-1, keepdim=True) if per_row and b.dim() > 1 else torch.full_like(b, big)
        f32 = 2.0 ** -24 * (256 if per_row else 16 * (rows / 256 + 256) ** 0.5 + 256)
        lim = u * b.abs() + f32 * size * 4 + (2.0 ** -24 if dtype == F16 else 0) + 1e-30
        if floor:
            lim = lim + floor.get(n, 0.0)
        assert a.shape == b.shape and bool(((a - b).abs() <= lim).all()), (what, n, float(((a - b).abs() - lim).max()), big)


@pytest.mark.parametrize("case", JOINTS, ids=lambda c: "x".join(map(str, c[0])) + f"-{c[1]}-{c[2]}-{c[5]}")
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_joint_and_its_gradients(dtype, case):
    shape, norm, gate, residual, res_scale, after = case
    t = _joint_inputs(31, dtype, *case)
    rows = math.prod(shape[:-1])
    for use in (("y", "z"), ("y",), ("z",)) if after else (("y",),):
        floor = _cancelled(t, norm, after, use) if shape[-1] == 1 else None                                       # (one value a row: a norm's gradient is nothing but rounding)
        _joint_close(_joint_run(t, norm, after, use=use), _joint_reference(t, norm, after, use=use), dtype, rows, use, floor)


def test_joint_many_rows_and_groups():
    """more rows than workgroups, a gate for each of many sequences; equal bits on every run"""
    for dtype, shape, gate in ((BF16, (3, 3001, 256), "vector"), (F32, (700, 5, 64), "batch"), (F16, (2, 9000, 72), "full")):
        case = (shape, "rms", gate, True, True, "layer")
        t = _joint_inputs(32, dtype, *case)
        a, b = _joint_run(t, "rms", "layer"), _joint_run(t, "rms", "layer")
        assert all(torch.equal(a[n], b[n]) for n in a)
        _joint_close(a, _joint_reference(t, "rms", "layer"), dtype, shape[0] * shape[1])


def test_joint_rows_of_zeros_and_not_numbers():
    A = _A()
    for norm in ("scale", "rms", "layer"):
        w = torch.ones(1 if norm == "scale" else 64).cuda()
        h = torch.randn(5, 64, generator=torch.Generator().manual_seed(33)).cuda()
        h[1] = 0
        h[3, 7] = math.nan
        h.requires_grad_()
        y = A.norm_gate_residual(h, norm=norm, weight=w)
        dh, = torch.autograd.grad(y, h, torch.ones_like(y))
        assert not y[1].any() and y[3].isnan().all() and y[[0, 2, 4]].isfinite().all()
        assert dh[1].isfinite().all() and dh[3].isnan().all() and dh[[0, 2, 4]].isfinite().all()
    # below the floor of a scale norm the divisor no longer follows the row
    h = (torch.randn(4, 32, generator=torch.Generator().manual_seed(34)) * 1e-7).cuda().requires_grad_()
    g = torch.tensor([3.0]).cuda()
    y = A.norm_gate_residual(h, norm="scale", weight=g)
    dh, = torch.autograd.grad(y, h, torch.ones_like(y))
    assert torch.allclose(y, h * 3e5, rtol=1e-6) and torch.allclose(dh, torch.full_like(dh, 3e5), rtol=1e-6)


def test_joint_strides_and_empty_calls():
    A = _A()
    for dtype in (F32, F16):
        wide = _rand(torch.Generator().manual_seed(35), 4, 9, 200, dtype=dtype)
        w = _rand(torch.Generator().manual_seed(36), 64, dtype=dtype)
        for lo in (0, 8, 3, 64):                                  # (3: rows off 16 bytes are read value by value, in another order of summation)
            h = wide[..., lo:lo + 64]
            y = A.norm_gate_residual(h, h, norm="rms", weight=w, gate=h)
            _joint_close({"y": y}, {"y": R.joint(h.double(), h.double(), h.double(), None, "rms", w.double(), None, None, None, None)[0]}, dtype, 36)
            if lo % 8 == 0:
                assert torch.equal(y, A.norm_gate_residual(h.contiguous(), h.contiguous(), norm="rms", weight=w, gate=h.contiguous()))
        part = wide[:, ::2, :64]                                  # rows evenly spaced within a sequence only: copied
        assert torch.equal(A.norm_gate_residual(part, norm="rms", weight=w), A.norm_gate_residual(part.contiguous(), norm="rms", weight=w))
        turned = wide[..., :64].transpose(0, 1)
        assert torch.equal(A.norm_gate_residual(turned, norm="rms", weight=w), A.norm_gate_residual(turned.contiguous(), norm="rms", weight=w))
        same = wide[:1, :1, :64].expand(4, 9, 64)
        assert torch.equal(A.norm_gate_residual(same, norm="rms", weight=w), A.norm_gate_residual(same.contiguous(), norm="rms", weight=w))
    h = torch.zeros(0, 5, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, z = A.norm_gate_residual(h, norm="rms", weight=w, next_norm="rms", next_weight=w)
    (y.sum() + z.sum()).backward()
    assert y.shape == z.shape == (0, 5, 64) and not w.grad.any()


def test_joint_captured_and_replayed():
    A = _A()
    t = _joint_inputs(37, BF16, (3, 50, 264), "rms", "batch", True, True, "layer")
    names = ("h", "x", "gate", "rs", "w", "w2", "b2")
    leaf = {n: t[n].detach().requires_grad_() for n in names}

    def step():
        y, z = A.norm_gate_residual(leaf["h"], leaf["x"], norm="rms", weight=leaf["w"], gate=leaf["gate"], res_scale=leaf["rs"], next_norm="layer", next_weight=leaf["w2"], next_bias=leaf["b2"])
        return [y.detach(), z.detach(), *torch.autograd.grad([y, z], [leaf[n] for n in names], [t["dy"], t["dz"]])]

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
        with torch.no_grad():
            for x in (*leaf.values(), t["dy"], t["dz"]):
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(turn)).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


# ------------------------------------------------------------------------------------------------------------------------ the whole unit

@pytest.mark.parametrize("rel_buckets", [0, 12])
def test_the_pose_heads_unit(rel_buckets, monkeypatch):
    """the unit as the pose network runs it -- norm, projection, attention with the gate, projection, scaled residual -- against its own composition in 64 bits on the
    CPU, values and every gradient (float32: products of at most 512 terms, 2^-24 each, in four layers after each other: 2e-5 of the largest entry)"""
    from tracklab_amd.backbones import rtmpose as P
    monkeypatch.setattr(P, "USE_TLK_GAU", True)
    torch.manual_seed(1)
    unit = P.GAU(256, 128, 2, rel_buckets=rel_buckets)
    with torch.no_grad():
        for p in unit.parameters():
            p.copy_(torch.randn_like(p) * (p.shape[-1] ** -0.5 if p.dim() > 1 and p.shape[-1] > 16 else 0.3) + (1.0 if p.dim() == 1 else 0.0))
    double = P.GAU(256, 128, 2, rel_buckets=rel_buckets).double()
    double.load_state_dict(unit.state_dict())
    x = torch.randn(6, 17, 256)
    up = torch.randn(6, 17, 256)
    xd = x.double().requires_grad_()
    want = double(xd)
    (want * up.double()).sum().backward()
    unit = unit.cuda()
    xc = x.cuda().requires_grad_()
    got = unit(xc)
    (got * up.cuda()).sum().backward()
    pairs = [(got, want), (xc.grad, xd.grad)] + [(a.grad, b.grad) for a, b in zip(unit.parameters(), double.parameters())]
    for i, (a, b) in enumerate(pairs):
        a, b = a.detach().double().cpu(), b.detach()
        assert float((a - b).abs().max()) <= 2e-5 * float(b.abs().max()), i


def test_the_pose_network_calls_the_operators(monkeypatch):
    """rtmpose(rel_buckets=...): the head runs on the operators (counted), in float16 as the pipeline holds it; without a bias nothing changes unless asked for"""
    from tracklab_amd import attention as A
    from tracklab_amd.backbones.rtmpose import rtmpose
    calls = []
    real = A.gated_attention
    monkeypatch.setattr(A, "gated_attention", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    x = torch.randn(3, 3, 256, 192, generator=torch.Generator().manual_seed(2)).half().cuda().contiguous(memory_format=torch.channels_last)
    plain, biased = rtmpose("t"), rtmpose("t", rel_buckets=8)
    with torch.no_grad():
        sx, sy = plain(x)
        assert not calls
        bx, by = biased(x)
    assert len(calls) == 1 and bx.shape == sx.shape and by.shape == sy.shape and bx.isfinite().all() and by.isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_a_block_of_both_operators(dtype):
    """two units after each other, the joint of the first being the second's first norm: the operators as a program strings them together, with gradients, against the same
    string in 64 bits from the same rounded weights (bf16: every tensor between the operators is rounded, 16 roundings of 2^-8 of the largest entry on the way)"""
    A = _A()
    g = torch.Generator().manual_seed(40)
    B, L, d, s, e = 3, 70, 64, 32, 96
    rnd = lambda *sh, std=1.0, mean=0.0: (torch.randn(*sh, generator=g) * std + mean).to(dtype)      # noqa: E731
    par = {"x": rnd(B, L, d), "n0": rnd(d, std=0.1, mean=1.0)}
    for i in range(2):
        par.update({f"wu{i}": rnd(e, d, std=d ** -0.5), f"wv{i}": rnd(e, d, std=d ** -0.5), f"wq{i}": rnd(s, d, std=d ** -0.5), f"wk{i}": rnd(s, d, std=d ** -0.5),
                    f"wo{i}": rnd(d, e, std=e ** -0.5), f"t{i}": rnd(16, 1, std=0.3), f"rs{i}": rnd(d, std=0.1, mean=1.0), f"n{i + 1}": rnd(d, std=0.1, mean=1.0)})
    up = rnd(B, L, d)
    buckets = A.relative_buckets(16, 40)
    lens = torch.tensor([70, 31, 50], dtype=torch.int32).cuda()

    def run(p, own):
        def attend(q, k, v, u, table, kind):
            if own:
                return A.gated_attention(q, k, v, u, kind=kind, bias=table, buckets=buckets, causal=True, lens=lens)
            away = torch.arange(L)[None] - torch.arange(L)[:, None]
            seen = (away <= 0)[None] & (torch.arange(L)[None, None] < lens.cpu()[:, None, None])
            sc = q @ k.transpose(1, 2) * s ** -0.5 + table[:, 0][buckets.cpu().long()[away.clamp(-40, 40) + 40]]
            w = (sc.relu() * seen) ** 2 if kind == "relu2" else torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
            return u * (w @ v)
        x = p["x"]
        z = A.norm_gate_residual(x, norm="rms", weight=p["n0"]) if own else R.joint(x, None, None, None, "rms", p["n0"], None, None, None, None)[0]
        for i, kind in enumerate(("relu2", "softmax")):
            u, v, q, k = (torch.nn.functional.linear(z, p[f"w{n}{i}"]) for n in "uvqk")
            o = torch.nn.functional.linear(attend(q, k, v, u, p[f"t{i}"], kind), p[f"wo{i}"])
            x, z = A.norm_gate_residual(o, x, res_scale=p[f"rs{i}"], next_norm="rms", next_weight=p[f"n{i + 1}"]) if own else \
                R.joint(o, x, None, p[f"rs{i}"], None, None, None, "rms", p[f"n{i + 1}"], None)
        return z

    own = {n: t.cuda().requires_grad_() for n, t in par.items()}
    ref = {n: t.double().requires_grad_() for n, t in par.items()}
    zo, zr = run(own, True), run(ref, False)
    go, gr = torch.autograd.grad(zo, list(own.values()), up.cuda()), torch.autograd.grad(zr, list(ref.values()), up.double())
    tol = 16 * R.U[dtype] if dtype == BF16 else 1e-4
    for n, a, b in zip(["z"] + list(own), (zo, *go), (zr, *gr)):
        a, b = a.detach().double().cpu(), b.detach()
        assert float((a - b).norm()) <= tol * float(b.norm()), n
