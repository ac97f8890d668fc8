"""The gated-attention operators without a GPU: what the C entries and the Python entry points refuse, the bucket map, the pose head's unit on the CPU."""
import ctypes as C
import math

import pytest
import torch

from tracklab_amd import attention as A
from tracklab_amd._lib import TlkError, lib

PTR = 1 << 20                                   # an aligned address that no refused call reads


def _gau(**over):
    a = A.GauArgs()
    a.dtype, a.kind, a.batch, a.len_q, a.len_k, a.heads, a.kv_heads, a.dim_k, a.dim_v, a.scale = 1, 0, 2, 5, 7, 4, 2, 64, 64, 0.125
    for s in (a.q_stride, a.k_stride, a.v_stride, a.gate_stride):
        s[:] = (4096, 256, 64)
    a.q = a.k = a.v = PTR
    for n, v in over.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


@pytest.mark.parametrize("over, words", [
    (dict(dtype=3), b"dtype"), (dict(kind=2), b"kind"), (dict(len_q=-1), b"lengths"), (dict(len_k=(1 << 28) + 1), b"lengths"), (dict(heads=3), b"multiple of kv_heads"),
    (dict(kv_heads=0), b"multiple of kv_heads"), (dict(dim_k=136), b"dim_k"), (dict(dim_k=12), b"dim_k"), (dict(dim_k=0), b"dim_k"), (dict(dim_v=20), b"dim_v"),
    (dict(num_buckets=4), b"bias needs"), (dict(table=PTR), b"bias needs"), (dict(num_buckets=4, table=PTR, bucket_of=PTR, max_distance=2049), b"max_distance"),
    (dict(q=None), b"null q"), (dict(v=None), b"null k or v"), (dict(k=PTR + 8), b"aligned"), (dict(gate=PTR + 2), b"aligned"),
    (dict(q_stride=(4096, 257, 64)), b"strides"), (dict(v_stride=(4096, -64, 64)), b"negative"),
])
def test_attention_entries_refuse(over, words):
    L = A._bound()
    a = _gau(**over)
    for rc in (L.tlk_gau_attention_workspace(C.byref(a), 0), L.tlk_gau_attention_fwd(C.byref(a), PTR, None, None, None, 0, None),
               L.tlk_gau_attention_bwd(C.byref(a), PTR, PTR, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 1 << 40, None)):
        assert rc == -1 and words in L.tlk_last_error(), L.tlk_last_error()


def test_attention_entries_refuse_missing_outputs_and_workspaces():
    L = A._bound()
    err = L.tlk_last_error
    a = _gau()
    assert L.tlk_gau_attention_fwd(None, PTR, None, None, None, 0, None) == -1 and b"null arguments" in err()
    assert L.tlk_gau_attention_fwd(C.byref(a), None, None, None, None, 0, None) == -1 and b"out" in err()
    assert L.tlk_gau_attention_fwd(C.byref(a), PTR + 4, None, None, None, 0, None) == -1 and b"aligned" in err()
    one = _gau(len_q=1, len_k=20000)                          # few rows over many keys: the keys are split
    need = L.tlk_gau_attention_workspace(C.byref(one), 0)
    assert need > 0
    assert L.tlk_gau_attention_fwd(C.byref(one), PTR, None, None, None, 0, None) == -1 and b"workspace" in err()
    assert L.tlk_gau_attention_fwd(C.byref(one), PTR, None, None, PTR, need - 1, None) == -1 and b"workspace" in err()
    soft = _gau(kind=1, gate=PTR)
    need = L.tlk_gau_attention_workspace(C.byref(soft), 1)
    args = [PTR] * 9
    for drop, words in ((0, b"dout"), (3, b"dq"), (4, b"dk"), (1, b"o_raw"), (2, b"lse"), (6, b"no place")):
        given = [None if i == drop else p for i, p in enumerate(args)]
        assert L.tlk_gau_attention_bwd(C.byref(soft), *given, need, None) == -1 and words in err(), (drop, err())
    assert L.tlk_gau_attention_bwd(C.byref(soft), *args, need - 1, None) == -1 and b"workspace" in err()
    # nothing to do is not an error
    assert L.tlk_gau_attention_fwd(C.byref(_gau(batch=0)), None, None, None, None, 0, None) == 0
    assert L.tlk_gau_attention_fwd(C.byref(_gau(len_q=0, q=None)), None, None, None, None, 0, None) == 0


def _norm(**over):
    a = A.NormArgs()
    a.dtype, a.norm, a.next_norm, a.dim, a.rows, a.gate_rows, a.h_stride, a.x_stride, a.gate_stride, a.eps, a.next_eps = 1, 2, 0, 64, 12, 1, 64, 64, 64, 1e-5, 1e-5
    a.h = a.weight = PTR
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over, words", [
    (dict(dtype=9), b"dtype"), (dict(norm=4), b"unknown norm"), (dict(dim=0), b"dim"), (dict(dim=8193, h_stride=9000), b"dim"), (dict(rows=-1), b"rows"), (dict(h=None), b"null input"),
    (dict(weight=None), b"weight"), (dict(next_norm=1), b"weight"), (dict(bias=PTR), b"bias"), (dict(res_scale=PTR), b"residual"), (dict(h_stride=63), b"row strides"),
    (dict(gate=PTR, gate_rows=5), b"gate_rows"), (dict(gate=PTR, gate_rows=0), b"gate_rows"), (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"),
    (dict(gate=PTR, gate_rows=2, rows=140000), b"65535"),
])
def test_joint_entries_refuse(over, words):
    L = A._bound()
    a = _norm(**over)
    g = A.NormGrads(*[PTR] * 8)
    for rc in (L.tlk_norm_gate_residual_fwd(C.byref(a), PTR, PTR if a.next_norm else None, None), L.tlk_norm_gate_residual_workspace(C.byref(a)),
               L.tlk_norm_gate_residual_bwd(C.byref(a), PTR, None, C.byref(g), PTR, 1 << 40, None)):
        assert rc == -1 and words in L.tlk_last_error(), L.tlk_last_error()


def test_joint_entries_refuse_missing_outputs_and_workspaces():
    L = A._bound()
    err = L.tlk_last_error
    a = _norm()
    assert L.tlk_norm_gate_residual_fwd(C.byref(a), None, None, None) == -1 and b"null output" in err()
    assert L.tlk_norm_gate_residual_fwd(C.byref(a), PTR, PTR, None) == -1 and b"next norm" in err()
    need = L.tlk_norm_gate_residual_workspace(C.byref(a))
    full = [PTR] * 8
    assert L.tlk_norm_gate_residual_bwd(C.byref(a), PTR, None, C.byref(A.NormGrads(*full)), PTR, need - 1, None) == -1 and b"workspace" in err()
    assert L.tlk_norm_gate_residual_bwd(C.byref(a), PTR, PTR, C.byref(A.NormGrads(*full)), PTR, need, None) == -1 and b"next norm" in err()
    assert L.tlk_norm_gate_residual_bwd(C.byref(a), PTR, None, C.byref(A.NormGrads(None, *full[1:])), PTR, need, None) == -1 and b"no place" in err()
    assert L.tlk_norm_gate_residual_bwd(C.byref(a), PTR, None, C.byref(A.NormGrads(PTR, PTR, PTR, PTR, None)), PTR, need, None) == -1 and b"no place" in err()
    assert L.tlk_norm_gate_residual_bwd(C.byref(a), PTR, None, None, PTR, need, None) == -1
    assert L.tlk_norm_gate_residual_fwd(C.byref(_norm(rows=0, h=None)), None, None, None) == 0


def test_python_entry_points_have_no_cpu_fallback():
    t = torch.zeros(1, 4, 2, 64)
    with pytest.raises(TlkError, match="no CPU fallback"):
        A.gated_attention(t, t, t)
    with pytest.raises(TlkError, match="no CPU fallback"):
        A.norm_gate_residual(t)
    with pytest.raises(TlkError, match="kind"):
        A.gated_attention(t, t, t, kind="sigmoid")
    with pytest.raises(TlkError, match="head dimension"):
        A.gated_attention(t[:, :, 0], t, t)


@pytest.mark.parametrize("n, d, both", [(32, 128, True), (32, 128, False), (16, 16, True), (7, 5, True), (4, 1, True), (2, 300, False), (64, 20, False)])
def test_relative_buckets(n, d, both):
    m = A.relative_buckets(n, d, both, device="cpu")
    assert m.dtype == torch.int32 and m.numel() == 2 * d + 1 and 0 <= int(m.min()) and int(m.max()) < n
    m = m.tolist()
    behind, ahead = m[:d + 1][::-1], m[d:]                     # distances 0, -1, -2, ... and 0, 1, 2, ...
    assert behind == sorted(behind) and behind[0] == 0
    if both:
        half = n // 2
        assert [b + half for b in behind[1:]] == ahead[1:]
        exact = max(1, half // 2)
        assert behind[:min(exact, d + 1)] == list(range(min(exact, d + 1)))
    else:
        assert set(ahead) == {0}
    with pytest.raises(TlkError):
        A.relative_buckets(1, 4)


def test_pose_unit_with_a_position_bias_on_the_cpu():
    """a bias table of zeros changes nothing; one that forbids every distance but zero leaves each token with itself; the CPU composition has gradients"""
    from tracklab_amd.backbones.rtmpose import GAU, rtmpose
    torch.manual_seed(0)
    plain = GAU(32, 16, 2).double()
    unit = GAU(32, 16, 2, rel_buckets=8, max_distance=4).double()
    unit.load_state_dict(plain.state_dict(), strict=False)
    x = torch.randn(3, 17, 32, dtype=torch.float64)
    assert torch.equal(unit(x), plain(x))
    with torch.no_grad():
        unit.rel_bias.fill_(-1e6)
        unit.rel_bias[0] = 0.0
    alone = unit(x)
    one = torch.cat([unit(x[:, i:i + 1]) for i in range(17)], 1)
    assert torch.allclose(alone, one, rtol=1e-12, atol=1e-12)
    unit(x).square().sum().backward()
    assert unit.rel_bias.grad[0].abs().sum() > 0
    net = rtmpose("t", device="cpu", dtype=torch.float32, channels_last=False, rel_buckets=8)
    assert net.gau.rel_bias.shape == (8, 1) and "gau.buckets" not in net.state_dict()
    assert "gau.rel_bias" not in rtmpose("t", device="cpu", dtype=torch.float32, channels_last=False).state_dict()


def test_the_reference_of_the_gpu_tests_agrees_with_reverse_differentiation():
    """tests/gated_attention_reference.py writes the gradients out; here they are checked against torch's float64 autograd of the forward formula"""
    import gated_attention_reference as R
    g = torch.Generator().manual_seed(3)
    B, Lq, Lk, H, Hk, dk, dv, D, nb = 2, 5, 9, 4, 2, 6, 5, 3, 4
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)      # noqa: E731
    q, k, v, gate, table, dout = rnd(B, Lq, H, dk), rnd(B, Lk, Hk, dk), rnd(B, Lk, Hk, dv), rnd(B, Lq, H, dv), rnd(nb, H), rnd(B, Lq, H, dv)
    buckets = torch.randint(0, nb, (2 * D + 1,), generator=g, dtype=torch.int32)
    lens, start = torch.tensor([9, 4], dtype=torch.int32), torch.tensor([4, -2], dtype=torch.int32)
    R.U[torch.float64] = 2.0 ** -53
    for kind in ("relu2", "softmax"):
        for causal in (False, True):
            t = [x.clone().requires_grad_() for x in (q, k, v, gate, table)]
            away = torch.arange(Lk)[None, None] - torch.arange(Lq)[None, :, None] - start[:, None, None]
            seen = (torch.arange(Lk)[None, None] < lens[:, None, None]) & ((away <= 0) | (not causal))
            s = torch.einsum("bihd,bjhd->bhij", t[0], t[1].repeat_interleave(2, 2)) * 0.3 + t[4][buckets.long()[away.clamp(-D, D) + D]].permute(0, 3, 1, 2)
            if kind == "relu2":
                w = (s.relu() * seen[:, None]) ** 2
            else:
                w = torch.softmax(s.masked_fill(~seen[:, None], -1e30), -1) * seen[:, None]
            out = torch.einsum("bhij,bjhd->bihd", w, t[2].repeat_interleave(2, 2)) * t[3]
            grads = torch.autograd.grad(out, t, dout)
            val, _ = R.attention(q, k, v, gate, table, buckets, lens, start, kind, causal, 0.3, dout)
            assert torch.allclose(val["out"], out.detach(), rtol=1e-12, atol=1e-12)
            for n, gr in zip(("dq", "dk", "dv", "dgate", "dtable"), grads):
                assert torch.allclose(val[n], gr, rtol=1e-10, atol=1e-11), (kind, causal, n)


def test_workspace_sizes_are_those_of_the_plan():
    L = lib() and A._bound()
    a = _gau(len_q=1, len_k=20000, batch=3, dim_v=128)
    n = L.tlk_gau_attention_workspace(C.byref(a), 0)
    assert n % (3 * 4 * (128 + 2) * 4) == 0                    # (splits, batch x heads rows, dim_v sums + maximum and sum)
    assert L.tlk_gau_attention_workspace(C.byref(_gau()), 0) == 0


def test_workspaces_must_be_aligned():
    L, err = A._bound(), A._bound().tlk_last_error
    one = _gau(len_q=1, len_k=20000)
    need = L.tlk_gau_attention_workspace(C.byref(one), 0)
    assert need > 0 and L.tlk_gau_attention_fwd(C.byref(one), PTR, None, None, PTR + 8, need, None) == -1 and b"aligned" in err()
    soft = _gau(kind=1)
    need = L.tlk_gau_attention_workspace(C.byref(soft), 1)
    assert L.tlk_gau_attention_bwd(C.byref(soft), *[PTR] * 8, PTR + 8, need, None) == -1 and b"aligned" in err()


def test_few_workgroups_over_many_keys_are_split():
    L = A._bound()
    size = lambda **over: L.tlk_gau_attention_workspace(C.byref(_gau(heads=1, kv_heads=1, batch=1, **over)), 0)      # noqa: E731
    assert size(len_q=128, len_k=512) == 0 and size(len_q=128, len_k=1024) == 2 * 128 * (64 + 2) * 4          # 512 keys a workgroup at least
    assert size(len_q=128 * 128, len_k=4096) > 0 and size(len_q=128 * 129, len_k=4096) == 0                   # a workgroup for every other CU
    assert size(len_q=128 * 128, len_k=2047) == 0 and size(len_q=128 * 128, len_k=2048) > 0                   # what the split saves against what its sums move
