"""The gated attention unit's operators on libtlk (``tlk_gau_attention_*``, ``tlk_norm_gate_residual_*``), with their gradients.

The pose networks' RTMCC head (tracklab/wrappers/pose_estimator/rtmlib_api.py:15-33; ``backbones/rtmpose.py``) ends in such a unit:
norm -> projection -> relu^2 attention over the keypoint tokens -> gate -> projection -> scaled residual.  Here its two hot pieces stand as
operators of their own, for the head's 17 tokens as for long sequences, padded batches and caches:

* ``gated_attention``     out = gate * (W v), W = relu(S)^2 or softmax(S), S = scale q k^T + a bias learned per bucket of the distance
* ``norm_gate_residual``  y = res_scale * x + gate * N1(h), z = N2(y)

Both are asynchronous on torch's current stream of the tensors' device, allocate through torch (so they can be captured into a graph), take no
CPU tensors (there is no CPU fallback) and raise ``TlkError`` for arguments they do not take.  Gradients come through torch's autograd; they
are computed without atomics: equal inputs give equal bits.  To capture a backward pass into a graph, use leaves of which no eager autograd
graph is alive (torch ties a leaf's accumulation to the stream of its first use).
"""
from __future__ import annotations

import ctypes as C
import math

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ._lib import TlkError, _dtype_code, check, lib

KINDS = {"relu2": 0, "softmax": 1}
NORMS = {None: 0, "none": 0, "scale": 1, "rms": 2, "layer": 3}


class GauArgs(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("dtype", "kind", "causal", "table_f32", "batch", "len_q", "len_k", "heads", "kv_heads", "dim_k", "dim_v",
                                         "num_buckets", "max_distance", "q_start")] + \
               [("scale", C.c_float)] + [(n, C.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride", "gate_stride")] + \
               [(n, C.c_void_p) for n in ("q", "k", "v", "gate", "table", "bucket_of", "lens", "q_start_dev")]


class NormArgs(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("dtype", "norm", "next_norm", "dim")] + [(n, C.c_int64) for n in ("rows", "gate_rows", "h_stride", "x_stride", "gate_stride")] + \
               [("eps", C.c_float), ("next_eps", C.c_float)] + [(n, C.c_void_p) for n in ("h", "x", "gate", "res_scale", "weight", "bias", "next_weight", "next_bias")]


class NormGrads(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("dh", "dx", "dgate", "dres_scale", "dweight", "dbias", "dnext_weight", "dnext_bias")]


def _bound():
    L = lib()
    if not getattr(L, "_gau_bound", False):
        P, LL = C.c_void_p, C.c_longlong
        L.tlk_gau_attention_workspace.argtypes, L.tlk_gau_attention_workspace.restype = [P, C.c_int], LL
        L.tlk_gau_attention_fwd.argtypes = [P] * 5 + [LL, P]
        L.tlk_gau_attention_bwd.argtypes = [P] * 10 + [LL, P]
        L.tlk_norm_gate_residual_workspace.argtypes, L.tlk_norm_gate_residual_workspace.restype = [P], LL
        L.tlk_norm_gate_residual_fwd.argtypes = [P] * 4
        L.tlk_norm_gate_residual_bwd.argtypes = [P] * 5 + [LL, P]
        L._gau_bound = True
    return L


def _need(ok, what):
    if not ok:
        raise TlkError(what)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _bytes(n, dev):
    if n < 0:
        check(int(n))
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


class _on:
    """launches go to the tensors' device, whichever is current"""
    __slots__ = ("ctx",)

    def __init__(self, dev):
        self.ctx = torch.cuda.device(dev) if torch.cuda.current_device() != dev.index else None

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *a):
        if self.ctx is not None:
            self.ctx.__exit__(*a)


# ------------------------------------------------------------------------------------------------------------------------- attention

def relative_buckets(num_buckets, max_distance, bidirectional=True, device="cuda"):
    """The bucket of every distance key - query in -max_distance .. max_distance, int32 (2 * max_distance + 1): exact near zero, then logarithmic up to
    max_distance, which all further distances share; bidirectional: one half of the buckets for keys behind the query, one for keys ahead of it.
    ``gated_attention`` takes any such map; ``torch.arange(2 * D + 1)`` gives every distance a bias of its own."""
    _need(max_distance >= 1 and num_buckets >= (4 if bidirectional else 2), "relative_buckets: needs max_distance >= 1 and at least 2 buckets a direction")
    half = num_buckets // 2 if bidirectional else num_buckets
    exact = max(1, half // 2)
    out = []
    for d in range(-max_distance, max_distance + 1):
        a = abs(d) if bidirectional else max(-d, 0)
        if a >= exact and max_distance > exact:
            a = exact + int(math.log(a / exact) / math.log(max_distance / exact) * (half - exact) + 1e-9)
        out.append(min(a, half - 1) + (half if bidirectional and d > 0 else 0))
    return torch.tensor(out, dtype=torch.int32, device=device)


def _fit(t, vn):
    """the tensor with a contiguous last dimension, 16-byte aligned rows and heads (as it is where it already has them), and its three strides"""
    s = t.stride()
    if (t.shape[-1] > 1 and s[3] != 1) or t.data_ptr() % 16 or any(t.shape[i] > 1 and s[i] % vn for i in range(3)) or (t.shape[1] > 1 and not t.shape[3] <= s[1] <= 1 << 22):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        s = t.stride()
    return t, tuple(s[i] if t.shape[i] > 1 else (t.shape[3] if i == 1 else 0) for i in range(3))


def _gau_args(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale):
    """the filled argument structure and the tensors it points to"""
    a = GauArgs()
    vn = 4 if q.dtype == torch.float32 else 8
    a.dtype, a.kind, a.causal = _dtype_code(q.dtype), kind, causal
    a.batch, a.len_q, a.heads, a.dim_k = q.shape
    a.len_k, a.kv_heads, a.dim_v = k.shape[1], k.shape[2], v.shape[3]
    a.scale = scale
    q, a.q_stride[:] = _fit(q, vn)
    k, a.k_stride[:] = _fit(k, vn)
    v, a.v_stride[:] = _fit(v, vn)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if gate is not None:
        gate, a.gate_stride[:] = _fit(gate, vn)
        a.gate = gate.data_ptr()
    if table is not None:
        a.num_buckets, a.max_distance, a.table_f32 = table.shape[0], buckets.numel() // 2, table.dtype == torch.float32
        a.table, a.bucket_of = table.data_ptr(), buckets.data_ptr()
    if lens is not None:
        a.lens = lens.data_ptr()
    if isinstance(q_start, torch.Tensor):
        a.q_start_dev = q_start.data_ptr()
    else:
        a.q_start = q_start
    return a, (q, k, v, gate, table)


def _gau_forward(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale, keep):
    """out, and for the backward pass what it needs of (o before the gate, log-sum-exp)"""
    L, dev = _bound(), q.device
    a, held = _gau_args(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale)
    shape = (a.batch, a.len_q, a.heads, a.dim_v)
    out = torch.empty(shape, dtype=q.dtype, device=dev)
    o = torch.empty_like(out) if keep and gate is not None else None
    lse = torch.empty(shape[:3], dtype=torch.float32, device=dev) if keep and kind == 1 else None
    with _on(dev):
        n = L.tlk_gau_attention_workspace(C.byref(a), 0)
        ws = _bytes(n, dev)
        check(L.tlk_gau_attention_fwd(C.byref(a), out.data_ptr(), _ptr(o), _ptr(lse), _ptr(ws), n, _stream(dev)))
    return out, (o if gate is not None else (out if kind == 1 else None)), lse


class _GatedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale):
        out, o, lse = _gau_forward(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale, True)
        ctx.plain = (kind, causal, scale, q_start if not isinstance(q_start, torch.Tensor) else None)
        ctx.save_for_backward(q, k, v, gate, table, buckets, lens, q_start if isinstance(q_start, torch.Tensor) else None, o, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, gate, table, buckets, lens, start, o, lse = ctx.saved_tensors
        kind, causal, scale, q_start = ctx.plain
        L, dev = _bound(), q.device
        a, held = _gau_args(q, k, v, gate, table, buckets, lens, start if start is not None else q_start, kind, causal, scale)
        dout = dout.contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=dev) if t is not None else None      # noqa: E731
        dq, dk, dv, dgate, dtable = new(q), new(k), new(v), new(gate), new(table)
        with _on(dev):
            n = L.tlk_gau_attention_workspace(C.byref(a), 1)
            ws = _bytes(n, dev)
            check(L.tlk_gau_attention_bwd(C.byref(a), _ptr(dout), _ptr(o), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dgate), _ptr(dtable), _ptr(ws), n, _stream(dev)))
        return dq, dk, dv, dgate, dtable, None, None, None, None, None, None


def gated_attention(q, k, v, gate=None, *, kind="relu2", scale=None, bias=None, buckets=None, causal=False, lens=None, q_start=0):
    """out = gate * (W v), W = relu(S)^2 (kind "relu2") or softmax(S) ("softmax"), S = scale * q k^T + bias[buckets[clip(j - i - q_start)], head].

    q (B, Lq, H, dk), k (B, Lk, Hk, dk), v (B, Lk, Hk, dv), gate (B, Lq, H, dv) or None: cuda tensors of one type (float32, float16, bfloat16), any strides
    (views of a projection are read in place where rows are 16-byte aligned, copied otherwise); H a multiple of Hk (heads share keys and values); dk <= 128.
    Without a head dimension -- (B, L, d), all of them -- there is one head and the result is (B, Lq, dv).
    scale: 1 / sqrt(dk) by default.  bias (num_buckets, H) of q's type or float32 with buckets (2 D + 1,) int32 (``relative_buckets``): learned, distances
    beyond D share the end entries (D <= 2048).  causal: key j is seen up to j <= i + q_start.  lens (B,) int32 on the device: keys at or behind it are not
    read (their memory may hold anything).  q_start: position of q's first row among the keys, an int or (B,) int32 on the device -- one new token at the
    end of a cache: q_start = lens - 1.  Rows that see no key give zeros.  All query rows are computed, those of a padded batch too.
    Non-finite values among the keys below lens follow IEEE arithmetic (a weight of zero times infinity is NaN)."""
    flat = q.dim() == 3
    if flat:
        _need(k.dim() == 3 and v.dim() == 3 and (gate is None or gate.dim() == 3), "gated_attention: q, k, v and gate must all have a head dimension, or none of them")
        q, k, v, gate = q.unsqueeze(2), k.unsqueeze(2), v.unsqueeze(2), gate.unsqueeze(2) if gate is not None else None
    _need(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "gated_attention: q, k and v must be (B, L, heads, d) or (B, L, d)")
    _need(kind in KINDS, f"gated_attention: kind must be one of {sorted(KINDS)}")
    B, Lq, H, dk = q.shape
    Lk, Hk, dv = k.shape[1], k.shape[2], v.shape[3]
    _need(q.is_cuda and q.dtype in (torch.float32, torch.float16, torch.bfloat16), "gated_attention: cuda tensors of float32, float16 or bfloat16 (no CPU fallback)")
    _need(tuple(k.shape) == (B, Lk, Hk, dk) and tuple(v.shape) == (B, Lk, Hk, dv), "gated_attention: shapes of q, k and v do not go together")
    _need(Hk > 0 and H > 0 and H % Hk == 0, "gated_attention: q's heads must be a multiple of k's")
    _need(1 <= dk <= 128 and dv >= 1, "gated_attention: 1 <= dk <= 128 and dv >= 1")
    _need(gate is None or tuple(gate.shape) == (B, Lq, H, dv), "gated_attention: gate must have the result's shape")
    _need((bias is None) == (buckets is None), "gated_attention: a bias needs its buckets")
    for t in (k, v, gate):
        _need(t is None or (t.dtype == q.dtype and t.device == q.device), "gated_attention: q, k, v and gate must share type and device")
    if bias is not None:
        _need(bias.dim() == 2 and bias.shape[1] == H and bias.shape[0] > 0 and bias.dtype in (q.dtype, torch.float32) and bias.device == q.device,
              "gated_attention: bias must be (num_buckets, heads) of q's type or float32")
        _need(buckets.dim() == 1 and buckets.numel() % 2 == 1 and buckets.numel() <= 4097 and buckets.dtype == torch.int32 and buckets.device == q.device,
              "gated_attention: buckets must be (2 * max_distance + 1,) int32, max_distance <= 2048")
        bias, buckets = bias.contiguous(), buckets.contiguous()
    for n, t in (("lens", lens), ("q_start", q_start)):
        if isinstance(t, torch.Tensor):
            _need(tuple(t.shape) == (B,) and t.dtype == torch.int32 and t.device == q.device, f"gated_attention: {n} must be (B,) int32 on q's device")
    lens = lens.contiguous() if lens is not None else None
    q_start = q_start.contiguous() if isinstance(q_start, torch.Tensor) else int(q_start or 0)
    scale = dk ** -0.5 if scale is None else float(scale)
    vn = 4 if q.dtype == torch.float32 else 8
    if dk % vn:                                            # widths that are no multiple of 16 bytes: zero columns change no product
        q, k = F.pad(q, (0, -dk % vn)), F.pad(k, (0, -dk % vn))
    if dv % vn:
        v, gate = F.pad(v, (0, -dv % vn)), F.pad(gate, (0, -dv % vn)) if gate is not None else None
    args = (q, k, v, gate, bias, buckets, lens, q_start, KINDS[kind], bool(causal), scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, gate, bias)):
        out = _GatedAttention.apply(*args)
    else:
        out = _gau_forward(*args, False)[0]
    if dv % vn:
        out = out[..., :dv]
    return out.squeeze(2) if flat else out


# ------------------------------------------------------------------------------------------------------------------------------ joint

def _row_view(t, d):
    """(tensor, stride of its rows) with every row's values contiguous and the rows evenly spaced"""
    s, n = t.stride(), t.dim()
    if d == 1 or s[-1] == 1:
        step, want = None, None
        for i in range(n - 2, -1, -1):
            if t.shape[i] == 1:
                continue
            if step is None:
                step = s[i]
            elif s[i] != want:
                break
            want = s[i] * t.shape[i]
        else:
            step = d if step is None else step
            if step >= d:
                return t, step
    return t.contiguous(), d


def _norm_args(h, x, gate, rs, w, b, w2, b2, norm, next_norm, eps, next_eps, gate_rows):
    a = NormArgs()
    d = h.shape[-1]
    a.dtype, a.norm, a.next_norm, a.dim = _dtype_code(h.dtype), norm, next_norm, d
    a.rows, a.gate_rows, a.eps, a.next_eps = h.numel() // d, gate_rows, eps, next_eps
    h, a.h_stride = _row_view(h, d)
    a.h = h.data_ptr()
    if x is not None:
        x, a.x_stride = _row_view(x, d)
        a.x = x.data_ptr()
    if gate is not None:
        gate, a.gate_stride = _row_view(gate, d)
        a.gate = gate.data_ptr()
    a.res_scale, a.weight, a.bias, a.next_weight, a.next_bias = _ptr(rs), _ptr(w), _ptr(b), _ptr(w2), _ptr(b2)
    return a, (h, x, gate)


def _joint_forward(h, x, gate, rs, w, b, w2, b2, *plain):
    L, dev = _bound(), h.device
    a, held = _norm_args(h, x, gate, rs, w, b, w2, b2, *plain)
    y = torch.empty(h.shape, dtype=h.dtype, device=dev)
    z = torch.empty(h.shape, dtype=h.dtype, device=dev) if plain[1] else None
    with _on(dev):
        check(L.tlk_norm_gate_residual_fwd(C.byref(a), y.data_ptr(), _ptr(z), _stream(dev)))
    return (y, z) if z is not None else y


class _NormGateResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, x, gate, rs, w, b, w2, b2, *plain):
        ctx.plain = plain
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, x, gate, rs, w, b, w2, b2)
        return _joint_forward(h, x, gate, rs, w, b, w2, b2, *plain)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz=None):
        saved = ctx.saved_tensors
        h = saved[0]
        L, dev = _bound(), h.device
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if t is not None else None for t in saved]
        if h.numel() == 0 or (dy is None and dz is None):
            return tuple(g.zero_() if g is not None else None for g in grads) + (None,) * len(ctx.plain)
        a, held = _norm_args(*saved, *ctx.plain)
        dy, dz = (t.contiguous() if t is not None else None for t in (dy, dz))
        g = NormGrads(*[_ptr(t) for t in grads])
        with _on(dev):
            n = L.tlk_norm_gate_residual_workspace(C.byref(a))
            ws = _bytes(n, dev)
            check(L.tlk_norm_gate_residual_bwd(C.byref(a), _ptr(dy), _ptr(dz), C.byref(g), _ptr(ws), n, _stream(dev)))
        return tuple(grads) + (None,) * len(ctx.plain)


def norm_gate_residual(h, residual=None, *, norm=None, weight=None, bias=None, eps=1e-5, gate=None, res_scale=None, next_norm=None, next_weight=None,
                       next_bias=None, next_eps=1e-5):
    """y = res_scale * residual + gate * N1(h), and with next_norm also z = N2(y): returns y or (y, z), in one pass over the rows.

    h, residual (..., d): cuda tensors of one type, d <= 8192 (rows evenly spaced are read in place, other layouts copied).  norm / next_norm: None,
    "scale" (v * weight / max(|v| / sqrt(d), eps), weight one value), "rms" (v * weight / sqrt(mean v^2 + eps), weight (d,)) or "layer" (weight (d,), bias
    (d,) or None).  gate: None, (d,), h's shape, or h's first dimensions followed by ones and d -- (B, 1, d): one gate for each sequence.
    res_scale: (d,) or None.  Statistics and sums are float32; z is normalised from y before its rounding."""
    _need(h.is_cuda and h.dtype in (torch.float32, torch.float16, torch.bfloat16), "norm_gate_residual: cuda tensors of float32, float16 or bfloat16 (no CPU fallback)")
    _need(h.dim() >= 1 and 1 <= h.shape[-1] <= 8192, "norm_gate_residual: rows of 1 to 8192 values")
    _need(norm in NORMS and next_norm in NORMS, "norm_gate_residual: a norm is None, 'scale', 'rms' or 'layer'")
    d, rows = h.shape[-1], h.numel() // h.shape[-1]
    n1, n2 = NORMS[norm], NORMS[next_norm]
    for t in (residual, gate, weight, bias, res_scale, next_weight, next_bias):
        _need(t is None or (t.dtype == h.dtype and t.device == h.device), "norm_gate_residual: tensors must share type and device")
    _need(residual is None or residual.shape == h.shape, "norm_gate_residual: the residual must have h's shape")
    _need(res_scale is None or (residual is not None and tuple(res_scale.shape) == (d,)), "norm_gate_residual: res_scale is (d,) and goes with a residual")
    for kind, w, b in ((n1, weight, bias), (n2, next_weight, next_bias)):
        _need((w is None) == (kind == 0), "norm_gate_residual: a norm needs its weight, and a weight its norm")
        _need(w is None or (w.numel() == 1 if kind == 1 else tuple(w.shape) == (d,)), "norm_gate_residual: a scale norm's weight is one value, the others' (d,)")
        _need(b is None or (kind == 3 and tuple(b.shape) == (d,)), "norm_gate_residual: only the layer norm takes a bias, (d,)")
    _need(eps >= 0 and next_eps >= 0, "norm_gate_residual: eps must not be negative")
    gate_rows = 1
    if gate is not None:
        if gate.dim() == 1:
            gate_rows = max(1, rows)
            _need(gate.shape[0] == d, "norm_gate_residual: gate does not go with h")
        elif gate.shape != h.shape:
            _need(gate.dim() == h.dim() and gate.shape[-1] == d, "norm_gate_residual: gate does not go with h")
            lead = 0
            while lead < h.dim() - 1 and gate.shape[lead] == h.shape[lead]:
                lead += 1
            _need(all(n == 1 for n in gate.shape[lead:-1]), "norm_gate_residual: a shared gate has h's first dimensions, then ones")
            gate_rows = math.prod(h.shape[lead:-1])
            _need(rows == 0 or gate_rows == 1 or rows // gate_rows <= 65535, "norm_gate_residual: more than 65535 shared gate rows")
            gate_rows = max(1, gate_rows)
    small = [t.contiguous() if t is not None else None for t in (res_scale, weight, bias, next_weight, next_bias)]
    args = (h, residual, gate, *small, n1, n2, float(eps), float(next_eps), gate_rows)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:8]):
        return _NormGateResidual.apply(*args)
    return _joint_forward(*args)
