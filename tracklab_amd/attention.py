"""The gated attention unit's operators on libtlk (``tlk_gau_attention_*``, ``tlk_norm_gate_residual_*``), with their gradients.

The pose networks' RTMCC head (tracklab/wrappers/pose_estimator/rtmlib_api.py:15-33; ``backbones/rtmpose.py``) ends in such a unit:
norm -> projection -> relu^2 attention over the keypoint tokens -> gate -> projection -> scaled residual.  Here its two hot pieces stand as
operators of their own, for the head's 17 tokens as for long sequences, padded batches and caches:

* ``gated_attention``     out = gate * (W v), W = relu(S)^2 or softmax(S), S = scale q k^T + a bias learned per bucket of the distance
* ``norm_gate_residual``  y = res_scale * x + gate * N1(h), z = N2(y)

Both are asynchronous on torch's current stream of the tensors' device, allocate through torch (so they can be captured into a graph), take no
CPU tensors (there is no CPU fallback) and raise ``TlkError`` for arguments they do not take.  Gradients come through torch's autograd; they
are computed without atomics: equal inputs give equal bits.  Forward-mode derivatives are refused.  To capture a backward pass into a graph, use leaves of which no eager autograd
graph is alive (torch ties a leaf's accumulation to the stream of its first use).
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import TlkError, _dtype_code, check, lib

KINDS = {"relu2": 0, "softmax": 1}
_TYPES = (torch.float32, torch.float16, torch.bfloat16)
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


# the same structures as one pack each: a call is mostly this module's own time on small inputs, and a ctypes field costs as much as a torch query
_GAU = struct.Struct("=14if4x12q8Q")
_NORM = struct.Struct("=4i5q2f8Q")
_GRADS = struct.Struct("=8Q")
assert _GAU.size == C.sizeof(GauArgs) and _NORM.size == C.sizeof(NormArgs) and _GRADS.size == C.sizeof(NormGrads)


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


def _no_tangent(what, *tensors):
    """the operators have no forward-mode derivative: a tangent would be lost without a word.  (Tangents live inside a level alone; asking every tensor takes 4 us.)"""
    for t in tensors if getattr(forward_ad, "_current_level", 0) >= 0 else ():
        _need(t is None or forward_ad.unpack_dual(t).tangent is None, what + ": no forward-mode derivatives")


def _ptr(t):
    return t.data_ptr() if t is not None else 0


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
    n0, n1, n2, n3 = t.shape
    s0, s1, s2, s3 = t.stride()
    if (s3 != 1 and n3 > 1) or t.data_ptr() % 16 or (n0 > 1 and s0 % vn) or (n2 > 1 and s2 % vn) or (n1 > 1 and (s1 % vn or not n3 <= s1 <= 1 << 22)):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        s0, s1, s2, s3 = t.stride()
    return t, (s0 if n0 > 1 else 0, s1 if n1 > 1 else n3, s2 if n2 > 1 else 0)


def _gau_args(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale):
    """the packed argument structure and the tensors it points to"""
    vn = 4 if q.dtype == torch.float32 else 8
    q, qs = _fit(q, vn)
    k, ks = _fit(k, vn)
    v, vs = _fit(v, vn)
    gs = (0, 0, 0)
    if gate is not None:
        gate, gs = _fit(gate, vn)
    B, Lq, H, dk = q.shape
    _, Lk, Hk, dv = v.shape
    start = isinstance(q_start, torch.Tensor)
    a = _GAU.pack(_dtype_code(q.dtype), kind, causal, table is not None and table.dtype == torch.float32, B, Lq, Lk, H, Hk, dk, dv,
                  table.shape[0] if table is not None else 0, buckets.numel() // 2 if table is not None else 0, 0 if start else q_start, scale, *qs, *ks, *vs, *gs,
                  q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(gate), _ptr(table), _ptr(buckets), _ptr(lens), q_start.data_ptr() if start else 0)
    return a, (q, k, v, gate)


def _gau_forward(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale, keep):
    """out, and for the backward pass what it needs of (o before the gate, a softmax row's maximum and sum)"""
    L, dev = _bound(), q.device
    a, held = _gau_args(q, k, v, gate, table, buckets, lens, q_start, kind, causal, scale)
    shape = (*q.shape[:3], v.shape[3])
    out = torch.empty(shape, dtype=q.dtype, device=dev)
    o = torch.empty(shape, dtype=torch.float32 if kind == 0 and q.dtype == torch.float16 else q.dtype, device=dev) if keep and gate is not None else None
    lse = torch.empty((*shape[:3], 2), dtype=torch.float32, device=dev) if keep and kind == 1 else None
    with _on(dev):
        n = L.tlk_gau_attention_workspace(a, 0) if k.shape[1] > 512 else 0            # (up to 512 keys a forward call needs none)
        ws = _bytes(n, dev)
        check(L.tlk_gau_attention_fwd(a, out.data_ptr(), _ptr(o), _ptr(lse), _ptr(ws), n, _stream(dev)))
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
            n = L.tlk_gau_attention_workspace(a, 1)
            ws = _bytes(n, dev)
            check(L.tlk_gau_attention_bwd(a, _ptr(dout), _ptr(o), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dgate), _ptr(dtable), _ptr(ws), n, _stream(dev)))
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
    _need(kind in KINDS, "gated_attention: kind must be 'relu2' or 'softmax'")
    B, Lq, H, dk = q.shape
    _, Lk, Hk, dv = v.shape
    dt, dev = q.dtype, q.device
    _need(q.is_cuda and dt in _TYPES, "gated_attention: cuda tensors of float32, float16 or bfloat16 (no CPU fallback)")
    _need(k.shape == (B, Lk, Hk, dk) and v.shape[0] == B, "gated_attention: shapes of q, k and v do not go together")
    _need(Hk > 0 and H > 0 and H % Hk == 0, "gated_attention: q's heads must be a multiple of k's")
    _need(1 <= dk <= 128 and dv >= 1, "gated_attention: 1 <= dk <= 128 and dv >= 1")
    _need(k.dtype == dt and v.dtype == dt and k.device == dev and v.device == dev, "gated_attention: q, k, v and gate must share type and device")
    if gate is not None:
        _need(gate.shape == (B, Lq, H, dv), "gated_attention: gate must have the result's shape")
        _need(gate.dtype == dt and gate.device == dev, "gated_attention: q, k, v and gate must share type and device")
    _need((bias is None) == (buckets is None), "gated_attention: a bias needs its buckets")
    if bias is not None:
        _need(bias.dim() == 2 and bias.shape[1] == H and bias.shape[0] > 0 and (bias.dtype == dt or bias.dtype == torch.float32) and bias.device == dev,
              "gated_attention: bias must be (num_buckets, heads) of q's type or float32")
        _need(buckets.dim() == 1 and buckets.shape[0] % 2 == 1 and buckets.shape[0] <= 4097 and buckets.dtype == torch.int32 and buckets.device == dev,
              "gated_attention: buckets must be (2 * max_distance + 1,) int32, max_distance <= 2048")
        bias, buckets = bias.contiguous(), buckets.contiguous()
    if lens is not None:
        _need(lens.shape == (B,) and lens.dtype == torch.int32 and lens.device == dev, "gated_attention: lens must be (B,) int32 on q's device")
        lens = lens.contiguous()
    if isinstance(q_start, torch.Tensor):
        _need(q_start.shape == (B,) and q_start.dtype == torch.int32 and q_start.device == dev, "gated_attention: q_start must be (B,) int32 on q's device")
        q_start = q_start.contiguous()
    else:
        q_start = int(q_start or 0)
        _need(-(1 << 29) <= q_start <= 1 << 29, "gated_attention: q_start must lie within 2^29")
    scale = dk ** -0.5 if scale is None else float(scale)
    vn = 4 if dt == torch.float32 else 8
    if dk % vn:                                            # widths that are no multiple of 16 bytes: zero columns change no product
        q, k = F.pad(q, (0, -dk % vn)), F.pad(k, (0, -dk % vn))
    if dv % vn:
        v, gate = F.pad(v, (0, -dv % vn)), F.pad(gate, (0, -dv % vn)) if gate is not None else None
    args = (q, k, v, gate, bias, buckets, lens, q_start, KINDS[kind], bool(causal), scale)
    _no_tangent("gated_attention", q, k, v, gate, bias)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (gate is not None and gate.requires_grad) or (bias is not None and bias.requires_grad)):
        out = _GatedAttention.apply(*args)
    else:
        out = _gau_forward(*args, False)[0]
    if dv % vn:
        out = out[..., :dv]
    return out.squeeze(2) if flat else out


# ------------------------------------------------------------------------------------------------------------------------------ joint

def _row_view(t, d):
    """(tensor, stride of its rows) with every row's values contiguous and the rows evenly spaced"""
    if t.is_contiguous():
        return t, d
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
    """the packed argument structure and the tensors it points to"""
    d = h.shape[-1]
    h, hs = _row_view(h, d)
    x, xs = _row_view(x, d) if x is not None else (None, 0)
    gate, gs = _row_view(gate, d) if gate is not None else (None, 0)
    a = _NORM.pack(_dtype_code(h.dtype), norm, next_norm, d, h.numel() // d, gate_rows, hs, xs, gs, eps, next_eps, h.data_ptr(), _ptr(x), _ptr(gate), _ptr(rs), _ptr(w),
                   _ptr(b), _ptr(w2), _ptr(b2))
    return a, (h, x, gate)


def _joint_forward(h, x, gate, rs, w, b, w2, b2, *plain):
    L, dev = _bound(), h.device
    a, held = _norm_args(h, x, gate, rs, w, b, w2, b2, *plain)
    y = torch.empty(h.shape, dtype=h.dtype, device=dev)
    z = torch.empty(h.shape, dtype=h.dtype, device=dev) if plain[1] else None
    with _on(dev):
        check(L.tlk_norm_gate_residual_fwd(a, y.data_ptr(), _ptr(z), _stream(dev)))
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
        g = _GRADS.pack(*[_ptr(t) for t in grads])
        with _on(dev):
            n = L.tlk_norm_gate_residual_workspace(a)
            ws = _bytes(n, dev)
            check(L.tlk_norm_gate_residual_bwd(a, _ptr(dy), _ptr(dz), g, _ptr(ws), n, _stream(dev)))
        return tuple(grads) + (None,) * len(ctx.plain)


def norm_gate_residual(h, residual=None, *, norm=None, weight=None, bias=None, eps=1e-5, gate=None, res_scale=None, next_norm=None, next_weight=None,
                       next_bias=None, next_eps=1e-5):
    """y = res_scale * residual + gate * N1(h), and with next_norm also z = N2(y): returns y or (y, z), in one pass over the rows.

    h, residual (..., d): cuda tensors of one type, d <= 8192 (rows evenly spaced are read in place, other layouts copied).  norm / next_norm: None,
    "scale" (v * weight / max(|v| / sqrt(d), eps), weight one value), "rms" (v * weight / sqrt(mean v^2 + eps), weight (d,)) or "layer" (weight (d,), bias
    (d,) or None).  gate: None, (d,), h's shape, or h's first dimensions followed by ones and d -- (B, 1, d): one gate for each sequence.
    res_scale: (d,) or None.  Statistics and sums are float32; z is normalised from y before its rounding."""
    _need(h.is_cuda and h.dtype in _TYPES, "norm_gate_residual: cuda tensors of float32, float16 or bfloat16 (no CPU fallback)")
    _need(h.dim() >= 1 and 1 <= h.shape[-1] <= 8192, "norm_gate_residual: rows of 1 to 8192 values")
    _need(norm in NORMS and next_norm in NORMS, "norm_gate_residual: a norm is None, 'scale', 'rms' or 'layer'")
    d, rows = h.shape[-1], h.numel() // h.shape[-1]
    n1, n2 = NORMS[norm], NORMS[next_norm]
    dt, dev = h.dtype, h.device
    for t in (residual, gate, weight, bias, res_scale, next_weight, next_bias):
        _need(t is None or (t.dtype == dt and t.device == dev), "norm_gate_residual: tensors must share type and device")
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
    _no_tangent("norm_gate_residual", *args[:8])
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:8]):
        return _NormGateResidual.apply(*args)
    return _joint_forward(*args)
