"""The gated-attention operators from their definition in 64 bits, with bounds on how far a kernel may be from them.

A rounding to a type is off by at most u = eps / 2 of the value (``U``).  A float32 sum of n products is off by at most n * 2^-24 of the sum of their
magnitudes (``n`` counts every product and addition on the way to a value).  The bounds follow the kernels' roundings: weights, score gradients and the gradient
behind the gate once to the type, results once; scores, statistics and sums in float32.
float16 weights and score gradients are held with a power of two per row that puts the largest magnitude at 0.5 .. 128 (its square: up to 2^14), so the
absolute step of float16 (2^-25) is at most 2^-24 of the row's largest score gradient, and 2^-23 of its largest weight (a square: twice the exponent).
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E32 = 2.0 ** -24


def attention(q, k, v, gate, table, buckets, lens, start, kind, causal, scale, dout=None):
    """q (B, Lq, H, dk), ... as the operator takes them -> (values, bounds), dicts of float64 tensors"""
    dt = q.dtype
    u = U[dt]
    uw = 0.0 if dt == torch.float32 else u                     # float32 weights are not rounded again
    q, k, v, gate, dout = (t.detach().double().cpu() if t is not None else None for t in (q, k, v, gate, dout))
    B, Lq, H, dk = q.shape
    Lk, Hk, dv = k.shape[1], k.shape[2], v.shape[3]
    G = H // Hk
    qh, kh, vh = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(G, 1), v.transpose(1, 2).repeat_interleave(G, 1)
    i, j = torch.arange(Lq)[None, :, None], torch.arange(Lk)[None, None, :]
    st = torch.zeros(B, dtype=torch.long) if start is None else (start.cpu().long() if isinstance(start, torch.Tensor) else torch.full((B,), int(start)))
    away = j - i - st[:, None, None]
    seen = torch.ones(B, Lq, Lk, dtype=torch.bool)
    if causal:
        seen &= away <= 0
    n_keys = torch.full((B,), Lk) if lens is None else lens.cpu().long().clamp(0, Lk)
    gone = torch.arange(Lk)[None] >= n_keys[:, None]           # keys that may hold anything
    kh = kh.masked_fill(gone[:, None, :, None], 0.0)
    vh = vh.masked_fill(gone[:, None, :, None], 0.0)
    seen &= ~gone[:, None]
    score = qh @ kh.transpose(2, 3) * scale
    mag = qh.abs() @ kh.abs().transpose(2, 3) * abs(scale)
    slot = None
    if table is not None:
        D, nb = buckets.numel() // 2, table.shape[0]
        slot = buckets.cpu().long().clamp(0, nb - 1)[away.clamp(-D, D) + D]                          # (B, Lq, Lk)
        bias = table.detach().double().cpu()[slot].permute(0, 3, 1, 2)
        score, mag = score + bias, mag + bias.abs().nan_to_num(posinf=0.0, neginf=0.0)
    seen = seen[:, None].expand(B, H, Lq, Lk)
    eps_s = (dk + 6) * E32 * mag.masked_fill(~seen, 0.0)                                              # of a score
    if kind == "relu2":
        pos = torch.where(seen, score.clamp(min=0.0), torch.zeros_like(score))
        w = pos * pos
        dw_ = 2 * pos * eps_s + eps_s ** 2 + 4 * E32 * w
    else:
        top = torch.where(seen, score, torch.full_like(score, -math.inf)).amax(-1, keepdim=True)
        e = torch.where(seen, torch.exp(score - top.clamp(min=-1e300)), torch.zeros_like(score))
        w = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
        # exp of a float32 argument s - max: the argument's rounding is absolute, s * 2^-23 at most
        rel = 2 * (eps_s + 4 * E32 * mag.masked_fill(~seen, 0.0)).amax(-1, keepdim=True) + (Lk + 16) * E32
        dw_ = w * torch.expm1(rel.clamp(max=1.0))
    held = 2.0 ** -23 if dt == torch.float16 else 0.0
    dwr = dw_ + uw * w + held * w.amax(-1, keepdim=True)                                               # the weight as an operand
    o = w @ vh
    absv = vh.abs()
    do_ = dwr @ absv + (Lk + 4) * E32 * (w @ absv)
    tiny = 2.0 ** -24 if dt == torch.float16 else 0.0                                                 # half of float16's smallest step, generously
    gh = gate.transpose(1, 2) if gate is not None else None
    out = o if gh is None else o * gh
    val = {"out": out}
    bnd = {"out": (do_ if gh is None else do_ * gh.abs()) + (u + 2 * E32) * (out.abs() + do_) + tiny}
    if dout is None:
        return _back(val, bnd)
    up = dout.transpose(1, 2)
    d_up = torch.zeros_like(up)
    o_r = do_ + u * (o.abs() + do_) + tiny                                                             # o as it was kept
    if gh is not None:
        val["dgate"] = up * o
        bnd["dgate"] = up.abs() * o_r + u * (val["dgate"].abs() + up.abs() * o_r) + tiny
        up = up * gh
        d_up = uw * up.abs() + E32 * up.abs() + tiny
    dwt = up @ vh.transpose(2, 3)
    d_dwt = d_up @ absv.transpose(2, 3) + (dv + 4) * E32 * (up.abs() @ absv.transpose(2, 3))
    if kind == "relu2":
        ds = 2 * pos * dwt
        d_ds = 2 * (pos + eps_s) * d_dwt + 2 * eps_s * dwt.abs() * seen + 4 * E32 * ds.abs()
    else:
        delta = (up * o).sum(-1, keepdim=True)
        d_delta = (d_up * (o.abs() + o_r) + up.abs() * o_r).sum(-1, keepdim=True) + (dv + 4) * E32 * (up * o).abs().sum(-1, keepdim=True)
        ds = w * (dwt - delta)
        # (the weight comes back from the row's log-sum-exp: one more rounded exponent)
        d_w = dw_ + w * 8 * E32 * (mag.masked_fill(~seen, 0.0) + math.log(Lk + 2) + 4)
        d_ds = (w + d_w) * (d_dwt + d_delta) + d_w * (dwt - delta).abs() + 4 * E32 * w * (dwt.abs() + delta.abs())
    d_dsq = d_ds + uw * ds.abs() + (2.0 ** -23 * ds.abs().amax(-1, keepdim=True) if dt == torch.float16 else 0.0) + tiny * 0
    d_dsk = d_ds + uw * ds.abs() + (2.0 ** -23 * ds.abs().amax(-2, keepdim=True) if dt == torch.float16 else 0.0)
    if dt == torch.float16:
        dwr = dw_ + uw * w + 2.0 ** -23 * w.amax(-2, keepdim=True)
    chunks = (dv + 255) // 256
    val["dq"] = ds @ kh * scale
    bnd["dq"] = (d_dsq @ kh.abs() + (Lk * chunks + 8) * E32 * (ds.abs() @ kh.abs())) * abs(scale)
    fold = lambda t: t.reshape(B, Hk, G, *t.shape[2:]).sum(2)                                          # noqa: E731
    val["dk"] = fold(ds.transpose(2, 3) @ qh) * scale
    bnd["dk"] = fold(d_dsk.transpose(2, 3) @ qh.abs() + (Lq * G * chunks + 8) * E32 * (ds.abs().transpose(2, 3) @ qh.abs())) * abs(scale)
    val["dv"] = fold(w.transpose(2, 3) @ up)
    bnd["dv"] = fold(dwr.transpose(2, 3) @ (up.abs() + d_up) + w.transpose(2, 3) @ d_up + (Lq * G + 8) * E32 * (w.transpose(2, 3) @ up.abs()))
    for n in ("dq", "dk", "dv"):
        bnd[n] = bnd[n] + (u + 2 * E32) * (val[n].abs() + bnd[n]) + tiny
    val, bnd = _back(val, bnd)
    if table is not None:
        ut = U[table.dtype]
        val["dtable"], bnd["dtable"] = torch.zeros(nb, H, dtype=torch.float64), torch.zeros(nb, H, dtype=torch.float64)
        flat = slot.reshape(-1)
        for h in range(H):
            val["dtable"][:, h].index_add_(0, flat, ds[:, h].reshape(-1))
            bnd["dtable"][:, h].index_add_(0, flat, (d_ds[:, h] + (B * Lq * Lk) ** 0.5 * 8 * E32 * ds[:, h].abs()).reshape(-1))
        bnd["dtable"] += ut * (val["dtable"].abs() + bnd["dtable"]) + (2.0 ** -24 if table.dtype == torch.float16 else 0.0)
    return val, bnd


def _back(val, bnd):
    return {n: t.transpose(1, 2) for n, t in val.items()}, {n: t.transpose(1, 2) for n, t in bnd.items()}


def joint(h, x, gate, rs, norm, w, b, next_norm, w2, b2, eps=1e-5, next_eps=1e-5):
    """y, z of norm_gate_residual in 64 bits, differentiable; the tensors are taken as they are (pass float64)"""
    def n(kind, v, wt, bs, e):
        size = v.shape[-1]
        if kind in (None, "none"):
            return v
        if kind == "scale":
            return v * wt / (v.pow(2).sum(-1, keepdim=True).sqrt() / math.sqrt(size)).clamp(min=e)
        if kind == "rms":
            return v * wt / (v.pow(2).mean(-1, keepdim=True) + e).sqrt()
        m = v.mean(-1, keepdim=True)
        y = (v - m) / ((v - m).pow(2).mean(-1, keepdim=True) + e).sqrt() * wt
        return y if bs is None else y + bs
    y = n(norm, h, w, b, eps)
    if gate is not None:
        y = y * gate
    if x is not None:
        y = y + (x if rs is None else x * rs)
    return y, (n(next_norm, y, w2, b2, next_eps) if next_norm else None)
