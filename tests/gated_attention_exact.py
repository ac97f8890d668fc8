"""gated_attention and its gradients from the definition in 64 bits on the tensors' device, for sizes at which sums cancel (a sequence and a head at a time).

The element bounds of gated_attention_reference.py add every rounding in absolute value and grow with the length; the tests that use this file bound the error's norm
instead.  A rounding is off by at most u = eps / 2 of the value, and, spread evenly within the step, by u / sqrt(3) in the root mean square; errors of different
pairs are independent and add in quadrature.  ``out`` takes two roundings (the weight as an operand, the result), dgate two (o as it was kept, the result), dq, dk and dv three
(the gradient behind the gate, the weight or score gradient as an operand, the result): at most u * sqrt(3 / 3) = u of the norm.  No rounding to the type enters
the bias gradient but its own: what remains are float32 sums."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attention(t, kind, causal=False, lens=None, start=0, scale=None):
    """t: q, k, v, gate, table, buckets, dout as the operator takes them -> out, dq, dk, dv, dgate, dtable in float64"""
    f = {n: None if t.get(n) is None else t[n].detach().double() for n in ("q", "k", "v", "gate", "table", "dout")}
    q, k, v = f["q"], f["k"], f["v"]
    B, Lq, H, dk = q.shape
    Lk, Hk, G = k.shape[1], k.shape[2], H // k.shape[2]
    dev = q.device
    scale = dk ** -0.5 if scale is None else scale
    res = {"out": torch.zeros(*q.shape[:3], v.shape[3], dtype=torch.float64, device=dev), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    if f["gate"] is not None:
        res["dgate"] = torch.zeros_like(res["out"])
    if f["table"] is not None:
        res["dtable"] = torch.zeros_like(f["table"])
        D = t["buckets"].numel() // 2
    i, j = torch.arange(Lq, device=dev)[:, None], torch.arange(Lk, device=dev)[None]
    for b in range(B):
        n = Lk if lens is None else min(Lk, max(0, int(lens[b])))
        away = j - i - (int(start[b]) if isinstance(start, torch.Tensor) else start)
        seen = (j < n) & ((away <= 0) | (not causal))
        for h in range(H):
            kh, vh, qh, up = k[b, :, h // G].contiguous(), v[b, :, h // G].contiguous(), q[b, :, h].contiguous(), f["dout"][b, :, h].contiguous()
            s = qh @ kh.t().contiguous() * scale
            if f["table"] is not None:
                slot = t["buckets"].long()[away.clamp(-D, D) + D]
                s = s + f["table"][:, h][slot]
            if kind == "relu2":
                root = torch.where(seen, s.clamp(min=0), torch.zeros_like(s))
                w = root * root
            else:
                w = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), -1).nan_to_num(nan=0.0)
            o = w @ vh
            if f["gate"] is not None:
                g = f["gate"][b, :, h]
                res["out"][b, :, h], res["dgate"][b, :, h], up = o * g, up * o, (up * g).contiguous()
            else:
                res["out"][b, :, h] = o
            dw = up @ vh.t().contiguous()
            ds = 2 * root * dw if kind == "relu2" else w * (dw - (up * o).sum(-1, keepdim=True))
            res["dq"][b, :, h] = ds @ kh * scale
            res["dk"][b, :, h // G] += ds.t().contiguous() @ qh * scale
            res["dv"][b, :, h // G] += w.t().contiguous() @ up
            if f["table"] is not None:
                res["dtable"][:, h].index_add_(0, slot.reshape(-1), ds.reshape(-1))
    return res


def run(t, kind, causal=False, lens=None, start=0, scale=None):
    """the operator's outputs and gradients under the same names"""
    from tracklab_amd import attention as A
    leaves = {n: t[n].detach().requires_grad_() for n in ("q", "k", "v", "gate", "table") if t.get(n) is not None}
    out = A.gated_attention(leaves["q"], leaves["k"], leaves["v"], leaves.get("gate"), kind=kind, scale=scale, bias=leaves.get("table"), buckets=t.get("buckets"), causal=causal,
                            lens=lens, q_start=start)
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(leaves, torch.autograd.grad(out, list(leaves.values()), t["dout"]))}}


def off(got, want):
    """norm of the error relative to the norm of the value"""
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-300))


def inputs(seed, dtype, B, Lq, Lk, H, Hk, dk, dv, gate=True, buckets=0, D=0, table_dtype=torch.float32, std=None):
    """tensors of unit spread (``std``: others by name) on the GPU, made from the seed alone"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    std = std or {}
    rnd = lambda n, *shape, dt=dtype: (torch.randn(*shape, generator=g, device="cuda") * std.get(n, 1.0)).to(dt)      # noqa: E731
    t = {"q": rnd("q", B, Lq, H, dk), "k": rnd("k", B, Lk, Hk, dk), "v": rnd("v", B, Lk, Hk, dv), "gate": rnd("gate", B, Lq, H, dv) if gate else None,
         "table": (rnd("table", buckets, H, dt=torch.float32) * 0.5).to(table_dtype) if buckets else None, "dout": rnd("dout", B, Lq, H, dv), "buckets": None}
    if buckets:
        from tracklab_amd import attention as A
        t["buckets"] = A.relative_buckets(buckets, D)
    return t
