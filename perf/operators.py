"""Cases of the gated-attention operators and their plain forms.

Two operators, both parts of a gated attention unit (the block behind the pose network's keypoint tokens):

* attention: out = gate * (W v), W = relu(S)^2 or softmax(S), S = scale * q k^T + a bias learned per bucket of the distance j - i
* norm: y = res_scale * x + gate * N1(h), z = N2(y)

``own`` False computes them from elementary torch operations in 32 bits; True calls ``tracklab_amd.attention``.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def _attention(name, dtype, B, Lq, Lk, H, Hk, dk, dv, kind, gate, buckets, distance, causal, ragged, train):
    return {"name": name, "op": "attention", "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hk": Hk, "dk": dk, "dv": dv, "kind": kind, "gate": gate,
            "buckets": buckets, "distance": distance, "causal": causal, "ragged": ragged, "train": train}


def _norm(name, dtype, B, L, d, norm, gate, residual, next_norm, train):
    return {"name": name, "op": "norm", "dtype": dtype, "B": B, "L": L, "d": d, "norm": norm, "gate": gate, "residual": residual, "next": next_norm, "train": train}


def listed():
    return [
        # the pose head's unit on the crops of 24 frames with 100 people each: 17 keypoint tokens, s = 128, e = 512
        _attention("pose_crops_f16", "f16", 2400, 17, 17, 1, 1, 128, 512, "relu2", True, 32, 16, False, False, False),
        # the same for the few people of one camera frame: latency
        _attention("pose_one_frame_f16", "f16", 8, 17, 17, 1, 1, 128, 512, "relu2", True, 32, 16, False, False, False),
        # fine-tuning the head at the framework's default precision
        _attention("pose_finetune_f32", "f32", 512, 17, 17, 1, 1, 128, 512, "relu2", True, 32, 16, False, False, True),
        # a causal unit over long sequences, scoring
        _attention("unit_long_bf16", "bf16", 4, 8192, 8192, 1, 1, 128, 1024, "relu2", True, 32, 128, True, False, False),
        # the same unit in training
        _attention("unit_train_bf16", "bf16", 4, 4096, 4096, 1, 1, 128, 1024, "relu2", True, 32, 128, True, False, True),
        # softmax heads that share keys and values, in training
        _attention("heads_train_bf16", "bf16", 4, 2048, 2048, 16, 4, 64, 64, "softmax", False, 32, 128, True, False, True),
        # a padded batch of odd lengths and widths seen in both directions, in training
        _attention("padded_train_f16", "f16", 6, 1021, 1021, 8, 8, 72, 104, "softmax", True, 48, 200, False, True, True),
        # one new token a sequence over caches of different lengths
        _attention("one_token_bf16", "bf16", 32, 1, 16384, 16, 4, 128, 128, "softmax", False, 32, 128, True, True, False),
        # the block's joint for one camera frame: latency
        _norm("joint_one_frame_f16", "f16", 8, 17, 256, "none", "none", True, "scale", False),
        # the same for 24 frames with 100 people each
        _norm("joint_crops_f16", "f16", 2400, 17, 256, "scale", "vector", True, "scale", False),
        # wide rows in training: norm, gate of every element, scaled residual, the next block's norm
        _norm("joint_train_bf16", "bf16", 4, 4096, 4096, "rms", "full", True, "rms", True),
        # odd widths, a gate for each sequence
        _norm("joint_train_f32", "f32", 7, 1201, 1000, "layer", "batch", True, "layer", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["crops", "unit", "heads", "token", "norm", "norm"])
    if what == "norm":
        d = rng.choice([8 * _log_int(rng, 8, 512), 8 * _log_int(rng, 8, 512), _log_int(rng, 65, 4095)])
        rows = _log_int(rng, 16, max(64, 2 ** 26 // d))
        B = rng.choice([1, 3, 8])
        norm, after = rng.choice([("none", "scale"), ("scale", "scale"), ("rms", "rms"), ("layer", "layer"), ("rms", "none"), ("layer", "scale")])
        return _draw(_norm("", rng.choice(["f16", "bf16", "f32"]), B, max(1, rows // B), d, norm, rng.choice(["none", "vector", "batch", "full"]), rng.random() < 0.8, after, rng.random() < 0.6))
    kind, dtype, train = rng.choice(["relu2", "softmax"]), rng.choice(["f16", "bf16", "f32"]), rng.random() < 0.5
    distance = rng.choice([16, 64, 128, 300])
    buckets = rng.choice([0, 16, 32, 48])
    if what == "crops":
        L = rng.randint(5, 133)
        return _draw(_attention("", dtype, _log_int(rng, 1, 20000 // L), L, L, 1, 1, rng.choice([64, 128]), rng.choice([128, 256, 512]), kind, True, buckets, 16, False, False, train))
    if what == "unit":
        L = _log_int(rng, 100, 4096)
        return _draw(_attention("", dtype if L < 1500 else rng.choice(["f16", "bf16"]), rng.randint(1, 3), L, L, 1, 1, 128, rng.choice([384, 512, 768, 1024]), kind, True, buckets, distance,
                                rng.random() < 0.6, rng.random() < 0.4, train))
    if what == "heads":
        L, Hk = _log_int(rng, 60, 2048), rng.choice([1, 2, 4])
        H, B = Hk * rng.choice([1, 2, 4]), rng.randint(1, 4)
        dk = rng.choice([64, 128, 8 * rng.randint(4, 16)])
        return _draw(_attention("", dtype if L < 700 else rng.choice(["f16", "bf16"]), B, L, L, H, Hk, dk, rng.choice([dk, 8 * rng.randint(4, 16)]), kind, rng.random() < 0.3, buckets, distance,
                                rng.random() < 0.6, rng.random() < 0.5, train))
    Hk = rng.choice([1, 2, 4])
    dk = rng.choice([64, 128])
    return _draw(_attention("", rng.choice(["f16", "bf16", "f32"]), rng.randint(1, 24), rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 64, 16384), Hk * rng.choice([1, 4, 7]), Hk, dk, dk,
                            kind, rng.random() < 0.3, buckets, distance, True, True, False))


def _draw(case):
    del case["name"]
    return case


def _lengths(c):
    """keys of each sequence: evenly spread from a third of the room to all of it (``prepare`` shuffles them)"""
    return [c["Lk"] - (c["Lk"] * 2 // 3) * b // max(1, c["B"] - 1) for b in range(c["B"])]


def _bucket_map(c):
    """bucket of every distance -D .. D (all that lie further share the last ones): exact near zero, then logarithmic; two halves where both directions occur"""
    D, n = c["distance"], c["buckets"]
    both = not c["causal"]
    half = n // 2 if both else n
    exact = half // 2
    out = []
    for d in range(-D, D + 1):
        a = abs(d) if both else max(-d, 0)
        b = a if a < exact else min(half - 1, exact + int(math.log(a / exact) / math.log(D / exact) * (half - exact) + 1e-9)) if D > exact else min(a, half - 1)
        out.append(b + (half if both and d > 0 else 0))
    return out


def prepare(case, seed):
    c = case
    dev, dt = "cuda", DTYPES[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dt)

    s = {"case": c}
    if c["op"] == "norm":
        B, L, d = c["B"], c["L"], c["d"]

        def weights(kind):
            return {"scale": lambda: (rand(1, std=0.1, mean=1.0), None), "rms": lambda: (rand(d, std=0.1, mean=1.0), None),
                    "layer": lambda: (rand(d, std=0.1, mean=1.0), rand(d, std=0.1)), "none": lambda: (None, None)}[kind]()

        s["h"] = rand(B, L, d)
        s["x"] = rand(B, L, d) if c["residual"] else None
        s["res_scale"] = rand(d, std=0.1, mean=1.0) if c["residual"] else None
        s["gate"] = {"none": lambda: None, "vector": lambda: rand(d, std=0.1, mean=0.5), "batch": lambda: rand(B, 1, d, std=0.3, mean=0.5), "full": lambda: rand(B, L, d)}[c["gate"]]()
        s["weight"], s["bias"] = weights(c["norm"])
        s["next_weight"], s["next_bias"] = weights(c["next"])
        s["dy"] = rand(B, L, d) if c["train"] else None
        s["dz"] = rand(B, L, d) if c["train"] and c["next"] != "none" else None
        s["leaves"] = ["h", "x", "res_scale", "gate", "weight", "bias", "next_weight", "next_bias"]
    else:
        B, Lq, Lk, H, Hk, dk, dv = c["B"], c["Lq"], c["Lk"], c["H"], c["Hk"], c["dk"], c["dv"]
        # a unit's gate and values are slices of one projection; its queries and keys come from another
        if c["gate"] and Lq == Lk and H == Hk:
            uv = rand(B, Lq, 2 * H * dv + 64)
            s["gate"] = uv[..., :H * dv].view(B, Lq, H, dv)
            s["v"] = uv[..., H * dv:2 * H * dv].view(B, Lk, H, dv)
        else:
            s["gate"] = rand(B, Lq, H, dv) if c["gate"] else None
            s["v"] = rand(B, Lk, Hk, dv)
        s["q"] = rand(B, Lq, H, dk)
        s["k"] = rand(B, Lk, Hk, dk)
        s["table"] = rand(c["buckets"], H, std=0.5) if c["buckets"] else None
        s["map"] = torch.tensor(_bucket_map(c), dtype=torch.int32, device=dev) if c["buckets"] else None
        lens = torch.tensor(_lengths(c), dtype=torch.int32, device=dev)[torch.randperm(B, generator=g, device=dev)] if c["ragged"] else None
        s["lens"] = lens
        # the new rows of a cache stand at its end
        s["start"] = lens - Lq if c["ragged"] and c["causal"] and Lq < Lk else None
        s["dout"] = rand(B, Lq, H, dv, std=0.02) if c["train"] else None
        s["leaves"] = ["q", "k", "v", "gate", "table"]
    if c["train"]:
        for n in s["leaves"]:
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
    return s


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_attention(state)


def _own(s):
    from tracklab_amd import attention as A
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        if c["op"] == "norm":
            norm, after = (None if n == "none" else n for n in (c["norm"], c["next"]))
            got = A.norm_gate_residual(s["h"], s["x"], norm=norm, weight=s["weight"], bias=s["bias"], gate=s["gate"], res_scale=s["res_scale"], next_norm=after,
                                       next_weight=s["next_weight"], next_bias=s["next_bias"])
            out = {"y": got[0], "z": got[1]} if after else {"y": got}
            douts = [s["dy"], s["dz"]][:len(out)]
        else:
            out = {"out": A.gated_attention(s["q"], s["k"], s["v"], s["gate"], kind=c["kind"], bias=s["table"], buckets=s["map"], causal=c["causal"], lens=s["lens"], q_start=s["start"])}
            douts = [s["dout"]]
        if c["train"]:
            names = [n for n in s["leaves"] if s[n] is not None]
            grads = torch.autograd.grad(list(out.values()), [s[n] for n in names], douts)
            out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


# ---------------------------------------------------------------------------------------------- plain forms, 32 bits

def _plain_norm_fwd(kind, v, w, b, eps=1e-5):
    """N(v) and what its gradient needs"""
    if kind == "none":
        return v, None, None
    d = v.shape[-1]
    if kind == "scale":
        n = v.square().sum(-1, keepdim=True).sqrt() * d ** -0.5
        inv = 1.0 / n.clamp(min=eps)
        return v * inv * w, v * inv, torch.where(n < eps, torch.zeros_like(inv), inv)
    if kind == "rms":
        inv = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
        return v * inv * w, v * inv, inv
    m = v - v.mean(-1, keepdim=True)
    inv = (m.square().mean(-1, keepdim=True) + eps).rsqrt()
    return m * inv * w + b, m * inv, inv


def _plain_norm_bwd(kind, dn, v, w, hat, inv, eps=1e-5):
    """gradients of N(v) to v, its weight and its bias"""
    if kind == "none":
        return dn, None, None
    if kind == "scale":
        n = v.square().sum(-1, keepdim=True).sqrt() * v.shape[-1] ** -0.5
        t = dn * w
        dv = t / n.clamp(min=eps) - hat * inv * (t * hat).mean(-1, keepdim=True)
        return dv, (dn * hat).sum().reshape(1), None
    t = dn * w
    dv = (t - hat * (t * hat).mean(-1, keepdim=True)) * inv
    if kind == "layer":
        dv = (t - t.mean(-1, keepdim=True) - hat * (t * hat).mean(-1, keepdim=True)) * inv
    return dv, (dn * hat).sum((0, 1)), dn.sum((0, 1)) if kind == "layer" else None


def _plain_norm(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    h, x, rs, gate, w, b, w2, b2, dy, dz = (None if s[n] is None else s[n].float() for n in ("h", "x", "res_scale", "gate", "weight", "bias", "next_weight", "next_bias", "dy", "dz"))
    n1, hat1, inv1 = _plain_norm_fwd(c["norm"], h, w, b)
    y = n1 if gate is None else n1 * gate
    y = y if x is None else y + x * rs
    z, hat2, inv2 = _plain_norm_fwd(c["next"], y, w2, b2)
    out = {"y": y, "z": z} if c["next"] != "none" else {"y": y}
    if c["train"]:
        if c["next"] != "none":
            back, out["dnext_weight"], out["dnext_bias"] = _plain_norm_bwd(c["next"], dz, y, w2, hat2, inv2)
            dy = dy + back
        if x is not None:
            out["dx"], out["dres_scale"] = dy * rs, (dy * x).sum((0, 1))
        if gate is not None:
            dg = dy * n1
            out["dgate"] = dg.sum((0, 1)) if c["gate"] == "vector" else dg.sum(1, keepdim=True) if c["gate"] == "batch" else dg
            dy = dy * gate
        out["dh"], out["dweight"], out["dbias"] = _plain_norm_bwd(c["norm"], dy, h, w, hat1, inv1)
    return {n: v.to(dt) for n, v in out.items() if v is not None}


def _plain_attention(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    B, Lq, Lk, H, Hk, dk, dv = c["B"], c["Lq"], c["Lk"], c["H"], c["Hk"], c["dk"], c["dv"]
    G = H // Hk
    dev = s["q"].device

    def heads(t):                                          # (B, L, heads, d) -> (B, heads, L, d)
        return t.float().transpose(1, 2).contiguous()

    q, k, v = heads(s["q"]), heads(s["k"]).repeat_interleave(G, 1), heads(s["v"]).repeat_interleave(G, 1)
    scale = dk ** -0.5
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    start = s["start"] if s["start"] is not None else torch.zeros(B, dtype=torch.int32, device=dev)
    i = torch.arange(Lq, device=dev)[None, :, None] + start[:, None, None]
    j = torch.arange(Lk, device=dev)[None, None, :]
    if s["table"] is not None:
        bucket = s["map"].long()[(j - i).clamp(-c["distance"], c["distance"]) + c["distance"]]             # (B or 1, Lq, Lk)
        score += s["table"].float().t()[:, bucket].transpose(0, 1)
    seen = torch.ones(1, Lq, Lk, dtype=torch.bool, device=dev)
    if c["causal"]:
        seen = seen & (j <= i)
    if s["lens"] is not None:
        seen = seen & (j < s["lens"][:, None, None])
    seen = seen[:, None]
    if c["kind"] == "relu2":
        pos = score.clamp(min=0) * seen
        wgt = pos.square()
    else:
        top = score.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
        e = torch.exp(score - top.clamp(min=-1e30)) * seen
        wgt = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
        del e
    o = torch.matmul(wgt, v)
    gate = heads(s["gate"]) if s["gate"] is not None else None
    out = {"out": (o * gate if gate is not None else o).transpose(1, 2)}
    if c["train"]:
        do = heads(s["dout"])
        if gate is not None:
            out["dgate"] = (do * o).transpose(1, 2)
            do = do * gate
        dvv = torch.matmul(wgt.transpose(2, 3).contiguous(), do)
        dw = torch.matmul(do, v.transpose(2, 3).contiguous())
        ds = 2 * pos * dw if c["kind"] == "relu2" else wgt * (dw - (wgt * dw).sum(-1, keepdim=True))
        del dw, wgt
        out["dq"] = (torch.matmul(ds, k) * scale).transpose(1, 2)
        dkk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
        out["dk"] = dkk.view(B, Hk, G, Lk, dk).sum(2).transpose(1, 2)
        out["dv"] = dvv.view(B, Hk, G, Lk, dv).sum(2).transpose(1, 2)
        if s["table"] is not None:
            # every distance first: with keys in reverse, row i of rows one longer than the count of distances starts i places further, so that a distance is a column
            ds = torch.nn.functional.pad(ds.sum(0, dtype=torch.float64).flip(2), (0, Lq)).view(H, -1)[:, :Lq * (Lk + Lq - 1)]
            by_distance = ds.view(H, Lq, Lk + Lq - 1).sum(1).flip(1)                                       # distances -(Lq - 1) .. Lk - 1
            away = torch.arange(1 - Lq, Lk, device=dev).clamp(-c["distance"], c["distance"]) + c["distance"]
            total = torch.zeros(H, c["buckets"], dtype=torch.float64, device=dev).index_add_(1, s["map"].long()[away], by_distance)
            out["dtable"] = total.t().float()
    return {n: v.to(dt).contiguous() for n, v in out.items()}


# ------------------------------------------------------------------------------------------------- work and exact values

def _pairs(c):
    """(query, key) pairs that are not masked, over all sequences, of one head"""
    lens = _lengths(c) if c["ragged"] else [c["Lk"]] * c["B"]
    total = 0
    for n in lens:
        start = n - c["Lq"] if c["ragged"] and c["causal"] and c["Lq"] < c["Lk"] else 0
        total += sum(min(n, max(0, i + start + 1)) for i in range(c["Lq"])) if c["causal"] else n * c["Lq"]
    return total


def work(case):
    c = case
    b = SIZE[c["dtype"]]
    if c["op"] == "norm":
        n = c["B"] * c["L"] * c["d"]
        gate = {"none": 0, "vector": c["d"], "batch": c["B"] * c["d"], "full": n}[c["gate"]]
        outs = 2 if c["next"] != "none" else 1
        moved = n * (1 + c["residual"] + outs) + gate
        if c["train"]:
            moved += n * (outs + 1 + c["residual"]) + gate
        return {"bytes": float(moved * b), "flops": 12.0 * n * (3 if c["train"] else 1)}
    q = c["B"] * c["Lq"] * c["H"]
    keys = (sum(_lengths(c)) if c["ragged"] else c["B"] * c["Lk"]) * c["Hk"]
    rows = q * (c["dk"] + c["dv"] * (2 if c["gate"] else 1)) + keys * (c["dk"] + c["dv"])
    if c["train"]:
        rows += q * (c["dk"] + c["dv"] * (2 if c["gate"] else 1)) + keys * (c["dk"] + c["dv"])
    return {"bytes": float(rows * b), "flops": 2.0 * _pairs(c) * c["H"] * (c["dk"] + c["dv"]) * (3 if c["train"] else 1)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(s) if case["op"] == "norm" else _exact_attention(s)


def _exact_norm(s):
    """both norms and the joint as one composition in 64 bits; its gradients by reverse differentiation of that composition"""
    c = s["case"]
    names = [n for n in s["leaves"] if s[n] is not None]
    t = {n: s[n].detach().double().requires_grad_(c["train"]) for n in names}

    def norm(kind, v, w, b):
        size = v.shape[-1]
        if kind == "scale":
            return v * w / torch.clamp(torch.linalg.vector_norm(v, dim=-1, keepdim=True) / math.sqrt(size), min=1e-5)
        if kind == "rms":
            return v * w / torch.sqrt((v * v).sum(-1, keepdim=True) / size + 1e-5)
        if kind == "layer":
            mean = v.sum(-1, keepdim=True) / size
            return (v - mean) / torch.sqrt(((v - mean) ** 2).sum(-1, keepdim=True) / size + 1e-5) * w + b
        return v

    with torch.set_grad_enabled(c["train"]):
        y = norm(c["norm"], t["h"], t.get("weight"), t.get("bias"))
        if "gate" in t:
            y = t["gate"] * y
        if "x" in t:
            y = y + t["res_scale"] * t["x"]
        out = {"y": y}
        if c["next"] != "none":
            out["z"] = norm(c["next"], y, t.get("next_weight"), t.get("next_bias"))
        if c["train"]:
            grads = torch.autograd.grad(list(out.values()), [t[n] for n in names], [s[n].double() for n in (["dy", "dz"] if "z" in out else ["dy"])])
            out.update({"d" + n: g for n, g in zip(names, grads)})
    return {n: v.detach() for n, v in out.items()}


def _exact_attention(s):
    """sequence by sequence and head by head from the definition, in 64 bits (short sequences: all at once)"""
    c = s["case"]
    B, Lq, Lk, H, Hk = c["B"], c["Lq"], c["Lk"], c["H"], c["Hk"]
    f = {n: None if s[n] is None else s[n].detach().double() for n in ("q", "k", "v", "gate", "table", "dout")}
    dev = s["q"].device
    out = {"out": torch.zeros(B, Lq, H, c["dv"], dtype=torch.float64, device=dev)}
    if c["train"]:
        out.update({"d" + n: torch.zeros_like(f[n], memory_format=torch.contiguous_format) for n in s["leaves"] if f[n] is not None})
    step = max(1, min(B, 40_000_000 // (Lq * Lk)))
    for b0 in range(0, B, step):
        part = slice(b0, min(B, b0 + step))
        nb = part.stop - b0
        first = s["start"][part].long() if s["start"] is not None else torch.zeros(nb, dtype=torch.long, device=dev)
        count = s["lens"][part].long() if s["lens"] is not None else torch.full((nb,), Lk, dtype=torch.long, device=dev)
        away = torch.arange(Lk, device=dev).view(1, 1, Lk) - torch.arange(Lq, device=dev).view(1, Lq, 1) - first.view(nb, 1, 1)
        mask = (torch.arange(Lk, device=dev).view(1, 1, Lk) < count.view(nb, 1, 1)).expand(nb, Lq, Lk)
        if c["causal"]:
            mask = mask & (away <= 0)
        slot = s["map"].long()[torch.clamp(away, -c["distance"], c["distance"]) + c["distance"]] if f["table"] is not None else None
        for h in range(H):
            qh, kh, vh = f["q"][part, :, h], f["k"][part, :, h // (H // Hk)], f["v"][part, :, h // (H // Hk)]
            score = torch.bmm(qh, kh.transpose(1, 2).contiguous()) / math.sqrt(c["dk"])
            if slot is not None:
                score = score + f["table"][:, h][slot]
            if c["kind"] == "relu2":
                root = torch.where(mask, torch.relu(score), torch.zeros_like(score))
                weight = root * root
            else:
                weight = torch.nan_to_num(torch.softmax(torch.where(mask, score, torch.full_like(score, -math.inf)), -1), nan=0.0)
            mixed = torch.bmm(weight, vh.contiguous())
            g = f["gate"][part, :, h] if f["gate"] is not None else None
            out["out"][part, :, h] = mixed if g is None else mixed * g
            if not c["train"]:
                continue
            up = f["dout"][part, :, h]
            if g is not None:
                out["dgate"][part, :, h] = up * mixed
                up = up * g
            out["dv"][part, :, h // (H // Hk)] += torch.bmm(weight.transpose(1, 2).contiguous(), up.contiguous())
            dweight = torch.bmm(up.contiguous(), vh.transpose(1, 2).contiguous())
            if c["kind"] == "relu2":
                dscore = 2 * root * dweight
            else:
                dscore = weight * (dweight - (up * mixed).sum(-1, keepdim=True))
            out["dq"][part, :, h] = torch.bmm(dscore, kh.contiguous()) / math.sqrt(c["dk"])
            out["dk"][part, :, h // (H // Hk)] += torch.bmm(dscore.transpose(1, 2).contiguous(), qh.contiguous()) / math.sqrt(c["dk"])
            if slot is not None:
                out["dtable"][:, h] += torch.zeros(c["buckets"], dtype=torch.float64, device=dev).index_add_(0, slot.reshape(-1), dscore.reshape(-1))
    return out
