"""Cases of the conditioned-image-block operators -- group norm with an activation over channels-last images, cross
attention from an image's positions to an encoder's states, and dropout from a counter-based generator -- with each
operator's plain form in elementary torch operations and its definition in 64 bits.

A case is one pass: the forward pass alone where a user serves, forward and backward where a user trains."""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_M32 = 0xFFFFFFFF


def listed():
    return [
        # one small feature map on its way through a served block: launch latency is all there is
        {"name": "norm_small", "op": "norm", "n": 1, "h": 16, "w": 16, "c": 64, "groups": 8, "act": "silu", "type": "f16",
         "train": False},
        # the convolution workload's batch of feature maps, normalised between two convolutions
        {"name": "norm_maps", "op": "norm", "n": 8, "h": 256, "w": 256, "c": 64, "groups": 8, "act": "silu", "type": "f16",
         "train": False},
        # a wide training step's mid-resolution maps, forward and backward
        {"name": "norm_train", "op": "norm", "n": 16, "h": 64, "w": 64, "c": 512, "groups": 32, "act": "silu", "type": "bf16",
         "train": True},
        # odd sizes in exact fp32: groups of ten channels, an image that no tile divides
        {"name": "norm_odd_f32", "op": "norm", "n": 3, "h": 37, "w": 53, "c": 60, "groups": 6, "act": "relu", "type": "f32",
         "train": True},
        # one new position a sequence against a ragged batch of a few hundred states: latency
        {"name": "attend_one", "op": "attend", "b": 8, "lq": 1, "lk": 700, "hq": 8, "hkv": 2, "d": 64, "type": "bf16",
         "ragged": True, "mask": False, "fused": False, "train": False},
        # one new position against a very long encoded sequence, queries sharing heads: bandwidth
        {"name": "attend_one_long", "op": "attend", "b": 4, "lq": 1, "lk": 100003, "hq": 16, "hkv": 4, "d": 128,
         "type": "f16", "ragged": False, "mask": False, "fused": True, "train": False},
        # 64x64 image positions against a few hundred conditioning states, narrow heads, served
        {"name": "attend_image", "op": "attend", "b": 8, "lq": 4096, "lk": 333, "hq": 8, "hkv": 8, "d": 40, "type": "f16",
         "ragged": True, "mask": False, "fused": True, "train": False},
        # a training step with padded conditioning states and one sample whose condition is dropped altogether
        {"name": "attend_train", "op": "attend", "b": 6, "lq": 4096, "lk": 1024, "hq": 8, "hkv": 8, "d": 64, "type": "bf16",
         "ragged": False, "mask": True, "fused": True, "train": True},
        # exact fp32 training on a small odd problem
        {"name": "attend_odd_f32", "op": "attend", "b": 3, "lq": 577, "lk": 201, "hq": 4, "hkv": 4, "d": 24, "type": "f32",
         "ragged": True, "mask": False, "fused": False, "train": True},
        # the largest: 128x128 positions against thousands of states, shared heads, forward and backward
        {"name": "attend_train_large", "op": "attend", "b": 2, "lq": 16384, "lk": 4099, "hq": 16, "hkv": 4, "d": 128,
         "type": "bf16", "ragged": False, "mask": False, "fused": False, "train": True},
        # one image's residual branch, forward and backward
        {"name": "dropout_small", "op": "dropout", "numel": 65537, "p": 0.1, "type": "f32", "residual": True, "train": True},
        # the convolution workload's maps added to their residual under dropout, forward and backward
        {"name": "dropout_maps", "op": "dropout", "numel": 8 * 256 * 256 * 64, "p": 0.1, "type": "bf16", "residual": True,
         "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "attend", "attend", "attend", "serve", "dropout"])
    kind = rng.choice(["f16", "bf16", "f32"])
    if op == "norm":
        per = rng.choice([1, 2, 3, 4, 6, 8, 10, 16, 24, 32])
        groups = _log(rng, 1, 64)
        c = per * groups
        n = _log(rng, 1, 16)
        side = max(1, int(math.sqrt(2 ** 25 / (n * c))))
        return {"op": "norm", "n": n, "h": _log(rng, 1, min(side, 300)), "w": _log(rng, 1, min(side, 300)), "c": c,
                "groups": groups, "act": rng.choice(["none", "relu", "silu", "gelu"]), "type": kind,
                "train": rng.random() < 0.5}
    if op == "dropout":
        return {"op": "dropout", "numel": _log(rng, 1, 2 ** 25), "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "type": kind,
                "residual": rng.random() < 0.5, "train": rng.random() < 0.5}
    b, hkv = _log(rng, 1, 8), rng.choice([1, 2, 3, 4, 8])
    if op == "serve":
        return {"op": "attend", "b": b, "lq": rng.choice([1, 1, 1, 2, 4]), "lk": _log(rng, 1, 2 ** 17 // b),
                "hq": hkv * rng.choice([1, 2, 4, 8]), "hkv": hkv, "d": rng.choice([32, 40, 64, 80, 128]), "type": kind,
                "ragged": rng.random() < 0.5, "mask": rng.random() < 0.3, "fused": rng.random() < 0.5, "train": False}
    hq = hkv * rng.choice([1, 1, 2, 4])
    lq = _log(rng, 1, 16384)
    most = max(1, 2 ** 29 // (b * hq * lq * (4 if kind == "f32" else 1)))
    return {"op": "attend", "b": b, "lq": lq, "lk": _log(rng, 1, min(8192, most)), "hq": hq, "hkv": hkv,
            "d": rng.choice([8, 16, 24, 32, 40, 48, 64, 72, 80, 96, 112, 128]), "type": kind, "ragged": rng.random() < 0.5,
            "mask": rng.random() < 0.3, "fused": rng.random() < 0.5, "train": rng.random() < 0.6}


# ---------------------------------------------------------------------------------------------------------- inputs


def _ragged(case):
    """Source lengths of a ragged batch, longest first: from the whole length down to an empty condition."""
    b, lk = case["b"], case["lk"]
    return [lk - (lk * i) // max(1, b - 1) if i < b - 1 or b < 3 else 0 for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    s = {"case": case}
    if case["op"] == "norm":
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        x = torch.randn(n, h, w, c, generator=g, device="cuda") * 1.5
        s["x"] = (x + torch.randn(c, generator=g, device="cuda")).to(t)  # channels with means of their own
        s["weight"] = 1 + 0.2 * torch.randn(c, generator=g, device="cuda")
        s["bias"] = 0.2 * torch.randn(c, generator=g, device="cuda")
        if case["train"]:
            s["dy"] = rand(n, h, w, c, scale=0.1)
    elif case["op"] == "attend":
        b, lq, lk, hq, hkv, d = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
        s["q"] = rand(b, lq, hq, d, scale=1.5)
        if case["fused"]:  # both are views of one projection of the encoder's states
            kv = rand(b, lk, 2, hkv, d)
            s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            s["k"], s["v"] = rand(b, lk, hkv, d), rand(b, lk, hkv, d)
        s["lengths"] = s["mask"] = None
        if case["ragged"]:
            lengths = _ragged(case)
            random.Random(seed).shuffle(lengths)
            s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        if case["mask"]:
            s["mask"] = torch.rand(b, lk, generator=g, device="cuda") < 0.8
            if b > 2:
                s["mask"][b - 1] = False
        if case["train"]:
            s["dout"] = rand(b, lq, hq, d, scale=0.1)
    else:
        n = case["numel"]
        s["x"] = rand(n)
        s["residual"] = rand(n) if case["residual"] else None
        s["seed"], s["offset"] = (seed * 0x9E3779B97F4A7C15) & (2 ** 63 - 1), seed % 1000
        if case["train"]:
            s["dy"] = rand(n, scale=0.1)
    return s


# --------------------------------------------------------------------------------------------------------- one pass


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "norm":
        return _norm(s, c)
    if c["op"] == "attend":
        return _attend(s, c)
    return _dropout(s, c)


def _run_own(s, c):
    import rdv_project_b200 as rdv

    if c["op"] == "norm":
        act = None if c["act"] == "none" else c["act"]
        if not c["train"]:
            return [rdv.group_norm(s["x"], c["groups"], s["weight"], s["bias"], activation=act)]
        y, stats = rdv.group_norm_forward(s["x"], c["groups"], s["weight"], s["bias"], activation=act)
        return [y, *rdv.group_norm_backward(s["dy"], s["x"], stats, c["groups"], s["weight"], s["bias"], activation=act)]
    if c["op"] == "attend":
        q, k, v, lengths, mask = s["q"], s["k"], s["v"], s["lengths"], s["mask"]
        if not c["train"]:
            return [rdv.cross_attention(q, k, v, lengths=lengths, mask=mask)]
        out, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths, mask=mask)
        return [out, *rdv.cross_attention_backward(s["dout"], q, k, v, out, lse, lengths=lengths, mask=mask)]
    y = rdv.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["residual"])
    return [y, rdv.dropout_backward(s["dy"], c["p"], s["seed"], s["offset"])] if c["train"] else [y]


# ----------------------------------------------------------------------------------------------- plain forms, 32 bits


def _act(z, act):
    """(activation, its derivative) of z."""
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return z * sig, sig * (1 + z * (1 - sig))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _norm(s, c):
    x, groups = s["x"], c["groups"]
    n, ch = x.shape[0], x.shape[-1]
    xf = x.float().reshape(n, -1, groups, ch // groups)
    w, b = s["weight"].reshape(groups, -1), s["bias"].reshape(groups, -1)
    d = xf - xf.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    xhat = d * rstd
    y, slope = _act(xhat * w + b, c["act"])
    out = [y.reshape(x.shape).to(x.dtype)]
    if c["train"]:
        dz = s["dy"].float().reshape(xf.shape) * slope
        dxhat = dz * w
        dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True) - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
        out += [dx.reshape(x.shape).to(x.dtype), (dz * xhat).sum((0, 1)).reshape(-1), dz.sum((0, 1)).reshape(-1)]
    return out


def _allowed(s, c, device):
    """[B, 1, 1, 1, Lk] truth values: which states a sample attends to, or None for all."""
    keep = None
    if s["lengths"] is not None:
        keep = torch.arange(c["lk"], device=device)[None] < s["lengths"][:, None]
    if s["mask"] is not None:
        keep = s["mask"] if keep is None else keep & s["mask"]
    return None if keep is None else keep[:, None, None, None]


def _attend(s, c):
    b, lq, lk, hq, hkv, d = (c[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
    scale = 1 / math.sqrt(d)
    kind = s["q"].dtype
    heads = (b, hkv, hq // hkv, lq, d)
    # [B, Hkv, G, Lq, D] against [B, Hkv, 1, Lk, D]
    q = s["q"].float().reshape(b, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    k = s["k"].float().permute(0, 2, 1, 3)[:, :, None]
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    keep = _allowed(s, c, q.device)
    if keep is not None:
        rows = keep.reshape(b, 1, 1, lk, 1)
        k, v = torch.where(rows, k, 0.0), torch.where(rows, v, 0.0)
    score = torch.matmul(q, k.transpose(-1, -2)) * scale
    if keep is not None:
        score = torch.where(keep, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v)
    out = [o.permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d).to(kind)]
    if c["train"]:
        do = s["dout"].float().reshape(b, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
        dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
        ds = torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)
        ds = ds * p * scale
        dq = torch.matmul(ds, k)
        dk = torch.matmul(ds.transpose(-1, -2), q).sum(2)
        out += [dq.reshape(heads).permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d).to(kind), dk.permute(0, 2, 1, 3).to(kind),
                dv.permute(0, 2, 1, 3).to(kind)]
    return out


def _times(x, const):
    """(high, low) 32-bit halves of the product of x (below 2^32, in 64 bits) and a 32-bit constant."""
    low = x * (const & 0xFFFF)
    upper = x * (const >> 16) + (low >> 16)
    return upper >> 16, ((upper << 16) | (low & 0xFFFF)) & _M32


def _words(seed, offset, numel, device):
    """Element i's random word: word i % 4 of the Philox 4x32 block with ten rounds at counter offset + i // 4 and
    key seed (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011)."""
    at = torch.arange((numel + 3) // 4, device=device, dtype=torch.int64) + offset
    c0, c1 = at & _M32, at >> 32
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        h0, l0 = _times(c0, 0xD2511F53)
        h1, l1 = _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:numel]


def _dropout(s, c):
    x = s["x"]
    keep = _words(s["seed"], s["offset"], x.numel(), x.device) >= int(round(c["p"] * 2 ** 32))
    scale = 1 / (1 - c["p"])
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return [y.to(x.dtype), torch.where(keep, s["dy"].float() * scale, 0.0).to(x.dtype)] if c["train"] else [y.to(x.dtype)]


# ------------------------------------------------------------------------------------------- definitions, 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "attend": _exact_attend, "dropout": _exact_dropout}[case["op"]](s, case)


def _exact_norm(s, c):
    """One sample at a time: y = act(w (x - mu) / sigma + b), and the gradients by the chain rule through mu and sigma."""
    ys, dxs = [], []
    dw = torch.zeros(c["c"], dtype=torch.float64, device="cuda")
    db = torch.zeros_like(dw)
    per = c["c"] // c["groups"]

    def spread(v):  # a group's value to its channels
        return v.repeat_interleave(per)[None]

    w, b = s["weight"].double(), s["bias"].double()
    for i in range(c["n"]):
        x = s["x"][i].reshape(-1, c["c"]).double()
        m = x.shape[0] * per
        mu = x.sum(0).reshape(-1, per).sum(1) / m
        cen = x - spread(mu)
        sigma = ((cen ** 2).sum(0).reshape(-1, per).sum(1) / m + 1e-5).sqrt()
        hat = cen / spread(sigma)
        z = hat * w + b
        if c["act"] == "silu":
            y, slope = z * torch.sigmoid(z), torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
        elif c["act"] == "relu":
            y, slope = z.clamp(min=0), (z > 0).double()
        elif c["act"] == "gelu":
            cdf = torch.special.ndtr(z)
            y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        else:
            y, slope = z, torch.ones_like(z)
        ys.append(y.reshape(s["x"].shape[1:]))
        if c["train"]:
            dz = s["dy"][i].reshape(-1, c["c"]).double() * slope
            db += dz.sum(0)
            dw += (dz * hat).sum(0)
            dhat = dz * w
            dsum = dhat.sum(0).reshape(-1, per).sum(1) / m
            dproj = (dhat * hat).sum(0).reshape(-1, per).sum(1) / m
            dxs.append(((dhat - spread(dsum) - hat * spread(dproj)) / spread(sigma)).reshape(s["x"].shape[1:]))
    return [torch.stack(ys), torch.stack(dxs), dw, db] if c["train"] else [torch.stack(ys)]


def _exact_attend(s, c):
    """One head of one sample at a time, over the states that it attends to alone."""
    b, lq, lk, hq, hkv, d = (c[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
    if b * hq * lq * lk * d > 2 ** 39:
        return None
    out = torch.zeros(b, lq, hq, d, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk = torch.zeros(b, lk, hkv, d, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    for i in range(b):
        at = torch.ones(lk, dtype=torch.bool, device="cuda")
        if s["lengths"] is not None:
            at[int(s["lengths"][i]):] = False
        if s["mask"] is not None:
            at &= s["mask"][i]
        at = at.nonzero()[:, 0]
        if not len(at):
            continue
        for h in range(hq):
            kv = h // (hq // hkv)
            q, k, v = s["q"][i, :, h].double(), s["k"][i, at, kv].double(), s["v"][i, at, kv].double()
            p = torch.softmax(q @ k.T / math.sqrt(d), 1)
            out[i, :, h] = p @ v
            if c["train"]:
                do = s["dout"][i, :, h].double()
                dv[i, at, kv] += p.T @ do
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dq[i, :, h] = ds @ k
                dk[i, at, kv] += ds.T @ q
    return [out, dq, dk, dv] if c["train"] else [out]


def _exact_dropout(s, c):
    """The generator on the host in Python's whole numbers would take minutes: its words come from unsigned 64-bit
    arithmetic of the host instead, whose products wrap, so a high half is taken from the four partial products."""
    import numpy as np

    n, dev = c["numel"], s["x"].device
    at = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(s["offset"])
    m, sh = np.uint64(_M32), np.uint64(32)
    ctr = [at & m, at >> sh, np.zeros_like(at), np.zeros_like(at)]
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
    for _ in range(10):
        a, e = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)  # 32 x 32 bits: no product wraps
        ctr = [(e >> sh) ^ ctr[1] ^ np.uint64(key[0]), e & m, (a >> sh) ^ ctr[3] ^ np.uint64(key[1]), a & m]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    word = torch.from_numpy(np.stack(ctr, 1).reshape(-1)[:n].astype(np.int64)).to(dev)
    factor = (word >= round(c["p"] * 2 ** 32)).double() / (1 - c["p"])
    y = s["x"].double() * factor
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return [y, s["dy"].double() * factor] if c["train"] else [y]


# ------------------------------------------------------------------------------------------------------------- work


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        n = case["n"] * case["h"] * case["w"] * case["c"]
        params = 4 * case["c"]
        # forward: x in, y out; training reads x and dy once more and writes dx
        return {"bytes": n * size * (5 if case["train"] else 2) + params * (6 if case["train"] else 2),
                "flops": n * (30 if case["train"] else 10)}
    if case["op"] == "dropout":
        n = case["numel"]
        return {"bytes": n * size * (2 + case["residual"] + (2 if case["train"] else 0)),
                "flops": n * (4 if case["train"] else 2)}
    b, lq, lk, hq, hkv, d = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
    seen = sum(_ragged(case)) if case["ragged"] else b * lk  # states attended to, over the batch
    if case["mask"] and b > 2:
        seen = seen * (b - 1) // b
    rows, states = b * lq * hq * d * size, seen * hkv * d * size
    byts = 2 * rows + 2 * states
    if case["train"]:  # out, dout, q, k and v in; dq, dk and dv out
        byts += 4 * rows + 2 * states + 2 * b * lk * hkv * d * size
    return {"bytes": byts, "flops": (14 if case["train"] else 4) * lq * hq * d * seen}
