"""The attention operators of a served decoder, as they are timed: plain forms and the framework's calls.

Five operators that follow one another in a decoder layer: the projection split into heads with the
query and key norms and the rotary positions in the same pass; attention with a sliding window and
sinks over shared key heads; the block tables and slots of a paged cache; the write of new keys and
values into its pages; and the attention of one new token over the pages.

``run`` computes the plain form in elementary torch operations, or, where ``own`` is true, makes the
calls that a program makes of ``edifice_amd.fused_scan``.  ``exact`` restates each in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False  # plain forms (False) or the framework's calls (True)

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one decoder layer's training step at the hybrid decoder's size (8 heads of 128), two queries a key head
        {"name": "rotary_train", "kind": "rotary", "B": 8, "T": 2048, "Hq": 8, "Hkv": 4, "d": 128, "rot": 128,
         "interleaved": False, "norm": True, "scaling": "none", "start": 0, "dtype": "bf16", "train": True},
        # a float32 model (the default type of a built one), half of each head rotated in pairs, positions
        # scaled for a longer context, ragged length
        {"name": "rotary_partial_f32", "kind": "rotary", "B": 2, "T": 1000, "Hq": 12, "Hkv": 4, "d": 96, "rot": 48,
         "interleaved": True, "norm": True, "scaling": "parts", "start": 0, "dtype": "f32", "train": True},
        # one decode step of 64 requests far into their texts
        {"name": "rotary_decode", "kind": "rotary", "B": 64, "T": 1, "Hq": 32, "Hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "norm": True, "scaling": "linear", "start": 100000, "dtype": "bf16", "train": False},
        # training step of causal attention at the 32-head benchmark's size, four queries a key head
        {"name": "window_train", "kind": "window", "B": 4, "T": 4096, "Hq": 32, "Hkv": 8, "d": 128, "window": 1024,
         "sinks": 4, "dtype": "bf16", "train": True},
        # a long prompt read before answering
        {"name": "window_prompt", "kind": "window", "B": 1, "T": 16384, "Hq": 16, "Hkv": 2, "d": 64, "window": 2048,
         "sinks": 16, "dtype": "bf16", "train": False},
        # a small float32 model's training step, ragged length and window
        {"name": "window_f32", "kind": "window", "B": 2, "T": 1000, "Hq": 8, "Hkv": 4, "d": 64, "window": 300,
         "sinks": 1, "dtype": "f32", "train": True},
        # one decode step of a ragged batch of conversations, one of its places empty
        {"name": "paged_batch", "kind": "paged", "B": 64, "longest": 4096, "Hq": 32, "Hkv": 8, "d": 128, "block": 16,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # one decode step of a few long documents: the split over the cache's length counts
        {"name": "paged_long", "kind": "paged", "B": 3, "longest": 131000, "Hq": 16, "Hkv": 2, "d": 128, "block": 64,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # the cache's bookkeeping before a batch of prompts
        {"name": "extend_prompt", "kind": "extend", "R": 64, "tokens": 2048, "block": 16, "longest": 2048, "fresh": True},
        # and before each decode step of many requests
        {"name": "extend_decode", "kind": "extend", "R": 500, "tokens": 1, "block": 16, "longest": 8192, "fresh": False},
        # keys and values of a batch of prompts into their pages
        {"name": "write_prompt", "kind": "write", "B": 8, "T": 2048, "Hkv": 8, "d": 128, "block": 16, "dtype": "bf16"},
        # and those of a decode step
        {"name": "write_decode", "kind": "write", "B": 64, "T": 1, "Hkv": 8, "d": 128, "block": 16, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "window", "window", "window", "paged", "paged", "extend", "write"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    hkv = rng.choice([1, 2, 4, 8])
    if kind == "rotary":
        d = rng.choice([32, 64, 80, 96, 128, 128, 256])
        return {"kind": kind, "B": rng.randint(1, 8), "T": _log(rng, 1, 2048), "Hq": hkv * rng.choice([1, 2, 3, 4]),
                "Hkv": hkv, "d": d, "rot": d // rng.choice([1, 1, 2]), "interleaved": rng.random() < 0.5,
                "norm": rng.random() < 0.7, "scaling": rng.choice(["none", "linear", "parts"]),
                "start": rng.choice([0, 0, rng.randint(1, 1000000)]), "dtype": dtype, "train": rng.random() < 0.6}
    if kind == "window":
        hq = hkv * rng.choice([1, 2, 4])
        T = _log(rng, 2, 8192)
        B = rng.randint(1, max(1, min(8, (1 << 30) // (hq * T * T))))
        return {"kind": kind, "B": B, "T": T, "Hq": hq, "Hkv": hkv,
                "d": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), "window": _log(rng, 2, 4096),
                "sinks": rng.choice([0, 1, 4, 16, 100]), "dtype": dtype, "train": rng.random() < 0.6}
    if kind == "paged":
        longest = _log(rng, 1, 65536)
        return {"kind": kind, "B": rng.randint(1, max(1, min(128, 262144 // longest))), "longest": longest,
                "Hq": hkv * rng.choice([1, 2, 4, 7, 8]), "Hkv": hkv, "d": rng.choice([64, 80, 96, 128, 128, 256]),
                "block": rng.choice([16, 16, 32, 64, 128]), "window": rng.choice([0, 0, _log(rng, 2, 8192)]),
                "sinks": rng.choice([0, 4, 20]), "dtype": dtype}
    if kind == "extend":
        tokens = rng.choice([1, _log(rng, 1, 4096)])
        return {"kind": kind, "R": _log(rng, 1, 1024), "tokens": tokens, "block": rng.choice([16, 32, 64, 128]),
                "longest": max(tokens, _log(rng, 64, 16384)), "fresh": rng.random() < 0.5}
    return {"kind": kind, "B": rng.randint(1, 16), "T": _log(rng, 1, 2048), "Hkv": hkv,
            "d": rng.choice([64, 80, 96, 128, 256]), "block": rng.choice([16, 32, 64, 128]), "dtype": dtype}


def _frequencies(case):
    """Angle per position of each rotated pair, float64 [rot / 2], and the amplitude of the rotation."""
    rot = case["rot"]
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "parts":  # slow turns (under 1 in 4096 positions) stretched by 8, fast ones (over 32) kept
        keep = ((4096.0 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        return f / 8.0 * (1.0 - keep) + f * keep, 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _pages(g, lengths, longest, block, spare):
    """A table [B, longest / block] of distinct pages in random order, -1 behind each length, and how many pages."""
    B, width = len(lengths), max(1, -(-longest // block))
    need = (lengths + block - 1) // block
    held = torch.arange(width, device=DEV)[None, :] < need[:, None]
    total = B * width + spare
    ids = torch.randperm(total, device=DEV, generator=g)[:B * width].view(B, width)
    return torch.where(held, ids, -1).to(torch.int32), total


def _lengths(g, B, longest):
    """Ragged lengths from 1 to the longest, which is there; in a batch of eight or more one place is empty."""
    n = torch.randint(1, longest + 1, (B,), device=DEV, generator=g)
    n[-1] = longest
    if B >= 8:
        n[B // 2] = 0
    return n.to(torch.int32)


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case.get("dtype", "bf16")]

    def n(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if kind == "rotary":
        B, T, Hq, Hkv, d = (case[c] for c in ("B", "T", "Hq", "Hkv", "d"))
        s = {"x": n(B, T, (Hq + 2 * Hkv) * d).to(dt)}
        s["freq"], s["amplitude"] = _frequencies(case)
        s["pos"] = (torch.arange(T, device=DEV)[None, :] + case["start"]
                    + torch.randint(0, 1000, (B, 1), device=DEV, generator=g)).to(torch.int32)
        s["wq"], s["wk"] = ((1 + 0.2 * n(d)).to(dt) if case["norm"] else None for _ in range(2))
        if case["train"]:
            s["grads"] = tuple(n(B, h, T, d).to(dt) for h in (Hq, Hkv, Hkv))
        return s
    if kind == "window":
        B, T, Hq, Hkv, d = (case[c] for c in ("B", "T", "Hq", "Hkv", "d"))
        s = {"q": n(B, Hq, T, d).to(dt), "k": n(B, Hkv, T, d).to(dt), "v": n(B, Hkv, T, d).to(dt)}
        if case["train"]:
            s["do"] = n(B, Hq, T, d).to(dt)
        return s
    if kind == "paged":
        B, Hkv, d, block = (case[c] for c in ("B", "Hkv", "d", "block"))
        lengths = _lengths(g, B, case["longest"])
        table, pages = _pages(g, lengths, case["longest"], block, 5)
        return {"q": n(B, case["Hq"], d).to(dt), "kc": n(pages, Hkv, block, d).to(dt),
                "vc": n(pages, Hkv, block, d).to(dt), "table": table, "lengths": lengths}
    if kind == "extend":
        R, block, tokens, longest = (case[c] for c in ("R", "block", "tokens", "longest"))
        new = torch.randint(1, longest + 1, (R,), device=DEV, generator=g).to(torch.int32)
        if case["fresh"]:
            old = torch.zeros_like(new)
            new = new.clamp(max=tokens)
        else:
            old = (new - tokens).clamp(min=0)
        table, pages = _pages(g, old, longest, block, R * (tokens // block + 2))
        used = torch.zeros(pages, dtype=torch.bool, device=DEV)
        used[table[table >= 0].long()] = True
        free = torch.randperm(pages, device=DEV, generator=g)
        return {"table": table, "old": old, "new": new, "free": free[~used[free]].to(torch.int32)}
    B, T, Hkv, d, block = (case[c] for c in ("B", "T", "Hkv", "d", "block"))
    lengths = torch.randint(max(1, T // 2), T + 1, (B,), device=DEV, generator=g)
    table, pages = _pages(g, lengths, T, block, 5)
    t = torch.arange(T, device=DEV)
    slots = table[:, t // block].long() * block + t % block
    slots = torch.where(t[None, :] < lengths[:, None], slots, -1).to(torch.int32)
    return {"k": n(B, Hkv, T, d).to(dt), "v": n(B, Hkv, T, d).to(dt), "slots": slots,
            "kc": torch.zeros(pages, Hkv, block, d, device=DEV, dtype=dt),
            "vc": torch.zeros(pages, Hkv, block, d, device=DEV, dtype=dt)}


def prepare(case, seed):
    s = _inputs(case, seed)
    if case.get("train"):
        for name in ("x", "wq", "wk", "q", "k", "v"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return dict(s, case=case)


def run(state):
    with torch.set_grad_enabled(own and bool(state["case"].get("train"))):
        return {"rotary": _rotary, "window": _window, "paged": _paged, "extend": _extend,
                "write": _write}[state["case"]["kind"]](state)


# ---- head split, norms and rotation --------------------------------------------------

def _rotary(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        out = fs.split_heads_rotary(s["x"], case["Hq"], case["Hkv"], s["freq"], s["pos"], s["wq"], s["wk"], eps=EPS,
                                    interleaved=case["interleaved"], amplitude=s["amplitude"])
        if not case["train"]:
            return list(out)
        leaves = [t for t in (s["x"], s["wq"], s["wk"]) if t is not None]
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, s["grads"]))
    Hq, Hkv, d, dt = case["Hq"], case["Hkv"], case["d"], s["x"].dtype
    heads = s["x"].float().unflatten(-1, (Hq + 2 * Hkv, d)).transpose(1, 2)
    xq, xk, xv = heads.split([Hq, Hkv, Hkv], 1)
    angle = (s["pos"].double()[:, None, :, None] * s["freq"]).remainder(2 * math.pi)
    cos, sin = ((f(angle) * s["amplitude"]).float() for f in (torch.cos, torch.sin))
    q, keep_q = _norm_turn(xq, s["wq"], cos, sin, case)
    k, keep_k = _norm_turn(xk, s["wk"], cos, sin, case)
    out = [q.to(dt), k.to(dt), xv.contiguous().to(dt)]
    if not case["train"]:
        return out
    gq, gk, gv = (g.float() for g in s["grads"])
    dq, dwq = _norm_turn_grad(gq, s["wq"], cos, sin, keep_q, case)
    dk, dwk = _norm_turn_grad(gk, s["wk"], cos, sin, keep_k, case)
    out.append(torch.cat([dq, dk, gv], 1).transpose(1, 2).flatten(2).to(dt))
    return out + ([dwq.to(dt), dwk.to(dt)] if case["norm"] else [])


def _turn(n, cos, sin, case):
    rot = case["rot"]
    if case["interleaved"]:
        a, b = n[..., 0:rot:2], n[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = n[..., :rot // 2], n[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, n[..., rot:]], -1)


def _norm_turn(x, w, cos, sin, case):
    if w is None:
        return _turn(x, cos, sin, case), None
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = x * r
    return _turn(xh * w.float(), cos, sin, case), (r, xh)


def _norm_turn_grad(g, w, cos, sin, keep, case):
    g = _turn(g, cos, -sin, case)
    if w is None:
        return g, None
    r, xh = keep
    gw = g * w.float()
    return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (g * xh).sum((0, 1, 2))


# ---- attention with a window and sinks -----------------------------------------------

def _window(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        o = fs.window_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"])
        if not case["train"]:
            return [o]
        return [o.detach()] + list(torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))
    B, T, Hq, Hkv, d = (case[c] for c in ("B", "T", "Hq", "Hkv", "d"))
    dt, scale = s["q"].dtype, d ** -0.5
    rows = Hq // Hkv * T  # the query heads of one key head, one after the other
    q, k, v = s["q"].float().reshape(B, Hkv, rows, d), s["k"].float(), s["v"].float()
    i = torch.arange(T, device=DEV)
    back = i[:, None] - i[None, :]
    hidden = (back < 0) | ((back >= case["window"]) & (i[None, :] >= case["sinks"]))
    p = (q @ k.transpose(-1, -2)).mul_(scale).view(B, Hkv, -1, T, T).masked_fill_(hidden, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(B, Hkv, rows, T)
    out = [(p @ v).view(B, Hq, T, d).to(dt)]
    if not case["train"]:
        return out
    do = s["do"].float().reshape(B, Hkv, rows, d)
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    return out + [dq.view(B, Hq, T, d).to(dt), dk.to(dt), dv.to(dt)]


# ---- attention of one token over pages -----------------------------------------------

def _paged(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        return [fs.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lengths"], window=case["window"],
                                   sinks=case["sinks"])]
    B, Hq, Hkv, d = (case[c] for c in ("B", "Hq", "Hkv", "d"))
    at = s["table"].clamp(min=0).long()
    k, v = (c[at].transpose(1, 2).reshape(B, Hkv, -1, d).float() for c in (s["kc"], s["vc"]))
    q = s["q"].float().view(B, Hkv, Hq // Hkv, d)
    j = torch.arange(k.shape[2], device=DEV)
    n = s["lengths"].long()[:, None]
    seen = j[None, :] < n
    if case["window"]:
        seen = seen & ((j[None, :] >= n - case["window"]) | (j[None, :] < case["sinks"]))
    p = (q @ k.transpose(-1, -2) * d ** -0.5).masked_fill(~seen[:, None, None, :], -math.inf)
    p = (p - p.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)  # an empty place answers with zeros
    return [(p @ v).view(B, Hq, d).to(s["q"].dtype)]


# ---- block tables and slots ----------------------------------------------------------

def _extend(s):
    case = s["case"]
    block, tokens = case["block"], case["tokens"]
    if own:
        from edifice_amd import fused_scan as fs
        slots, positions, used = fs.paged_extend(s["table"], s["old"], s["new"], s["free"], block, tokens)
        return [s["table"], slots, positions, used]
    old, new, table = s["old"].long(), s["new"].long(), s["table"]
    width = table.shape[1]
    have = ((old + block - 1) // block).clamp(max=width)
    want = torch.maximum(((new + block - 1) // block).clamp(max=width), have)
    count = want - have
    first = count.cumsum(0) - count
    c = torch.arange(width, device=DEV)[None, :]
    fresh = (c >= have[:, None]) & (c < want[:, None])
    draw = first[:, None] + c - have[:, None]
    got = s["free"][draw.clamp(0, len(s["free"]) - 1)]
    table = torch.where(fresh, torch.where(draw < len(s["free"]), got, -1), table)
    p = old[:, None] + torch.arange(tokens, device=DEV)[None, :]
    there = p < new[:, None]
    page = table.gather(1, (p // block).clamp(max=width - 1)).long()
    held = there & (p // block < width) & (page >= 0)
    slots = torch.where(held, page * block + p % block, -1).to(torch.int32)
    return [table, slots, torch.where(there, p, -1).to(torch.int32), count.sum(0, keepdim=True).to(torch.int32)]


# ---- new keys and values into their pages --------------------------------------------

def _write(s):
    if own:
        from edifice_amd import fused_scan as fs
        fs.paged_cache_write(s["k"], s["v"], s["slots"], s["kc"], s["vc"])
        return [s["kc"], s["vc"]]
    b, t = torch.nonzero(s["slots"] >= 0, as_tuple=True)
    slot, block = s["slots"][b, t].long(), s["case"]["block"]
    s["kc"][slot // block, :, slot % block] = s["k"][b, :, t]
    s["vc"][slot // block, :, slot % block] = s["v"][b, :, t]
    return [s["kc"], s["vc"]]


def work(case):
    kind = case["kind"]
    size = 4 if case.get("dtype") == "f32" else 2
    if kind == "rotary":
        n = case["B"] * case["T"] * (case["Hq"] + 2 * case["Hkv"]) * case["d"]
        return {"bytes": (5 if case["train"] else 2) * n * size, "flops": (18 if case["train"] else 7) * n}
    if kind == "window":
        T, W, S = case["T"], min(case["window"], case["T"]), case["sinks"]
        pairs = W * (W + 1) // 2 + (T - W) * W  # inside the window
        far = T - W  # queries past the first window see sinks outside it, at most S each
        pairs += far * S - (min(S, far) * (min(S, far) - 1) // 2 + max(0, S - far) * far)
        qo, kv = (case["B"] * case[h] * T * case["d"] * size for h in ("Hq", "Hkv"))
        flops = 4 * case["d"] * pairs * case["B"] * case["Hq"]
        if case["train"]:
            return {"bytes": 5 * qo + 6 * kv, "flops": 3.5 * flops}
        return {"bytes": 2 * qo + 2 * kv, "flops": flops}
    if kind == "paged":  # ragged lengths, half the longest on average
        n = (case["B"] - 1) * (case["longest"] + 1) / 2 * (1 - (case["B"] >= 8) / case["B"]) + case["longest"]
        if case["window"]:
            n = min(n, case["B"] * (case["window"] + case["sinks"]))
        keys = n * case["Hkv"] * case["d"]
        return {"bytes": 2 * keys * size + 2 * case["B"] * case["Hq"] * case["d"] * size,
                "flops": 4 * n * case["Hq"] * case["d"]}
    if kind == "extend":
        return {"bytes": 4 * (case["R"] * (2 + 2 * case["tokens"] + 2 * (-(-case["tokens"] // case["block"])))), "flops": 0}
    n = case["B"] * case["T"] * case["Hkv"] * case["d"]
    return {"bytes": 2 * 2 * 0.75 * n * size, "flops": 0}  # prompts fill three quarters of their batch on average


def exact(case, seed):
    kind = case["kind"]
    if kind in ("extend", "write"):  # whole numbers, and values that are only moved
        return None
    s = _inputs(case, seed)
    if kind == "rotary":
        Hq, Hkv, d, rot = case["Hq"], case["Hkv"], case["d"], case["rot"]
        x = s["x"].double()
        B, T = x.shape[:2]
        leaves = [x] + [w.double() for w in (s["wq"], s["wk"]) if w is not None]
        for t in leaves:
            t.requires_grad_(case["train"])
        unit = torch.polar(torch.full((1,), s["amplitude"], device=DEV, dtype=torch.float64),
                           s["pos"].double()[:, :, None] * s["freq"])[:, :, None, :]
        with torch.enable_grad():
            heads = x.view(B, T, Hq + 2 * Hkv, d)
            out = []
            for at, h, w in ((0, Hq, 1), (Hq, Hkv, 2)):
                u = heads[:, :, at:at + h]
                if case["norm"]:
                    u = u / torch.sqrt((u * u).sum(-1, keepdim=True) / d + EPS) * leaves[w]
                pair = u[..., :rot].unflatten(-1, (rot // 2, 2) if case["interleaved"] else (2, rot // 2))
                pair = pair if case["interleaved"] else pair.transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
                z = z if case["interleaved"] else z.transpose(-1, -2)
                out.append(torch.cat([z.reshape(B, T, h, rot), u[..., rot:]], -1).transpose(1, 2))
            out.append(heads[:, :, Hq + Hkv:].transpose(1, 2))
            if not case["train"]:
                return out
            grads = torch.autograd.grad(out, leaves, [g.double() for g in s["grads"]])
        return [t.detach() for t in out] + list(grads)
    if kind == "window":
        B, T, Hq, Hkv, d = (case[c] for c in ("B", "T", "Hq", "Hkv", "d"))
        W, S, G = case["window"], case["sinks"], Hq // Hkv
        if B * Hq * T * min(T, W + 512) > 3e9:
            return None
        o = torch.empty(B, Hq, T, d, dtype=torch.float64, device=DEV)
        if case["train"]:
            dq, dk, dv = torch.empty_like(o), *(torch.zeros(B, Hkv, T, d, dtype=torch.float64, device=DEV) for _ in range(2))
        for b in range(B):
            for h in range(Hkv):
                kd, vd = s["k"][b, h].double(), s["v"][b, h].double()
                for lo in range(0, T, 512):  # a band of queries against the keys that any of them sees
                    hi = min(T, lo + 512)
                    first = max(0, lo - W + 1)
                    js = torch.cat([torch.arange(min(S, first), device=DEV), torch.arange(first, hi, device=DEV)])
                    i = torch.arange(lo, hi, device=DEV)[:, None]
                    see = (js <= i) & ((js > i - W) | (js < S))
                    ks, vs = kd[js], vd[js]
                    qs = s["q"][b, h * G:(h + 1) * G, lo:hi].double()
                    a = torch.where(see, torch.matmul(qs, ks.t()) / math.sqrt(d), -torch.inf)
                    p = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
                    ob = torch.matmul(p, vs)
                    o[b, h * G:(h + 1) * G, lo:hi] = ob
                    if case["train"]:
                        g = s["do"][b, h * G:(h + 1) * G, lo:hi].double()
                        e = p * (torch.matmul(g, vs.t()) - (g * ob).sum(-1, keepdim=True)) / math.sqrt(d)
                        dq[b, h * G:(h + 1) * G, lo:hi] = torch.matmul(e, ks)
                        dk[b, h].index_add_(0, js, torch.matmul(e.flatten(0, 1).t(), qs.flatten(0, 1)))
                        dv[b, h].index_add_(0, js, torch.matmul(p.flatten(0, 1).t(), g.flatten(0, 1)))
        return [o, dq, dk, dv] if case["train"] else [o]
    B, Hq, Hkv, d = (case[c] for c in ("B", "Hq", "Hkv", "d"))
    o = torch.zeros(B, Hq, d, dtype=torch.float64, device=DEV)
    lengths = s["lengths"].tolist()
    for b in range(B):
        if lengths[b]:
            j = torch.arange(lengths[b], device=DEV)
            if case["window"]:
                j = j[(j >= lengths[b] - case["window"]) | (j < case["sinks"])]
            page = s["table"][b].long()[j // case["block"]]
            k, v = (c[page, :, j % case["block"]].transpose(0, 1).double() for c in (s["kc"], s["vc"]))
            q = s["q"][b].double().view(Hkv, Hq // Hkv, d)
            a = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(d)
            o[b] = torch.matmul(torch.softmax(a, -1), v).view(Hq, d)
    return [o]
