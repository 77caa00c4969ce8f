"""Packed texts and an 8-bit cache, as they are timed: plain forms and the framework's calls.

Four operators of a decoder whose texts differ in length: causal attention over texts laid end to end, whose queries
may be the last ones of longer keys; the write of keys and values into pages of 8 bits with a scale for each page and
head; reading such pages back; and the attention of one new token over them.

``run`` computes the plain form in elementary torch operations, or, where ``own`` is true, makes the calls that a
program makes of ``edifice_amd.fused_scan``.  ``exact`` restates each in 64 bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False  # plain forms (False) or the framework's calls (True)

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LEAST = 2.0 ** -100  # the smallest scale of a page that holds anything but zeros


def listed():
    return [
        # a training step on twelve documents laid end to end, at the 32-head benchmark's width, four queries a key head
        {"name": "packed_train", "kind": "packed", "texts": 12, "longest": 4096, "fresh": 0, "Hq": 32, "Hkv": 8, "d": 128,
         "window": 0, "sinks": 0, "dtype": "bf16", "train": True},
        # three prompts read before answering, one of them long, with narrow heads and a window
        {"name": "packed_prompt", "kind": "packed", "texts": 3, "longest": 10000, "fresh": 0, "Hq": 16, "Hkv": 2, "d": 64,
         "window": 4000, "sinks": 16, "dtype": "bf16", "train": False},
        # a small float32 model's training step on five short texts
        {"name": "packed_f32", "kind": "packed", "texts": 5, "longest": 700, "fresh": 0, "Hq": 8, "Hkv": 4, "d": 64,
         "window": 0, "sinks": 0, "dtype": "f32", "train": True},
        # eight conversations go on: up to 64 new tokens each over what their places hold
        {"name": "packed_continue", "kind": "packed", "texts": 8, "longest": 8192, "fresh": 64, "Hq": 32, "Hkv": 8,
         "d": 128, "window": 0, "sinks": 0, "dtype": "bf16", "train": False},
        # keys and values of a batch of prompts into pages of 8-bit numbers
        {"name": "write_prompt", "kind": "write", "B": 8, "T": 2048, "held": 0, "Hkv": 8, "d": 128, "block": 16,
         "codes": "int8", "dtype": "bf16"},
        # those of one decode step of 64 requests, into pages that hold some tokens already
        {"name": "write_decode", "kind": "write", "B": 64, "T": 1, "held": 20, "Hkv": 8, "d": 128, "block": 16,
         "codes": "e4m3", "dtype": "bf16"},
        # what eight places hold, read back for the prompts that go on from there
        {"name": "read_places", "kind": "read", "B": 8, "longest": 8192, "Hkv": 8, "d": 128, "block": 16,
         "codes": "e4m3", "dtype": "bf16"},
        # a small float32 model's two places
        {"name": "read_f32", "kind": "read", "B": 2, "longest": 600, "Hkv": 4, "d": 64, "block": 32,
         "codes": "int8", "dtype": "f32"},
        # one decode step of a ragged batch of conversations, one of its places empty
        {"name": "attend_batch", "kind": "attend", "B": 64, "longest": 4096, "Hq": 32, "Hkv": 8, "d": 128, "block": 16,
         "window": 0, "sinks": 0, "codes": "int8", "dtype": "bf16"},
        # one decode step of a few long documents: the split over the cache's length counts
        {"name": "attend_long", "kind": "attend", "B": 3, "longest": 131000, "Hq": 16, "Hkv": 2, "d": 128, "block": 64,
         "window": 0, "sinks": 0, "codes": "e4m3", "dtype": "bf16"},
        # one short conversation of a float32 model
        {"name": "attend_one", "kind": "attend", "B": 1, "longest": 600, "Hq": 8, "Hkv": 4, "d": 64, "block": 16,
         "window": 0, "sinks": 0, "codes": "int8", "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["packed", "packed", "packed", "write", "read", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    codes = rng.choice(["int8", "e4m3"])
    hkv = rng.choice([1, 2, 4, 8])
    if kind == "packed":
        hq = hkv * rng.choice([1, 2, 4])
        longest = _log(rng, 2, 8192)
        return {"kind": kind, "texts": rng.randint(1, max(1, min(64, (1 << 32) // (hq * longest * longest)))),
                "longest": longest, "fresh": rng.choice([0, 0, _log(rng, 1, 512)]), "Hq": hq, "Hkv": hkv,
                "d": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), "window": rng.choice([0, 0, _log(rng, 2, 4096)]),
                "sinks": rng.choice([0, 4, 20]), "dtype": dtype, "train": rng.random() < 0.6}
    d, block = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([16, 16, 32, 64, 128])
    if kind == "write":
        return {"kind": kind, "B": rng.randint(1, 16), "T": _log(rng, 1, 2048), "held": rng.choice([0, _log(rng, 1, 200)]),
                "Hkv": hkv, "d": d, "block": block, "codes": codes, "dtype": dtype}
    longest = _log(rng, 1, 65536 if kind == "attend" else 8192)
    if kind == "read":
        return {"kind": kind, "B": rng.randint(1, max(1, min(64, 65536 // longest))), "longest": longest, "Hkv": hkv,
                "d": d, "block": block, "codes": codes, "dtype": dtype}
    return {"kind": kind, "B": rng.randint(1, max(1, min(128, 262144 // longest))), "longest": longest,
            "Hq": hkv * rng.choice([1, 2, 4, 7, 8]), "Hkv": hkv, "d": d, "block": block,
            "window": rng.choice([0, 0, _log(rng, 2, 8192)]), "sinks": rng.choice([0, 4, 20]), "codes": codes,
            "dtype": dtype}


def _ragged(count, longest, empty):
    """Lengths from 1 to the longest, which is the last one, the same for every seed; of four or more, one text holds one
    token, and where ``empty`` allows it another none."""
    rng = random.Random(1000003 * count + longest)
    n = [rng.randint(1, longest) for _ in range(count)]
    if count >= 4:
        n[1] = 1
        if empty:
            n[2] = 0
    n[-1] = longest
    return n


def _texts(case):
    """(query lengths, key lengths) of a packed case: the same where every text is read whole, else the keys of what is
    held already with up to ``fresh`` new tokens as its end."""
    keys = _ragged(case["texts"], case["longest"], True)
    if not case["fresh"]:
        return keys, keys
    rng = random.Random(7 * case["texts"] + case["fresh"])
    return [min(m, rng.randint(1, case["fresh"])) for m in keys], keys


def _offsets(lengths):
    return torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device=DEV)


# ---- pages of 8-bit numbers ----------------------------------------------------------

def _pow2(k):
    """2^k, exactly, for whole k from -126 to 127."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _least_scale(amax, codes):
    """The smallest scale that a page and head with that largest size needs: a 127th of it, or the power of two from a
    448th of it on; NaN where a value is not finite."""
    if codes == "int8":
        n = amax * torch.tensor(1 / 127, dtype=torch.float32, device=DEV)
    else:
        m, e = torch.frexp(amax)  # amax = m 2^e, m from a half to one; 448 = 7/8 2^9
        n = _pow2((e - 9 + (m > 0.875).to(torch.int32)).clamp(min=-100))
    n = torch.where(amax > 0, n.clamp(min=LEAST), torch.zeros_like(n))
    return torch.where(torch.isfinite(amax), n, torch.nan)


def _to_codes(x, codes):
    """Values in units of their scale to 8 bits, ties to even."""
    return x.round().clamp(-127, 127).to(torch.int8) if codes == "int8" else x.to(torch.float8_e4m3fn)


def _inverse(scale):
    """One over each scale, zero where the scale is none."""
    return torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))


def _filled(g, pages, Hkv, block, d, codes):
    """A cache of random keys or values, some channels of them larger than the others, as codes and scales."""
    x = torch.randn(pages, Hkv, block, d, device=DEV, generator=g)
    x = x * torch.exp(0.7 * torch.randn(Hkv, 1, d, device=DEV, generator=g))
    s = _least_scale(x.abs().amax((2, 3)), codes)
    return _to_codes(x * _inverse(s)[:, :, None, None], codes), s


def _pages(g, lengths, block, spare):
    """A table [B, widest] of distinct pages in random order, -1 behind each length, and how many pages there are."""
    need = torch.tensor([-(-n // block) for n in lengths], device=DEV)
    width = max(1, -(-max(lengths) // block))
    total = len(lengths) * width + spare
    ids = torch.randperm(total, device=DEV, generator=g)[:len(lengths) * width].view(-1, width)
    return torch.where(torch.arange(width, device=DEV)[None, :] < need[:, None], ids, -1).to(torch.int32), total


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]

    def n(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if kind == "packed":
        nq, nk = _texts(case)
        Hq, Hkv, d, N, M = case["Hq"], case["Hkv"], case["d"], sum(nq), sum(nk)
        s = {"q": n(Hq, N, d).to(dt), "k": n(Hkv, M, d).to(dt), "v": n(Hkv, M, d).to(dt), "nq": nq, "nk": nk,
             "offsets": _offsets(nq), "key_offsets": _offsets(nk)}
        if case["train"]:
            s["do"] = n(Hq, N, d).to(dt)
        return s
    Hkv, d, block, codes = (case[c] for c in ("Hkv", "d", "block", "codes"))
    if kind == "write":
        B, T = case["B"], case["T"]
        held = torch.randint(0, case["held"] + 1, (B,), device=DEV, generator=g)
        fresh = torch.randint(max(1, T // 2), T + 1, (B,), device=DEV, generator=g)
        table, pages = _pages(g, [case["held"] + T] * B, block, 5)
        t = torch.arange(T, device=DEV)[None, :]
        at = held[:, None] + t
        slots = table.gather(1, at // block).long() * block + at % block
        s = {"slots": torch.where(t < fresh[:, None], slots, -1).to(torch.int32)}
        # the tokens that come outgrow those that are held now and then, as a text's later ones do
        s["k"], s["v"] = ((1.2 * n(B, Hkv, T, d) * torch.exp(0.7 * n(Hkv, 1, d))).to(dt) for _ in range(2))
    else:
        B = case["B"]
        lengths = _ragged(B, case["longest"], kind == "attend" and B >= 8)
        table, pages = _pages(g, lengths, block, 5)
        s = {"table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV), "total": sum(lengths),
             "offsets": _offsets(lengths)}
        if kind == "attend":
            s["q"] = n(B, case["Hq"], d).to(dt)
    (s["kc"], s["ks"]), (s["vc"], s["vs"]) = (_filled(g, pages, Hkv, block, d, codes) for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case.get("train"):
        for name in ("q", "k", "v"):
            s[name].requires_grad_(True)
    return dict(s, case=case)


def run(state):
    with torch.set_grad_enabled(own and bool(state["case"].get("train"))):
        return {"packed": _packed, "write": _write, "read": _read, "attend": _attend}[state["case"]["kind"]](state)


# ---- attention over texts laid end to end --------------------------------------------

def _padded(offsets, n):
    """Row of token i of each text [texts, longest], whether it is one, and each row's text and place in it."""
    off = offsets.long()
    i = torch.arange(max(n), device=DEV)[None, :]
    there = i < (off[1:] - off[:-1])[:, None]
    row = torch.arange(sum(n), device=DEV)
    text = torch.bucketize(row, off[1:], right=True)
    return (off[:-1, None] + i).clamp(max=max(sum(n) - 1, 0)), there, text, row - off[text]


def _packed(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        o = fs.packed_attention(s["q"], s["k"], s["v"], s["offsets"], s["key_offsets"] if case["fresh"] else None,
                                window=case["window"], sinks=case["sinks"])
        if not case["train"]:
            return [o]
        return [o.detach()] + list(torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))
    Hkv, d, G = case["Hkv"], case["d"], case["Hq"] // case["Hkv"]
    dt, scale = s["q"].dtype, d ** -0.5
    iq, there, text, place = _padded(s["offsets"], s["nq"])
    ik, known, ktext, kplace = _padded(s["key_offsets"], s["nk"])
    S, tq, tk = len(s["nq"]), iq.shape[1], ik.shape[1]

    def rows(x):  # [H, N, d] -> [Hkv, texts, G longest, d]: the query heads of a key head one after the other
        x = x.float()[:, iq] * there[None, :, :, None]
        return x.unflatten(0, (Hkv, G)).transpose(1, 2).reshape(Hkv, S, G * tq, d)

    def back(x):
        return x.view(Hkv, S, G, tq, d).transpose(1, 2).flatten(0, 1)[:, text, place].to(dt)

    q, k, v = rows(s["q"]), (s["k"].float()[:, ik] * known[None, :, :, None]), s["v"].float()[:, ik]
    ahead = (known.sum(1) - there.sum(1))[:, None, None]
    p, j = torch.arange(tq, device=DEV)[None, :, None] + ahead, torch.arange(tk, device=DEV)[None, None, :]
    hidden = (j > p) | ~known[:, None, :]
    if case["window"]:
        hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
    hidden = hidden[None, :, None]
    w = (q @ k.transpose(-1, -2)).mul_(scale).view(Hkv, S, G, tq, tk).masked_fill_(hidden, -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    w = w.div_(w.sum(-1, keepdim=True).clamp(min=1e-30)).view(Hkv, S, G * tq, tk)
    out = [back(w @ v)]
    if not case["train"]:
        return out
    do = rows(s["do"])
    dv = w.transpose(-1, -2) @ do
    dw = do @ v.transpose(-1, -2)
    dw = dw.sub_((dw * w).sum(-1, keepdim=True)).mul_(w).mul_(scale)
    dq, dk = dw @ k, dw.transpose(-1, -2) @ q
    return out + [back(dq), dk[:, ktext, kplace].to(dt), dv[:, ktext, kplace].to(dt)]


# ---- keys and values into 8-bit pages ------------------------------------------------

def _values(codes, scale):
    return codes.to(torch.float32) * scale[:, :, None, None]


def _write(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        fs.paged_cache_write(s["k"], s["v"], s["slots"], s["kc"], s["vc"], s["ks"], s["vs"])
    else:
        block = case["block"]
        b, t = torch.nonzero(s["slots"] >= 0, as_tuple=True)
        slot = s["slots"][b, t].long()
        page, at = slot // block, slot % block
        _write_one(s["k"][b, :, t].float(), page, at, s["kc"], s["ks"], case["codes"])
        _write_one(s["v"][b, :, t].float(), page, at, s["vc"], s["vs"], case["codes"])
    return [_values(s["kc"], s["ks"]), _values(s["vc"], s["vs"]), s["ks"], s["vs"]]


def _write_one(x, page, at, cache, scale, codes):
    """x [tokens, Hkv, d] into cache [pages, Hkv, block, d] and scale [pages, Hkv], in place."""
    pages, _, block, _ = cache.shape
    rows = page[:, None].expand(-1, x.shape[1])
    amax = torch.full_like(scale, -1.0).scatter_reduce_(0, rows, x.abs().amax(-1), "amax")
    touched = amax >= 0  # this cache holds finite values alone
    begun = torch.zeros(pages, dtype=torch.bool, device=DEV)
    begun[page[at == 0]] = True
    need = _least_scale(amax.clamp(min=0.0), codes)
    m0, e0 = torch.frexp(scale)
    m1, e1 = torch.frexp(need)
    k = (e1 - e0 + (m1 > m0).to(torch.int32)).clamp(min=0)  # doublings until the old scale suffices
    k = torch.where((need > 0) & (scale > 0) & touched & ~begun[:, None], k, 0).clamp(max=126)
    new = torch.where(begun[:, None] | (scale <= 0), need, scale * _pow2(k))
    new = torch.where(touched, new, scale)
    # the codes that are held shrink with the scale's growth; those of the written slots are replaced after that
    cache.copy_(_to_codes(cache.to(torch.float32) * _pow2(-k)[:, :, None, None], codes))
    scale.copy_(new)
    fresh = _to_codes(x * _inverse(new)[page][:, :, None], codes)
    cache.view(torch.int8)[page, :, at] = fresh.view(torch.int8)


# ---- pages read back -----------------------------------------------------------------

def _read(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        return list(fs.paged_cache_read(s["kc"], s["vc"], s["table"], s["offsets"], s["total"], s["ks"], s["vs"],
                                        dtype=DTYPES[case["dtype"]]))
    row = torch.arange(s["total"], device=DEV)
    off = s["offsets"].long()
    text = torch.bucketize(row, off[1:], right=True)
    place = row - off[text]
    page, at = s["table"][text, place // case["block"]].long(), place % case["block"]

    def rows(cache, scale):
        x = cache.view(torch.int8)[page, :, at].view(cache.dtype).to(torch.float32) * scale[page][:, :, None]
        return x.transpose(0, 1).to(DTYPES[case["dtype"]]).contiguous()

    return [rows(s["kc"], s["ks"]), rows(s["vc"], s["vs"])]


# ---- attention of one token over 8-bit pages -----------------------------------------

def _attend(s):
    case = s["case"]
    if own:
        from edifice_amd import fused_scan as fs
        return [fs.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lengths"], window=case["window"],
                                   sinks=case["sinks"], k_scale=s["ks"], v_scale=s["vs"])]
    B, Hq, Hkv, d = (case[c] for c in ("B", "Hq", "Hkv", "d"))
    at = s["table"].clamp(min=0).long()

    def rows(cache, scale):
        x = cache.view(torch.int8)[at].view(cache.dtype).to(torch.float32) * scale[at][..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, -1, d)

    k, v = rows(s["kc"], s["ks"]), rows(s["vc"], s["vs"])
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


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "packed":
        nq, nk = _texts(case)
        pairs = 0
        for n, m in zip(nq, nk):
            p = np.arange(m - n, m, dtype=np.float64) + 1  # keys up to each query
            if case["window"]:
                p = np.minimum(p, case["window"]) + np.minimum(np.maximum(p - case["window"], 0), case["sinks"])
            pairs += float(p.sum())
        flops = 4 * case["d"] * pairs * case["Hq"]
        qo, kv = case["Hq"] * sum(nq) * case["d"] * size, case["Hkv"] * sum(nk) * case["d"] * size
        if case["train"]:
            return {"bytes": 5 * qo + 6 * kv, "flops": 3.5 * flops}
        return {"bytes": 2 * qo + 2 * kv, "flops": flops}
    if kind == "write":  # a row fills three quarters of its batch on average; the values are read, a byte each is written
        n = case["B"] * (0.75 * case["T"] if case["T"] > 1 else 1) * case["Hkv"] * case["d"]
        return {"bytes": 2 * n * (size + 1), "flops": 0}
    lengths = _ragged(case["B"], case["longest"], kind == "attend" and case["B"] >= 8)
    if kind == "read":
        return {"bytes": 2 * sum(lengths) * case["Hkv"] * case["d"] * (1 + size), "flops": 0}
    if case["window"]:
        lengths = [min(n, case["window"]) + min(max(n - case["window"], 0), case["sinks"]) for n in lengths]
    n = sum(lengths)
    return {"bytes": 2 * n * case["Hkv"] * (case["d"] + 4 / case["block"]) + 2 * case["B"] * case["Hq"] * case["d"] * size,
            "flops": 4 * n * case["Hq"] * case["d"]}


# ---- the definitions in 64 bits ------------------------------------------------------

def _exact_packed(case, s):
    Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
    nq, nk, G = s["nq"], s["nk"], Hq // Hkv
    if Hq * sum(n * m for n, m in zip(nq, nk)) > 3e9:
        return None
    o = torch.zeros(Hq, sum(nq), d, dtype=torch.float64, device=DEV)
    dq = torch.zeros_like(o)
    dk, dv = (torch.zeros(Hkv, sum(nk), d, dtype=torch.float64, device=DEV) for _ in range(2))
    at, kat = 0, 0
    for n, m in zip(nq, nk):
        ks = slice(kat, kat + m)
        for h in range(Hkv):
            kd, vd = s["k"][h, ks].double(), s["v"][h, ks].double()
            for lo in range(0, n, 512):  # a band of queries
                hi = min(n, lo + 512)
                pos = torch.arange(lo, hi, device=DEV)[:, None] + (m - n)
                j = torch.arange(m, device=DEV)[None, :]
                see = j <= pos
                if case["window"]:
                    see = see & ((j > pos - case["window"]) | (j < case["sinks"]))
                hs, rows = slice(h * G, (h + 1) * G), slice(at + lo, at + hi)
                qd = s["q"][hs, rows].double()
                a = torch.where(see, torch.matmul(qd, kd.t().contiguous()) / math.sqrt(d), -torch.inf)
                p = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
                ob = torch.matmul(p, vd)
                o[hs, rows] = ob
                if case["train"]:
                    go = s["do"][hs, rows].double()
                    e = p * (torch.matmul(go, vd.t().contiguous()) - (go * ob).sum(-1, keepdim=True)) / math.sqrt(d)
                    dq[hs, rows] = torch.matmul(e, kd)
                    dk[h, ks] += torch.matmul(e.flatten(0, 1).t(), qd.flatten(0, 1))
                    dv[h, ks] += torch.matmul(p.flatten(0, 1).t(), go.flatten(0, 1))
        at, kat = at + n, kat + m
    return [o, dq, dk, dv] if case["train"] else [o]


def _exact_scale(amax, codes):
    if amax == 0:
        return 0.0
    if codes == "int8":  # a float32 number: the product with the float32 nearest to a 127th
        return max(float(np.float32(amax * float(np.float32(1 / 127)))), LEAST)
    return max(2.0 ** math.ceil(math.log2(amax / 448.0)), LEAST)


def _exact_write(case, s):
    block, codes = case["block"], case["codes"]
    if case["B"] * case["T"] * case["Hkv"] > 20000:
        return None
    slots = s["slots"].cpu().numpy()
    out, scales = [], []
    for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.double().cpu().numpy()
        c, sc = cache.to(torch.float32).double().cpu().numpy(), scale.double().cpu().numpy()
        by_page = {}
        for b, t in zip(*np.nonzero(slots >= 0)):
            by_page.setdefault(int(slots[b, t]) // block, []).append((int(slots[b, t]) % block, int(b), int(t)))
        for page, tokens in by_page.items():
            begun = any(a == 0 for a, _, _ in tokens)
            for h in range(case["Hkv"]):
                need = _exact_scale(max(float(np.abs(x[b, h, t]).max()) for _, b, t in tokens), codes)
                old = sc[page, h]
                new, fall = (need, 1.0) if begun or old <= 0 else (old, 1.0)
                while not (begun or old <= 0) and new < need:
                    new, fall = 2 * new, 2 * fall
                if fall > 1:
                    c[page, h] = _exact_codes(c[page, h] / fall, codes)
                for a, b, t in tokens:
                    c[page, h, a] = _exact_codes(x[b, h, t] / new, codes) if new > 0 else 0.0
                sc[page, h] = new
        out.append(torch.from_numpy(c * sc[:, :, None, None]))
        scales.append(torch.from_numpy(sc))
    return [t.to(DEV) for t in out + scales]


def _exact_codes(y, codes):
    if codes == "int8":
        return np.clip(np.rint(y), -127, 127)
    e = np.maximum(np.frexp(np.abs(y))[1] - 1, -6)  # three bits below the leading one, from 2^-6 on a fixed step
    return np.rint(np.ldexp(y, 3 - e)) * np.ldexp(1.0, e - 3)


def _exact_read(case, s):
    lengths, table, block = s["lengths"].tolist(), s["table"].cpu().long(), case["block"]
    out = []
    for cache, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        x = cache.to(torch.float32).double() * scale.double()[:, :, None, None]
        texts = [x[table[b, :-(-n // block)].to(DEV)].transpose(1, 2).flatten(0, 1)[:n] for b, n in enumerate(lengths)]
        out.append(torch.cat(texts).transpose(0, 1))
    return out


def _exact_attend(case, s):
    B, Hq, Hkv, d = (case[c] for c in ("B", "Hq", "Hkv", "d"))
    o = torch.zeros(B, Hq, d, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        if n:
            j = torch.arange(n, device=DEV)
            if case["window"]:
                j = j[(j >= n - case["window"]) | (j < case["sinks"])]
            page = s["table"][b].long()[j // case["block"]]
            k, v = (c.view(torch.int8)[page, :, j % case["block"]].view(c.dtype).to(torch.float32).double()
                    * w.double()[page][..., None] for c, w in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            a = torch.matmul(s["q"][b].double().view(Hkv, Hq // Hkv, d), k.permute(1, 2, 0).contiguous()) / math.sqrt(d)
            o[b] = torch.matmul(torch.softmax(a, -1), v.transpose(0, 1).contiguous()).view(Hq, d)
    return [o]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"packed": _exact_packed, "write": _exact_write, "read": _exact_read, "attend": _exact_attend}[case["kind"]](
        case, s)
