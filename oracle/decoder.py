"""Float64 restatement (torch, CPU) of the served decoder's attention operators, test infrastructure only:
the head split with norms and rotary positions, attention with a window and sinks, the paged cache.

Each is written from its definition, row by row where that is the plainest, and the differentiable ones
are differentiable by torch autograd (pinned by finite differences in tests/test_oracle_decoder.py).
"""
from __future__ import annotations

import math

import torch


def rotate(n, angles, interleaved, amplitude):
    """n [..., T, d], angles [..., T, rot / 2] (radians): the first rot elements turned in pairs."""
    half = angles.shape[-1]
    rot = 2 * half
    a, b = (n[..., 0:rot:2], n[..., 1:rot:2]) if interleaved else (n[..., :half], n[..., half:rot])
    c, s = torch.cos(angles) * amplitude, torch.sin(angles) * amplitude
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, n[..., rot:]], -1)


def split_heads_rotary(x, num_heads, num_kv_heads, freq=None, positions=None, wq=None, wk=None, eps=1e-6,
                       interleaved=False, amplitude=1.0):
    B, T, width = x.shape
    d = width // (num_heads + 2 * num_kv_heads)
    heads = x.reshape(B, T, -1, d).transpose(1, 2)
    q, k, v = heads.split([num_heads, num_kv_heads, num_kv_heads], 1)
    pos = torch.arange(T) if positions is None else positions
    pos = pos.double().expand(B, T)
    out = []
    for u, w in ((q, wq), (k, wk)):
        if w is not None:
            u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + eps) * w
        if freq is not None:
            u = rotate(u, pos[:, None, :, None] * freq, interleaved, amplitude)
        out.append(u)
    return out[0], out[1], v


def window_mask(T, window, sinks):
    """[T, T]: query i sees key j."""
    i, j = torch.arange(T)[:, None], torch.arange(T)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def window_probabilities(q, k, window, sinks):
    G, T, d = q.shape[1] // k.shape[1], q.shape[2], q.shape[3]
    s = q @ k.repeat_interleave(G, 1).transpose(-1, -2) / math.sqrt(d)
    return torch.softmax(s.masked_fill(~window_mask(T, window, sinks), -math.inf), -1)


def window_attention(q, k, v, window, sinks=0):
    return window_probabilities(q, k, window, sinks) @ v.repeat_interleave(q.shape[1] // k.shape[1], 1)


def paged_attention(q, k_cache, v_cache, table, lengths, window=0, sinks=0):
    """q [B, H, d]; also returns sum_j P_j |v_j|, the size of an output's terms."""
    B, H, d = q.shape
    blocks, hkv, block, _ = k_cache.shape
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * block)
        keys = [j for j in range(n) if (window == 0 or j >= n - window or j < sinks)
                and 0 <= int(table[b, j // block]) < blocks]
        if not keys:
            continue
        pages = torch.tensor([int(table[b, j // block]) for j in keys])
        offs = torch.tensor([j % block for j in keys])
        for h in range(H):
            k, v = k_cache[pages, h * hkv // H, offs], v_cache[pages, h * hkv // H, offs]
            p = torch.softmax(k @ q[b, h] / math.sqrt(d), 0)
            out[b, h], mag[b, h] = p @ v, p @ v.abs()
    return out, mag


def paged_extend(table, old, new, free, block, tokens):
    """Lists in, (table, slots, positions, used) out: the definition, one token at a time."""
    table = [list(r) for r in table]
    width, at = len(table[0]), 0
    slots, positions = [], []
    for r, (o, n) in enumerate(zip(old, new)):
        o, n = max(o, 0), max(n, 0)
        for c in range(min(-(-o // block), width), min(-(-n // block), width)):
            table[r][c] = free[at] if at < len(free) else -1
            at += 1
        ps = [o + t if o + t < n else -1 for t in range(tokens)]
        positions.append(ps)
        slots.append([table[r][p // block] * block + p % block
                      if p >= 0 and p // block < width and table[r][p // block] >= 0 else -1 for p in ps])
    return table, slots, positions, at


def round_code(y, code):
    """y to the nearest number of 8 bits, ties to even: "int8" (-127 .. 127) or "e4m3" (three bits behind the leading one,
    a fixed step below 2^-6; |y| <= 448)."""
    if code == "int8":
        return torch.round(y).clamp(-127, 127)
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def least_scale(amax, code):
    """The scale (a float32 number) that values up to amax (float) need."""
    if not math.isfinite(amax):
        return math.nan
    if amax == 0:
        return 0.0
    if code == "int8":
        r = torch.tensor(amax, dtype=torch.float32) * torch.tensor(1 / 127, dtype=torch.float32)
        return max(float(r), 2.0 ** -100)
    e = -100
    while 448 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def paged_cache_write8(x, slots, cache, scale, code):
    """x [B, Hkv, T, d], slots (list of lists), cache [num_blocks, Hkv, block, d] (the numbers as float64) and scale
    [num_blocks, Hkv], the last two changed in place: one page at a time, from the definition.  A value is divided by its
    scale as the operator's definition has it, x (1 / s) with the float32 quotient, before it is rounded."""
    blocks, hkv, block, _ = cache.shape
    pages = {}
    for b, row in enumerate(slots):
        for t, s in enumerate(row):
            if 0 <= s < blocks * block:
                pages.setdefault(s // block, []).append((s % block, b, t))
    for page, tokens in pages.items():
        offs = [o for o, _, _ in tokens]
        others = [o for o in range(block) if o not in offs]
        for h in range(hkv):
            amax = max(float(x[b, h, t].abs().nan_to_num(math.inf, posinf=math.inf).max()) for _, b, t in tokens)
            need, old = least_scale(amax, code), float(scale[page, h])
            if 0 in offs:
                new = need
            elif old <= 0:
                new = need
                cache[page, h, others] = 0.0
            elif math.isnan(old) or math.isnan(need):
                new = math.nan
            else:
                new, halvings = old, 0
                while new < need:
                    new, halvings = 2 * new, halvings + 1
                if halvings:
                    cache[page, h, others] = round_code(cache[page, h, others] / 2.0 ** halvings, code)
            for o, b, t in tokens:
                if new > 0:
                    inv = 1.0 / torch.tensor(new, dtype=torch.float32)
                    cache[page, h, o] = round_code((x[b, h, t].float() * inv).double(), code)
                else:
                    cache[page, h, o] = 0.0
            scale[page, h] = new


def paged_cache_read(values, table, offsets, total):
    """values [num_blocks, Hkv, block, d] -> [Hkv, total, d]."""
    blocks, hkv, block, d = values.shape
    out = torch.zeros(hkv, total, d, dtype=values.dtype)
    for b in range(len(offsets) - 1):
        for i, row in enumerate(range(offsets[b], offsets[b + 1])):
            if 0 <= row < total and i < table.shape[1] * block and 0 <= int(table[b, i // block]) < blocks:
                out[:, row] = values[int(table[b, i // block]), :, i % block]
    return out


def packed_attention(q, k, v, offsets, key_offsets, window=0, sinks=0):
    """q [H, N, d], k, v [Hkv, M, d], lists of offsets: one text after the other; differentiable."""
    G = q.shape[0] // k.shape[0]
    rows = []
    for s in range(len(offsets) - 1):
        a, b, c, e = offsets[s], offsets[s + 1], key_offsets[s], key_offsets[s + 1]
        rows.append(text_probabilities(q[:, a:b], k[:, c:e], window, sinks) @ v[:, c:e].repeat_interleave(G, 0))
    rows.append(torch.zeros_like(q[:, offsets[-1]:]))
    return torch.cat(rows, 1)


def text_probabilities(q, k, window, sinks):
    """q [H, n, d] at the end of k [Hkv, m, d]: the probabilities [H, n, m], zeros where a query sees no key."""
    n, m = q.shape[1], k.shape[1]
    p, j = torch.arange(n)[:, None] + m - n, torch.arange(m)[None, :]
    see = j <= p
    if window:
        see = see & ((p - j < window) | (j < sinks))
    a = q @ k.repeat_interleave(q.shape[0] // k.shape[0], 0).transpose(-1, -2) / math.sqrt(q.shape[2])
    some = see.any(1, keepdim=True)
    return torch.softmax(a.masked_fill(~see & some, -math.inf), -1) * some if m else a
