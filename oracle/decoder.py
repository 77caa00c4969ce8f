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
