"""Float64 CPU restatement of the paged attention cache: block tables, rotary
positions and attention over tables.  Written one row (and, for attention, one
token and head) at a time from the definitions; imports neither the package nor
torch.
"""

from __future__ import annotations

import math

import numpy as np


def tables(lengths, T, table, held, free, n_free, block, n_new=None, shared=0):
    """``(slots, held, n_free, table, free)`` after T tokens a row (``n_new[b]``)."""
    table, free, held = np.array(table), np.array(free), list(held)
    B, width = table.shape
    new = [T] * B if n_new is None else [min(max(int(n), 0), T) for n in n_new]
    need = [max(-(-(int(n) + m) // block), shared) for n, m in zip(lengths, new)]
    top = int(n_free)
    for b in range(B):
        if need[b] <= width:
            for c in range(need[b], held[b]):
                free[top] = table[b, c]
                top += 1
    stack, asked, ok = top, 0, [True] * B
    for b in range(B):
        grow = need[b] - held[b]
        if need[b] > width:
            ok[b] = False
        elif grow > 0:
            asked += grow
            ok[b] = asked <= stack
            if ok[b]:
                for c in range(held[b], need[b]):
                    top -= 1
                    table[b, c] = free[top]
        if ok[b]:
            held[b] = need[b]
    slots = np.full((B, T), -1, np.int64)
    for b in range(B):
        for t in range(new[b] if ok[b] else 0):
            p = int(lengths[b]) + t
            slots[b, t] = table[b, p // block] * block + p % block
    return slots, np.array(held), top, table, free


def frequencies(rot, base, scaling=None):
    """Radians per position of each pair, and the rotated dims' factor."""
    inv = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    if scaling is None:
        return inv, 1.0
    s = scaling["factor"]
    if scaling["type"] == "linear":
        return inv / s, 1.0
    context = scaling["original_max_position_embeddings"]
    turns = {n: rot * math.log(context / (n * 2 * math.pi)) / (2 * math.log(base))
             for n in (scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0))}
    lo, hi = turns[scaling.get("beta_fast", 32.0)], turns[scaling.get("beta_slow", 1.0)]
    if scaling.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rot - 1)
    keep = 1.0 - np.clip((np.arange(rot // 2) - lo) / (hi - lo if hi != lo else 0.001), 0.0, 1.0)
    log_s = max(math.log(s), 0.0)
    factor = (1.0 + 0.1 * scaling.get("mscale", 1.0) * log_s) / (1.0 + 0.1 * scaling.get("mscale_all_dim", 0.0) * log_s)
    factor = scaling.get("attention_factor", factor)
    return inv * keep + inv / s * (1.0 - keep), factor


def norm_rotate(x, w, eps, pos, inv, factor, interleaved):
    """x ``[T, H, D]`` at positions pos ``[T]``: RMSNorm (w None: none), then the
    first ``2 len(inv)`` dims turned by ``pos * inv``."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y = x.copy()
    half = len(inv)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    ang = np.asarray(pos, np.float64)[:, None, None] * inv
    y[..., a] = (x[..., a] * np.cos(ang) - x[..., b] * np.sin(ang)) * factor
    y[..., b] = (x[..., b] * np.cos(ang) + x[..., a] * np.sin(ang)) * factor
    return y


def attend(q, keys, values, table, pos0, scale, n_new=None, gate=None):
    """q ``[B, T, Hq, D]`` over pools ``[N, Hkv, block, D]``; gate ``[B, T, Hq, D]``."""
    B, T, Hq, D = q.shape
    _, Hkv, block, _ = keys.shape
    out = np.zeros((B, T, Hq, D))
    for b in range(B):
        for t in range(T if n_new is None else int(n_new[b])):
            L = int(pos0[b]) + t + 1
            pages = table[b, : -(-L // block)]
            for h in range(Hq):
                k = keys[pages, h // (Hq // Hkv)].reshape(-1, D)[:L]
                v = values[pages, h // (Hq // Hkv)].reshape(-1, D)[:L]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k @ q[b, t, h] * scale
                    p = np.exp(s - s.max())
                    out[b, t, h] = (p / p.sum()) @ v
    return out if gate is None else out / (1.0 + np.exp(-gate))
