"""What paged generation keeps on the GPU, by its definition and one entry at a
time: 4-bit rows, pages of sequences, beams (the reference samples one sequence
without a cache, model.py:617-652)."""
from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise4(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Values and exponent bytes [..., ceil(D / 32)] of rows [..., D] held as
    e2m1 codes times, for every 32 values, the smallest power of two 2^e (-126
    <= e <= 125) with the largest magnitude <= 6 * 2^e; the nearest code, of two as
    near the even one; 32 values with one that is not finite are all NaN (255)."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    G = -(-D // 32)
    y = np.zeros((*x.shape[:-1], 32 * G))
    y[..., :D] = x
    y = y.reshape(*x.shape[:-1], G, 32)
    bad = ~np.isfinite(y).all(-1)
    y = np.where(bad[..., None], 0.0, y)
    top = np.abs(y).max(-1)
    m, p = np.frexp(top)
    e = np.clip(np.where(top > 0, np.where(m <= 0.75, p - 3, p - 2), -126), -126, 125)
    z = y * np.exp2(-e.astype(np.float64))[..., None]
    off = np.abs(np.abs(z)[..., None] - MAGNITUDES)
    least = off.min(-1, keepdims=True)
    even = np.where(off == least, np.arange(8) % 2 + np.arange(8) / 100, np.inf).argmin(-1)
    q = MAGNITUDES[even] * np.where(np.signbit(z), -1.0, 1.0) * np.exp2(e.astype(np.float64))[..., None]
    q = np.where(bad[..., None], np.nan, q).reshape(*x.shape[:-1], 32 * G)[..., :D]
    return q, np.where(bad, 255, e + 127).astype(np.uint8)


def values4(codes: np.ndarray, exps: np.ndarray) -> np.ndarray:
    """Values of code bytes [..., D / 2] with exponent bytes [..., ceil(D / 32)]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = MAGNITUDES[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(exps == 255, np.nan, np.exp2(exps.astype(np.float64) - 127))
    return v * np.repeat(s, 32, -1)[..., :v.shape[-1]]


def plan(table, free, top: int, P: int, S: int, lengths, counts, T: int, window: int = 0):
    """Lists changed as ``paged_plan`` changes its tensors: (top, slots, missing)."""
    cap = len(table[0]) * S if len(table) else 0
    give, take = [], []
    for n, row in enumerate(table):
        has = [0 <= x < P for x in row]
        a = min(max(int(lengths[n]), 0), cap)
        b = min(max(a + int(counts[n]), 0), cap)
        if window:
            low = e = max(0, min(a, b) - window) // S
            while e > 0 and has[e - 1]:
                e -= 1
            give += [(n, i) for i in range(e, low)]
        give += [(n, i) for i in range(-(-b // S), -(-a // S)) if has[i]]
        if b > a:
            first = max(max(0, b - window) // S if window else 0, a // S)
            take += [(n, i) for i in range(first, -(-b // S)) if not has[i]]
    room, missing = top + len(give), 0
    if len(take) > room:
        missing = len(take) - room
    elif room > P:
        missing = -1
    else:
        for j, (n, i) in enumerate(give):
            free[room - 1 - j] = table[n][i]
            table[n][i] = -1
        for j, (n, i) in enumerate(take):
            table[n][i] = free[room - 1 - j]
        top = room - len(take)
    slots = [[-1] * T for _ in table]
    for n, row in enumerate(table):
        for t in range(min(T, max(int(counts[n]), 0))):
            pos = int(lengths[n]) + t
            if 0 <= pos < cap and 0 <= row[pos // S] < P:
                slots[n][t] = row[pos // S] * S + pos % S
    return top, slots, missing


def reorder(table: np.ndarray, lengths, parents: np.ndarray, S: int, P: int):
    """The new table, and the copies (source page, page, rows) it asks for."""
    N, B = parents.shape
    old = table.reshape(N, B, -1)
    new, copies = old.copy(), []
    for n in range(N):
        full, rows = max(int(lengths[n]), 0) // S, max(int(lengths[n]), 0) % S
        par = [int(p) if 0 <= p < B else b for b, p in enumerate(parents[n])]
        spare = [b for b in range(B) if b not in par]
        seen = set()
        for b in range(B):
            own = par[b] if par[b] not in seen else spare.pop(0)
            if par[b] in seen and rows and full < old.shape[2]:
                src, dst = int(old[n, par[b], full]), int(old[n, own, full])
                if 0 <= src < P and 0 <= dst < P:
                    copies.append((src, dst, rows))
            seen.add(par[b])
            new[n, b, :full], new[n, b, full:] = old[n, par[b], :full], old[n, own, full:]
    return new.reshape(table.shape), copies


def select(logits: np.ndarray, scores: np.ndarray, K: int, ended=None, pad: int = 0):
    """(scores float64, tokens, parents) [N, K]; of equal scores the lower beam's first, within a beam the larger
    logit's, then the lower token."""
    N, B, V = logits.shape
    out, tok, par = np.zeros((N, K)), np.zeros((N, K), np.int64), np.zeros((N, K), np.int64)
    for n in range(N):
        c, order = np.full((B, V), -np.inf), np.zeros((B, V))
        for b in range(B):
            s = float(scores[n, b])
            if not (s > -np.inf and s < np.inf):
                continue
            if ended is not None and ended[n, b]:
                c[b, pad] = s
                continue
            x = logits[n, b].astype(np.float64)
            if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
                continue
            m = x.max()
            c[b] = s + (x - m - np.log(np.exp(x - m).sum()))
            order[b] = np.where(x > -np.inf, x, 0.0)
        beam = np.repeat(np.arange(B), V)
        at = np.lexsort((-order.ravel(), beam, -c.ravel()))[:K]
        out[n], tok[n], par[n] = c.ravel()[at], at % V, at // V
    return out, tok, par
