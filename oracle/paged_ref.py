"""Paged K/V cache in 64 bits: the definition of appending, reading back and
decoding, one token at a time (the reference keeps no cache, model.py:736-739,
so the oracle here is the formula).

A cache is ``dict(k=..., v=...)`` of float64 arrays [P, Hk, S, D] holding the
rows' values; ``quantise`` gives the values a quantised row stands for."""
from __future__ import annotations

import math

import numpy as np


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Values and exponent bytes of rows [..., D] held as e4m3 codes times the
    smallest power of two 2^e (e >= -126) with the largest finite magnitude
    <= 448 * 2^e; codes rounded to nearest even, infinities NaN."""
    x = np.asarray(x, np.float64)
    fin = np.isfinite(x)
    top = np.where(fin, np.abs(x), 0.0).max(-1, keepdims=True)
    m, p = np.frexp(top)
    e = np.maximum(np.where(top > 0, np.where(m <= 0.875, p - 9, p - 8), -126), -126)
    y = np.where(fin, x, 0.0) * np.exp2(-e.astype(np.float64))
    step = np.exp2(np.maximum(np.frexp(y)[1] - 1, -6) - 3.0)  # 8 steps to a binade, 2^-9 the smallest
    q = np.rint(y / step) * step * np.exp2(e.astype(np.float64))
    return np.where(fin, q, np.nan), (e[..., 0] + 127).astype(np.uint8)


def place(table, pages: int, S: int, n: int, pos: int):
    """(page, row) of a position, or None."""
    if pos < 0 or pos // S >= table.shape[1]:
        return None
    page = int(table[n, pos // S])
    return (page, pos % S) if 0 <= page < pages else None


def append(buf: np.ndarray, new: np.ndarray, table, start, counts) -> None:
    """buf [P, Hk, S, D] in place; new [N, T, Hk, D] as the pages hold it."""
    for n in range(new.shape[0]):
        for t in range(min(int(counts[n]), new.shape[1])):
            at = place(table, buf.shape[0], buf.shape[2], n, int(start[n]) + t)
            if at is not None:
                buf[at[0], :, at[1]] = new[n, t]


def read(buf: np.ndarray, table, start, counts, T: int) -> np.ndarray:
    out = np.zeros((len(start), T, buf.shape[1], buf.shape[3]))
    for n in range(len(start)):
        for t in range(min(int(counts[n]), T)):
            at = place(table, buf.shape[0], buf.shape[2], n, int(start[n]) + t)
            if at is not None:
                out[n, t] = buf[at[0], :, at[1]]
    return out


def decode(q: np.ndarray, k: np.ndarray, v: np.ndarray, table, lengths, scale: float, window: int = 0,
           include_self: bool = True, norm: str = "mass"):
    """out [N, H, D], and what its error is measured by: the keys in range
    [N], and per row the weighted magnitude sum tau |v| / norm [N, H, D] and
    the largest sum_d |q_d k_d| / scale over its keys [N, H]."""
    N, H, D = q.shape
    P, Hk, S, _ = k.shape
    out, mag = np.zeros((N, H, D)), np.zeros((N, H, D))
    keys, dots = np.zeros(N, int), np.zeros((N, H))
    for n in range(N):
        length = min(max(int(lengths[n]), 0), table.shape[1] * S)
        hi = length if include_self else length - 1
        lo = max(0, length - 1 - window) if window else 0
        keys[n] = max(hi - lo, 0)
        at = [a for a in (place(table, P, S, n, s) for s in range(lo, hi)) if a is not None]
        if not at:
            continue
        pg, rw = np.array(at).T
        for h in range(H):
            hk = h // (H // Hk)
            K, V = k[pg, hk, rw], v[pg, hk, rw]
            with np.errstate(over="ignore"):
                tau = 1.0 / (1.0 + np.exp(-(K @ q[n, h]) / scale))
            f = 1.0 / max(tau.sum(), 1e-6) if norm == "mass" else 1.0 / max(keys[n], 1) if norm == "count" else 1.0
            out[n, h], mag[n, h] = f * (tau @ V), f * (tau @ np.abs(V))
            dots[n, h] = (np.abs(K) @ np.abs(q[n, h])).max() / abs(scale)
    return out, keys, mag, dots


def decode_bound(out, keys, mag, dots, D: int, eps: float) -> np.ndarray:
    """How far a row computed in float32 and rounded once may be from ``out``:

    * a score of D float32 products and the logistic function: (D + 8) 2^-24
      of sum |q k| / scale, plus 8 ulp, relative in tau;
    * tau as the sums take it: 2^-23 relative; 2^-16 for 16-bit results, room
      that no kernel needs (tests/test_paged_weights_gpu.py has the tight bound);
    * sums over the keys and the splits: (keys + 16) 2^-24 relative;
    numerator and mass alike (twice), then half a step of the output type."""
    u = 2.0 ** -24
    rel = (D + 8) * u * dots + 8 * u + (2.0 ** -16 if eps > 1e-4 else 2.0 ** -23) + (keys[:, None] + 16) * u
    arith = 2.0 * rel[..., None] * mag
    return arith + 0.5 * eps * (np.abs(out) + arith) + 1e-30
