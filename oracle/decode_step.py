"""The operators of a decode step over forked sequences, from their definitions (test infrastructure only)."""
from __future__ import annotations

import numpy as np


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, interleaved: bool) -> np.ndarray:
    """Rows [T, H, D] turned by cos / sin [T, R / 2], in the arrays' own precision: a product or a sum at a time."""
    half = cos.shape[1]
    out = x.copy()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, s = cos[:, None], sin[:, None]
    ra, rb = a * c - b * s, b * c + a * s
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = ra, rb
    else:
        out[..., :half], out[..., half:2 * half] = ra, rb
    return out


def adjust_row(x: np.ndarray, seen, generated, rep: float, pres: float, freq: float, bias=None, allowed=None) -> np.ndarray:
    """One row of logits (its own precision): ``seen`` and ``generated`` are lists of token ids, ``allowed`` bool [V]."""
    x, V, t = x.copy(), len(x), x.dtype.type
    with np.errstate(invalid="ignore", over="ignore"):
        for v in {v for v in seen if 0 <= v < V}:
            x[v] = x[v] / t(rep) if x[v] > 0 else x[v] * t(rep)
        times = {}
        for v in generated:
            if 0 <= v < V:
                times[v] = times.get(v, 0) + 1
        for v, n in times.items():
            x[v] = (x[v] - t(freq) * t(n)) - t(pres)
        if bias is not None:
            x = x + bias.astype(x.dtype)
        if allowed is not None:
            x = np.where(allowed, x, t(-np.inf))
    return x


def attention(q, k, v, visible: int, scale: float):
    """One query row [D] over keys [n, D], of which it sees the first ``visible``: (o [D], log-sum-exp), in 64 bits."""
    if visible <= 0:
        return np.zeros(len(q)), -np.inf
    s = k[:visible].astype(np.float64) @ q.astype(np.float64) * scale
    m = s.max()
    p = np.exp(s - m)
    return p @ v[:visible].astype(np.float64) / p.sum(), m + np.log(p.sum())
