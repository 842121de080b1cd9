"""Beam selection from its definition in 64 bits (test infrastructure only)."""
from __future__ import annotations

import numpy as np


def log_probs(x: np.ndarray) -> np.ndarray:
    """log softmax of the last axis in float64; NaN is -inf, +inf the largest float32, a row of -inf stays -inf."""
    x = np.nan_to_num(x.astype(np.float64), nan=-np.inf, posinf=float(np.finfo(np.float32).max), neginf=-np.inf)
    m = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = np.where(np.isneginf(m), -np.inf, x - np.where(np.isneginf(m), 0, m))
        return np.where(np.isneginf(m), -np.inf, d - np.log(np.exp(d).sum(-1, keepdims=True)))


def select(logits: np.ndarray, scores: np.ndarray, n: int, finished=None, eos: int = -1):
    """(scores float64, tokens, parents) [B, n]: by score, then lower beam, then larger logit, then lower token."""
    B, K, V = logits.shape
    x = np.nan_to_num(logits.astype(np.float64), nan=-np.inf, posinf=float(np.finfo(np.float32).max), neginf=-np.inf)
    lp = log_probs(logits)
    if finished is not None:
        one = np.full(V, -np.inf)
        one[eos] = 0
        lp[finished], x[finished] = one, one
    with np.errstate(invalid="ignore"):
        total = scores.astype(np.float64)[..., None] + lp
    total = np.where(np.isnan(total), -np.inf, total)
    beam = np.broadcast_to(np.arange(K)[:, None], (K, V)).ravel()
    token = np.broadcast_to(np.arange(V), (K, V)).ravel()
    out = []
    for b in range(B):
        t, v = total[b].ravel(), x[b].ravel()
        order = np.lexsort((token, -v, beam, -t))[:n]
        out.append((t[order], token[order], beam[order]))
    return tuple(np.stack(a) for a in zip(*out))
