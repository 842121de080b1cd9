"""One query row over a sequence's keys in 64 bits, and how far 16-bit operands may take its output (test infrastructure only).

The bound is on the 2-norm of a head's output error, for keys and values that the kernels multiply as they are given here.
With w_j = exp(s_j - max s), l = sum w_j and o = sum w_j v_j / l, each w_j is off by its own relative error d_j, which moves o by
sum w_j d_j (v_j - o) / l (to first order).  For independent d_j of mean 0 with |d_j| <= d this sum's norm passes
t d S, S = sqrt(sum w_j^2 (|v_j|^2 + |o|^2)) / l, with a probability below 2 exp(-t^2 / 2) (Hoeffding's inequality for
vectors): 3e-8 for t = 6, over the few thousand rows that a test looks at 1e-4.  d is made of
* the rounding of a probability to the operand type, `p_unit` = eps / 2;
* the error e of a logit: D 2^-23 sum |q k| for the sums in 32 bits, and t q_unit |q k|_2 for queries that are
  rounded too (of another type than the pool's, or in fixed point);
* the sums of o in 32 bits, which lose a step of 2^-23 with each of n / 16 partial products and joins: (n / 16 + 64) 2^-23.
A probability below its type's smallest normal value is off by half of a step, `p_step`, of its own: t p_step |u|_2 / l, with
u_j the norms of what it multiplies.  The output's rounding adds 2^-11 |o| + 2^-25 sqrt(D); exponentials and joins 2^-16 |o|.
"""
from __future__ import annotations

import math

import torch

T = 6.0


def attend(q, k, v, scale):
    """o [H, D], lse [H] and the weights w [H, n] of q [H, D] over k, v [n, H, D], all in float64."""
    s = torch.einsum("hd,nhd->hn", q, k) * scale
    top = s.amax(1, keepdim=True)
    w = (s - top).exp()
    l = w.sum(1)
    return torch.einsum("hn,nhd->hd", w, v) / l[:, None], l.log() + top[:, 0], w


def norm_bound(q, k, v, scale, o, w, p_unit, q_step=0.0, p_step=2.0**-25, p_times=None):
    """[H]: the bound above.  q_step [H, D]: most that a query's entry is off; p_times [n, H]: what a small probability multiplies
    (default: the values' norms)."""
    n, _, D = k.shape
    l = w.sum(1)
    size = torch.einsum("hd,nhd->hn", q.abs(), k.abs()).amax(1) * scale
    e = D * 2.0**-23 * size
    if isinstance(q_step, torch.Tensor):
        e = e + T * (torch.einsum("hd,nhd->hn", q_step**2, k**2).amax(1)).sqrt() * scale
    vn = v.norm(dim=2)  # [n, H]
    S = (w.T**2 * (vn**2 + o.norm(dim=1)**2)).sum(0).sqrt() / l
    small = (vn if p_times is None else p_times).norm(dim=0) / l
    return (T * ((p_unit + e + (n / 16 + 64) * 2.0**-23) * S + p_step * small)
            + (2.0**-11 + 2.0**-16) * o.norm(dim=1) + 2.0**-25 * math.sqrt(D))


def lse_bound(q, k, scale, lse, q_step=0.0):
    """[H]: how far the log-sum-exp may be off: a logit's error, sums of n positive terms in 32 bits, the rounding to fp16."""
    n, _, D = k.shape
    e = D * 2.0**-23 * torch.einsum("hd,nhd->hn", q.abs(), k.abs()).amax(1) * scale
    if isinstance(q_step, torch.Tensor):
        e = e + T * (torch.einsum("hd,nhd->hn", q_step**2, k**2).amax(1)).sqrt() * scale
    return torch.expm1(e) + 2.0**-16 + math.sqrt(n) * 2.0**-22 + 2.0**-11 * lse.abs() + 2.0**-25
