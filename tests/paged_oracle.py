"""Attention over a paged cache, what its tokens get of it, and eviction by that, restated
on the CPU in 64 bits: numpy and torch, none of the package's code."""
from __future__ import annotations

import math

import numpy as np
import torch


def attention(q, k, v, scale, visible):
    """One sequence and one K/V head: q [rows, D], k, v [keys, D], visible [rows] keys of each
    row.  Returns (out, lse, p, largest sum of |q k scale| over the keys a row sees)."""
    q, k, v = (t.to(torch.float64) for t in (q, k, v))
    rows, keys = q.shape[0], k.shape[0]
    seen = torch.arange(keys)[None] < torch.as_tensor(visible)[:, None]
    s = torch.where(seen, (q @ k.T) * scale, -math.inf)
    lse = torch.logsumexp(s, 1) if keys else torch.full((rows,), -math.inf, dtype=torch.float64)
    none = ~seen.any(1)
    p = torch.where(seen & ~none[:, None], torch.exp(s - lse[:, None]), 0.0)
    # a product with what a row does not see is left out, not 0 times it
    out = torch.stack([p[r, :n] @ v[:n] for r, n in enumerate(seen.sum(1).tolist())]) \
        if rows else torch.zeros(0, v.shape[1], dtype=torch.float64)
    mags = torch.where(seen, (q.abs() @ k.abs().T) * abs(scale), 0.0)
    return out, lse, p, mags.amax(1) if keys else torch.zeros(rows, dtype=torch.float64)


def score_error(mags, dim):
    """How far a score, in units of e, may be off: its products are exact, each of the sums of
    `dim` terms within 2^-23 of the sum of their magnitudes, the scale and the product with it
    rounded (2^-22 in all), and 2^-20 for the exponential."""
    return mags * (dim * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -20


def tolerance(out, p, v, mags, dtype):
    """How far an output may be from the 64-bit one, by element.  Roundings: the output's own
    (half a step of its type); every weight p to the type (half a step, in the numerator alone;
    of fp16's below 2^-14 of the reference's weight, 2^-25 of that, with a sum of 1 and more
    to divide by); a score off by ds changes its weight by e^ds - 1 in numerator and
    denominator.  Sums of `keys` terms in 32 bits: 2^-23 each."""
    half = torch.finfo(dtype).eps / 2
    keys, dim = v.shape
    big = p @ v.to(torch.float64).abs()
    rel = half + 2 * torch.expm1(score_error(mags, dim)) + keys * 2.0 ** -23
    tol = half * out.abs() + (1 + half) * rel[:, None] * big
    top = v.abs().max().item() if v.numel() else 0.0
    if dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * top
    return tol + torch.finfo(dtype).smallest_normal * half * 2 + keys * 2.0 ** -126 * top


def weights_tolerance(p, mags, dim, before, total):
    """How far a token's sum may be off: every p by its score's error, that of the row's sum and
    2^-22 for the division and product; the sum of `rows` terms and the value before it, 2^-23
    each."""
    rows, keys = p.shape
    rel = torch.expm1(2 * score_error(mags, dim)) + keys * 2.0 ** -23 + 2.0 ** -22
    return (p * rel[:, None]).sum(0) + (rows + 1) * 2.0 ** -23 * (p.sum(0) + before.abs()) \
        + 2.0 ** -24 * total.abs() + rows * 2.0 ** -126


def choose(w, n, budget, recent):
    """The places, in order, of the tokens that stay of n with weights w."""
    stay = min(n, budget)
    recent = min(recent, stay)
    others = n - recent
    # NaN above all, -0 as 0; of equal ones the earlier
    def key(t):
        x = float(w[t])
        return (0, 0.0, t) if math.isnan(x) else (1, -(x + 0.0), t)
    best = sorted(range(others), key=key)[:stay - recent]
    return sorted(best) + list(range(others, n))


def rows_of(cache: np.ndarray, table, n):
    """Tokens [n, head, D] of a sequence, from a cache [block, token, head, D]."""
    T = cache.shape[1]
    return np.stack([cache[int(table[t // T]), t % T] for t in range(n)]) if n else \
        cache[:0].reshape(0, *cache.shape[2:])
