"""The 4-bit KV cache (OCP MXFP4) and attention over it, restated on the CPU in
64 bits: numpy and torch, none of the package's code."""
from __future__ import annotations

import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(x: np.ndarray):
    """Float64 rows [..., D] as (codes [..., D] of 0..15, scale bytes [..., D/32])."""
    shape = x.shape
    x = np.asarray(x, np.float64).reshape(-1, 32)
    codes = np.zeros(x.shape, np.uint8)
    scales = np.zeros(x.shape[0], np.uint8)
    for i, row in enumerate(x):
        if not np.isfinite(row).all():
            scales[i] = 255
            continue
        a = np.abs(row).max()
        e = -127
        if a > 0:
            m, e = np.frexp(a)
            m, e = 2 * m, int(e) - 1
            e = min(e + (m > 1.75), 127)
        s = max(e - 2, -127)
        scales[i] = s + 127
        q = np.abs(row) / np.ldexp(1.0, s)
        d = np.abs(q[:, None] - GRID[None])
        best = d.min(1)
        for j in range(32):
            near = np.flatnonzero(d[j] == best[j])
            c = near[0] if len(near) == 1 else next(n for n in near if n % 2 == 0)
            codes[i, j] = c | (8 if np.signbit(row[j]) else 0)
    return codes.reshape(shape), scales.reshape(*shape[:-1], shape[-1] // 32)


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.ldexp(1.0, scales.astype(int) - 127)
    s = np.where(scales == 255, np.nan, s)
    return v * np.repeat(s, 32, -1)


def pack_chunk(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """[T, H, D] codes and [T, H, D/32] scales as one chunk's bytes."""
    c = codes.transpose(1, 0, 2)
    b = (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)
    return np.concatenate([b.reshape(-1), scales.transpose(1, 2, 0).reshape(-1)])


def unpack_chunk(chunk: np.ndarray, T: int, H: int, D: int):
    b = chunk[:T * H * D // 2].reshape(H, T, D // 2)
    c = np.empty((H, T, D), np.uint8)
    c[..., 0::2], c[..., 1::2] = b & 15, b >> 4
    s = chunk[T * H * D // 2:].reshape(H, D // 32, T)
    return c.transpose(1, 0, 2), s.transpose(2, 0, 1)


def chunk_values(chunk: np.ndarray, T: int, H: int, D: int) -> np.ndarray:
    """[T, H, D] values of a chunk's bytes."""
    return decode(*unpack_chunk(chunk, T, H, D))


def as_type(x: np.ndarray, dtype: torch.dtype) -> torch.Tensor:
    """Values in `dtype`; finite ones past its largest become that one."""
    t = torch.from_numpy(np.ascontiguousarray(x))
    top = torch.finfo(dtype).max
    return torch.where(t.isfinite(), t.clamp(-top, top), t).to(dtype)


def attention(q, k, v, scale, visible):
    """One sequence and one K/V head in 64 bits: q [rows, D], k, v [keys, D],
    visible [rows] keys of each row.  Returns (out, lse, weighted |v|, largest sum
    of |q k| scale over the keys a row sees)."""
    q, k, v = (t.to(torch.float64) for t in (q, k, v))
    rows, D = q.shape
    out, big = torch.zeros(rows, D, dtype=torch.float64), torch.zeros(rows, D, dtype=torch.float64)
    lse = torch.full((rows,), -float("inf"), dtype=torch.float64)
    mags = torch.zeros(rows, dtype=torch.float64)
    for r in range(rows):
        n = int(visible[r])
        if n <= 0:
            continue
        s = (k[:n] @ q[r]) * scale
        lse[r] = torch.logsumexp(s, 0)
        p = torch.softmax(s, 0)
        out[r] = p @ v[:n]
        big[r] = p @ v[:n].abs()
        mags[r] = ((k[:n].abs() @ q[r].abs()) * abs(scale)).max()
    return out, lse, big, mags


def tolerance(out, big, mags, keys, dtype, vmax):
    """How far an output may be from the 64-bit one, by element.
    Roundings: the output's own (half a step of its type); every weight p to 8
    significant bits (2^-8, the numerator alone) for bf16, 16 for fp16; a score off by
    ds changes its weight by e^ds - 1 in numerator and denominator.  ds: 128 products
    summed by the matrix instruction, then others, each sum within 2^-14 of the sum
    of magnitudes here (32-bit sums: 2^-24 a term; the instruction aligns a step's
    products before adding, which a probe saw cost 2^-16), and 2^-20 of the score and
    of the exponential for the exp.  Sums of `keys` terms in 32 bits: 2^-23 each."""
    half = torch.finfo(dtype).eps / 2
    p = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16
    ds = mags * (2.0 ** -14 + 2.0 ** -20) + 2.0 ** -20
    rel = p + 2 * torch.expm1(ds) + keys * 2.0 ** -23
    tiny = torch.finfo(dtype).smallest_normal * half * 2
    return half * out.abs() + (1 + half) * rel[:, None] * big + tiny + keys * 2.0 ** -126 * vmax
