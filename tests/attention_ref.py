"""Attention over packed sequences and over a paged cache in float64, from the definitions, and how far a kernel may be off.

Tolerances. u is half the storage type's eps, the most a rounding is off relative to the value (bf16 2^-8, f16 2^-11); values under
the smallest normal one are off by half the smallest step instead (f16 2^-25; bf16's is out of reach here). Scores, exponentials and sums are
fp32: a score of dh products is off by at most (dh + 4) 2^-24 times the sum of its products' sizes (times scale), and the exponential and
the softmax's normalisation add 2^-20, together E; a probability is then off by 2 E relative to itself. What is rounded to the
storage type on the way is the operand of the second product (the probability p, in the gradients also ds) and, for the gradients,
the output that D = sum dout out is formed from. Each bound sums what its formula's terms can be off by.
"""
from __future__ import annotations

import numpy as np

from frame_hip import synth

U = {2: 2.0 ** -11, 3: 2.0 ** -8}
TINY = {2: 2.0 ** -25, 3: 2.0 ** -133}


def values(a, dtype):
    return synth.to_float(a, dtype).astype(np.float64)


def softmax_error(q, k, scale):
    """E of the file's comment, per query row."""
    dh = q.shape[-1]
    return (dh + 4) * 2.0 ** -24 * scale * (np.abs(q) @ np.abs(k).T).max(1, initial=0.0, keepdims=True) + 2.0 ** -20


def attend(q, k, v, seen, scale, dtype):
    """One head: q [n, dh], k, v [m, dh], seen [n, m] -> out, its tolerance, p, lse, the tolerance of lse. Rows that see nothing: zeros and -inf."""
    s = np.where(seen, scale * (q @ k.T), -np.inf) if k.shape[0] else np.full((q.shape[0], 0), -np.inf)
    top = s.max(1, initial=-np.inf, keepdims=True)
    e = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = e.sum(1, keepdims=True)
    p = e / np.where(total > 0, total, 1.0)
    with np.errstate(divide="ignore"):
        lse = (np.where(np.isfinite(top), top, 0.0) + np.log(total))[:, 0]
    out = p @ v
    E = softmax_error(q, k, scale) + (k.shape[0] + 64) * 2.0 ** -24
    u, size = U[dtype], p @ np.abs(v)
    tol = 1.02 * u * (size + np.abs(out)) + 2 * E * size + TINY[dtype] * (1 + np.abs(v).sum(0))
    return out, tol, p, lse, 2 * E[:, 0] + 2.0 ** -22 * np.abs(np.where(np.isfinite(lse), lse, 0.0))


def gradients(q, k, v, dout, out, p, scale, dtype):
    """One head's dq, dk, dv and their tolerances."""
    dp = dout @ v.T
    d = (p * dp).sum(1, keepdims=True)
    ds = p * (dp - d)
    u, t = U[dtype], TINY[dtype]
    E = softmax_error(q, k, scale) + (k.shape[0] + 64) * 2.0 ** -24
    dp_size = np.abs(dout) @ np.abs(v).T
    # D from the rounded output, in fp32; dp in fp32
    off_d = (u + 140 * 2.0 ** -24) * (np.abs(dout) * np.abs(out)).sum(1, keepdims=True)
    off_ds = 1.02 * u * np.abs(ds) + p * (1.02 * off_d + 140 * 2.0 ** -24 * dp_size) + 2 * E * np.abs(ds) + t
    off_p = 1.02 * u * p + 2 * E * p + t * (p > 0)
    parts = []
    for value, off, operand in ((ds, off_ds, k), (ds.T, off_ds.T, q), (p.T, off_p.T, dout)):
        factor = scale if operand is not dout else 1.0
        total = factor * (value @ operand)
        tol = factor * (off @ np.abs(operand))
        # the fp32 sum of the products
        tol += factor * (value.shape[1] + 4) * 2.0 ** -24 * (np.abs(value) @ np.abs(operand))
        parts.append((total, tol))
    return parts


def rounded(total, tol, dtype):
    """The tolerance after the result's own rounding."""
    return 1.02 * U[dtype] * np.abs(total) + 1.02 * tol + TINY[dtype]


def check(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    bad &= ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside the bound; first at {i}: got {got[i]!r}, want {want[i]!r}, "
                             f"bound {tol[i]:.3g}")


def e4m3_values(b):
    """The values of e4m3 bytes."""
    b = b.astype(np.int64)
    e, f = (b >> 3) & 15, (b & 7).astype(np.float64)
    size = np.where(e > 0, (8 + f) * 2.0 ** (e - 10.0), f * 2.0 ** -9)
    size = np.where((b & 127) == 127, np.nan, size)
    return np.where(b >= 128, -size, size)


def quantise(rows):
    """(e4m3 values as numbers, scale bytes) of float64 rows [..., dh]: the cache's definition."""
    finite = np.isfinite(rows)
    top = np.where(finite, np.abs(rows), 0.0).max(-1)
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(top / 448.0))
    e = np.where(top > 0, e, 0.0)
    e = np.where(top > 448.0 * 2.0 ** e, e + 1, e)
    e = np.where(top > 0, np.maximum(e, -126), 0.0)
    y = np.where(finite, rows, 0.0) / (2.0 ** e)[..., None]
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.where(finite, np.round(y / step) * step, np.nan), (e + 127).astype(np.uint8)
