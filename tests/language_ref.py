"""Token embedding, the loss over a vocabulary and their gradients in float64, from the definitions, and how far a kernel may be off.

Tolerances. u is half the storage type's eps, the most a rounding is off relative to the value (bf16 2^-8, f16 2^-11, f32 2^-24); values
under the smallest normal one are off by half the smallest step instead. Sums are fp32: one of n terms is off by at most (n + 4) 2^-24 times
the sum of the terms' sizes, whatever its order. A logit of dim products is such a sum, Ez at most; an exponential of a difference of
logits adds 2^-20 relative (its argument's roundings, 3 2^-24 of up to 40, and the instruction's own 2^-22). So the log-sum-exp is off by
Ez + 2^-20 + (vocab + 64) 2^-24 and its own rounding, and a probability formed from it by twice that relative to itself. The derivative
(probability less 1 at the target) is rounded to the storage type as an operand of the gradients' products, f16 after a product with 2^14.
"""
from __future__ import annotations

import numpy as np

from attention_ref import check, values  # noqa: F401  (the same values and the same comparison)

U = {0: 2.0 ** -24, 2: 2.0 ** -11, 3: 2.0 ** -8}
TINY = {0: 2.0 ** -150, 2: 2.0 ** -25, 3: 2.0 ** -134}
F32_SUM = 2.0 ** -24


def rounded(total, tol, dtype):
    """The tolerance after the result's own rounding."""
    return 1.02 * U[dtype] * np.abs(total) + 1.02 * tol + TINY[dtype]


def embed(table, ids, scale, dtype):
    named = (ids >= 0) & (ids < table.shape[0])
    out = np.where(named[:, None], table[np.where(named, ids, 0)] * scale, 0.0)
    return out, rounded(out, F32_SUM * np.abs(out), dtype) * (out != 0)


def embed_grad(dout, ids, vocab, scale, base, dtype):
    total, size = np.zeros((2, vocab, dout.shape[1]))
    named = (ids >= 0) & (ids < vocab)
    np.add.at(total, ids[named], dout[named] * scale)
    np.add.at(size, ids[named], np.abs(dout[named] * scale))
    if base is not None:
        total, size = total + base, size + np.abs(base)
    most = np.bincount(ids[named], minlength=vocab)[:, None]
    tol = rounded(total, (most + 4) * F32_SUM * size, dtype)
    return total, np.where(most > 0, tol, 0.0)  # rows that no token names: exact


class Loss:
    """x [n, dim], w [vocab, dim] in float64, targets [n]; the loss, its rows, the gradients for dloss, and tolerances."""

    def __init__(self, x, w, targets, mean, dtype, loss_dtype=0):
        self.w, self.dtype = w, dtype
        n, vocab = x.shape[0], w.shape[0]
        self.counted = (targets >= 0) & (targets < vocab)
        self.x, self.targets = x[self.counted], targets[self.counted]
        m = self.x.shape[0]
        self.n, self.vocab = n, vocab
        ez = (x.shape[1] + 4) * F32_SUM * (np.abs(self.x) @ np.abs(w).T).max(1, initial=0.0)
        z = self.x @ w.T
        top = z.max(1, initial=-np.inf, keepdims=True)
        lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0] if m else np.zeros(0)
        row = lse - z[np.arange(m), self.targets]
        self.off = ez + 2.0 ** -20 + (vocab + 64) * F32_SUM
        lse_tol = self.off + 2.0 ** -22 * np.abs(lse)
        row_tol = lse_tol + ez + 2.0 ** -23 * np.abs(row)
        self.lse, self.lse_tol = self._rows(lse), self._rows(lse_tol)
        self.row, self.row_tol = self._rows(row), self._rows(row_tol)
        self.share = 1.0 / max(m, 1) if mean else 1.0
        self.loss = row.sum() * self.share
        self.loss_tol = rounded(self.loss, row_tol.sum() * self.share, loss_dtype)
        self.p = np.exp(z - lse[:, None])
        self.g = self.p.copy()
        self.g[np.arange(m), self.targets] -= 1.0

    def _rows(self, some):
        out = np.zeros(self.n)
        out[self.counted] = some
        return out

    def gradients(self, dloss):
        f, u, t = dloss * self.share, U[self.dtype], TINY[self.dtype] * (2.0 ** -14 if self.dtype == 2 else 1.0)
        # the probability's error, twice the log-sum-exp's (formed again from a logit), the subtraction's and the rounding's
        off = self.p * (2 * self.off + 2.0 ** -20)[:, None] + F32_SUM + 1.02 * u * np.abs(self.g) + t
        dx, dx_tol = np.zeros((2, self.n, self.w.shape[1]))
        dx[self.counted] = f * (self.g @ self.w)
        dx_tol[self.counted] = abs(f) * ((off + (self.vocab + 8) * F32_SUM * np.abs(self.g)) @ np.abs(self.w))
        dw = f * (self.g.T @ self.x)
        dw_tol = abs(f) * ((off + (self.x.shape[0] + 8) * F32_SUM * np.abs(self.g)).T @ np.abs(self.x))
        tol = [rounded(v, e + 2.0 ** -22 * np.abs(v), self.dtype) for v, e in ((dx, dx_tol), (dw, dw_tol))]
        tol[0][~self.counted] = 0.0
        return (dx, tol[0]), (dw, tol[1])
