"""The loss over a vocabulary where 32 bits run out: logits whose neighbours are far apart, and logits so far from zero that a log-sum-exp has few
bits left. Every logit here is exact in fp32 in whatever order its products are summed, so float64 has the kernels' own logits."""
import numpy as np
import pytest

import language_ref as ref
from frame_hip import synth
from test_gpu_vocab_loss import Loss, say

pytestmark = pytest.mark.gpu
F16, BF16 = 2, 3


def store(a, dtype):
    s = synth.to_storage(np.asarray(a, np.float32), dtype)
    assert np.array_equal(ref.values(s, dtype), np.asarray(a, np.float64)), "an input of these tests is not exact"
    return s


@pytest.mark.parametrize("tokens", [70, 600])
@pytest.mark.parametrize("case", [(BF16, 8, 8), (BF16, 11, 12), (BF16, 30, 30), (BF16, 57, 57), (F16, 15, 8)], ids=str)
def test_logits_whose_neighbours_are_far_apart(hip, case, tokens):
    """Logits of +-64 k 2^(a + b), k = 1 .. 200, up to 2^127: softmax is 1 at the largest and 0 at all others, in 32 bits as in 64."""
    dtype, a, b = case
    say(f"logits up to 2^{a + b + 13}, {tokens} rows, dtype={dtype}")
    p = Loss(hip, dtype, tokens, 200, 64, 0.1)
    k = np.random.default_rng(5).permutation(np.arange(1, 201)).astype(np.float64)
    sign = np.where(np.arange(tokens) % 2 == 0, 1.0, -1.0)
    p.w = store(np.repeat((k * 2.0 ** b)[:, None], 64, 1), dtype)
    p.x = store(np.repeat((sign * 2.0 ** a)[:, None], 64, 1), dtype)
    z = 64 * 2.0 ** (a + b) * sign[:, None] * k[None, :]
    rows = np.arange(tokens)[p.counted]
    target, top = p.targets[p.counted], z.argmax(1)[p.counted]
    loss, row, lse = p.forward()
    assert np.array_equal(lse[rows], z[rows, top].astype(np.float32))  # 200 is 8 bits
    assert np.array_equal(row[rows], (z[rows, top] - z[rows, target]).astype(np.float32))
    want = row[rows].astype(np.float64).mean()
    assert abs(loss - want) <= 2.0 ** -23 * want
    dx, dw = (ref.values(g, dtype) for g in p.backward(lse))
    g = np.zeros((rows.size, 200))
    g[np.arange(rows.size), top] += 1
    g[np.arange(rows.size), target] -= 1
    for got, want in ((dx[rows], g @ ref.values(p.w, dtype) / rows.size), (dw, g.T @ ref.values(p.x, dtype)[rows] / rows.size)):
        # exact sums but for the factor's rounding and product, and the result's rounding
        ref.check(got, want, ref.rounded(want, 2.0 ** -22 * np.abs(want), dtype), "gradient")


def confident(hip, dtype, tokens, vocab, shift):
    """Logits of `shift` and a few more, all multiples of 1/16; a row's target is the first or the last token, 16 to 30 above its usual logit.
    Column 1 of w is 1 at the first token and 0 elsewhere: dx there is the derivative at that token."""
    p = Loss(hip, dtype, tokens, vocab, 64, 0.1)
    rng = np.random.default_rng(17)
    w = rng.integers(-4, 5, (vocab, 64)) / 4.0
    x = rng.integers(-2, 3, (tokens, 64)) / 4.0
    w[:, :3] = 0
    w[:, 0] = w[0, 1] = w[-1, 2] = 1
    raised = rng.integers(64, 121, tokens) / 4.0
    even = np.arange(tokens) % 2 == 0
    x[:, 0], x[:, 1], x[:, 2] = shift, np.where(even, raised, 0), np.where(even, 0, raised)
    p.x, p.w = store(x, dtype), store(w, dtype)
    p.targets = np.where(p.counted, np.where(even, 0, vocab - 1), -1).astype(np.int32)
    return p, x @ w.T, even & p.counted


SHIFTS = [0.0, -800.0, 800.0, 30000.0]


@pytest.mark.parametrize("shape", [(90, 1000), (700, 1500), (2048, 9000)], ids=str)
@pytest.mark.parametrize("shift", SHIFTS)
def test_a_probability_is_at_most_one(hip, shape, shift):
    """However few bits the log-sum-exp has left, it is not less than its row's largest logit: the derivative at a target is never positive."""
    say(f"derivatives at confident targets, shift {shift}, {shape}")
    p, z, first = confident(hip, F16, *shape, shift) if shift == 30000.0 else confident(hip, BF16, *shape, shift)
    _, _, lse = p.forward()
    assert (lse[p.counted] >= z.max(1)[p.counted]).all()
    # the log-sum-exp is off by its rounding, a logarithm's and a sum's errors
    exact = z.max(1) + np.log(np.exp(z - z.max(1, keepdims=True)).sum(1))
    ref.check(lse[p.counted].astype(np.float64), exact[p.counted], 1.01 * 2.0 ** -24 * np.abs(exact[p.counted]) + 2.0 ** -17, "lse")
    dx, _ = p.backward(lse, 2.0 ** 10)
    d = ref.values(dx, p.dtype)[first, 1] * p.counted.sum() / 2.0 ** 10
    assert (d <= 0).all(), d.max()
    want = np.expm1(z[first, 0] - exact[first])
    # a probability's error is its exponent's, by the log-sum-exp's; two roundings follow
    ref.check(d, want, 1.02 * (2.0 ** -24 * np.abs(exact[first]) + 2.0 ** -16) + 2.1 * ref.U[p.dtype] * np.abs(want) + 2.0 ** -20, "derivative")


@pytest.mark.parametrize("shape", [(5, 300), (90, 1000), (700, 1500), (2048, 9000)], ids=str)
@pytest.mark.parametrize("shift", SHIFTS)
def test_losses_of_confident_rows(hip, shape, shift):
    """Losses of 1e-9 to 1e-3, as exact around logits of hundreds as around zero. Off by the sum's roundings, 64 of at most 2^-24 (32 in a lane, the
    rest in joins) and the logarithm's 2^-22, and relative to themselves by their exponents' (products of up to 60 rounded three times)."""
    say(f"losses of confident rows, shift {shift}, {shape}")
    p, z, _ = confident(hip, F16 if shift == 30000.0 else BF16, *shape, shift)
    loss, row, _ = p.forward()
    n, z, target = p.counted.sum(), z[p.counted], p.targets[p.counted]
    d = z - z[np.arange(n), target][:, None]
    d[np.arange(n), target] = -np.inf
    want = np.log1p(np.exp(d).sum(1))
    tol = 68 * 2.0 ** -24 + 2.0 ** -18 * want
    assert (row >= 0).all() and np.median(want) < 1e-5
    ref.check(row[p.counted].astype(np.float64), want, tol, "row_loss")
    assert abs(loss - want.mean()) <= tol.mean() + 2.0 ** -23 * want.mean()


@pytest.mark.parametrize("shape", [(5, 300), (90, 1000), (700, 1500), (2048, 9000)], ids=str)
@pytest.mark.parametrize("shift", SHIFTS)
def test_losses_of_confident_rows_keep_their_bits(hip, shape, shift):
    """The same to a part of themselves: the other tokens' exponents (up to 30, three roundings), their sum's logarithm (up to 13) and its
    distance from the target's logit (up to 33) are off by less than 2^-16 in all, 256 roundings of one."""
    say(f"losses of confident rows to their last bits, shift {shift}, {shape}")
    p, z, _ = confident(hip, F16 if shift == 30000.0 else BF16, *shape, shift)
    loss, row, _ = p.forward()
    n, z, target = p.counted.sum(), z[p.counted], p.targets[p.counted]
    d = z - z[np.arange(n), target][:, None]
    d[np.arange(n), target] = -np.inf
    want = np.log1p(np.exp(d).sum(1))
    ref.check(row[p.counted].astype(np.float64), want, 2.0 ** -16 * want, "row_loss")
    assert abs(loss - want.mean()) <= (2.0 ** -16 + 2.0 ** -23) * want.mean()


def test_a_target_of_infinite_logit(hip):
    """+infinity makes its row NaN whoever's it is; a target of -infinity has an infinite loss; the only token has a loss of 0."""
    say("the target's logit is infinite; a vocabulary of one")
    p = Loss(hip, BF16, 20, 300, 64)
    p.x[:, 0], p.w[:, 0] = 0, 0
    lse0 = p.forward()[2]
    p.x[:, 0] = 0x3f80  # 1.0
    p.targets[:] = np.where(np.arange(20) < 10, 7, 8)
    p.w[7, 0] = 0xff80  # -infinity
    _, row, lse = p.forward()
    assert (row[:10] == np.inf).all() and np.isfinite(row[10:]).all() and np.isfinite(lse).all() and (lse <= lse0).all()
    p.w[7, 0] = 0x7f80  # +infinity
    _, row, lse = p.forward()
    assert np.isnan(row).all() and np.isnan(lse).all()
    q = Loss(hip, BF16, 20, 1, 64)
    _, row, lse = q.forward()
    assert (row == 0).all() and np.isfinite(lse).all()
