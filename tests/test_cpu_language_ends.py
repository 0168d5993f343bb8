"""What the token embedding's and the vocabulary loss' entry points refuse, decided on the host before any launch (no GPU needed), and the
float64 reference's own gradients against differences."""
import ctypes

import numpy as np
import pytest

import language_ref as ref
from frame_hip import abi

F32, F16, BF16 = 0, 2, 3
P = 4096  # an aligned address that nothing reads: every call here is refused, or has nothing to do
INVALID, UNIMPLEMENTED = 1, 4


def table(**over):
    f = dict(dtype=BF16, tokens=10, vocab=100, dim=64, row_stride=64, scale=1.0)
    f.update(over)
    return abi.TokenEmbedding(**f)


def loss(**over):
    f = dict(dtype=BF16, loss_dtype=F32, mean=1, tokens=10, vocab=100, dim=64, x_stride=64, w_stride=64)
    f.update(over)
    return abi.VocabLoss(**f)


@pytest.mark.parametrize("over,code", [
    (dict(dtype=1), UNIMPLEMENTED), (dict(dtype=6), UNIMPLEMENTED), (dict(tokens=-1), INVALID), (dict(vocab=0), INVALID),
    (dict(vocab=2 ** 31), INVALID), (dict(dim=0), INVALID), (dict(dim=2 ** 21, row_stride=2 ** 21), INVALID),
    (dict(tokens=2 ** 29), INVALID), (dict(tokens=2 ** 28, dim=2 ** 20, row_stride=2 ** 20), INVALID), (dict(row_stride=63), INVALID),
    (dict(row_stride=2 ** 41), INVALID), (dict(vocab=2 ** 30, dim=512, row_stride=512), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
], ids=str)
def test_embedding_sizes_are_refused(over, code):
    lib, r = abi.lib(), ctypes.byref(table(**over))
    assert lib.fh_embedding_fwd(r, P, P, P, None) == code
    assert lib.fh_last_error()
    assert lib.fh_embedding_grad_workspace(r) == -1
    assert lib.fh_embedding_grad(r, P, P, P, P, P, 1 << 50, None) == code


def test_embedding_pointers_are_refused():
    lib, r = abi.lib(), ctypes.byref(table())
    assert lib.fh_embedding_fwd(None, P, P, P, None) == INVALID
    for i in range(3):
        for bad in (None, P + 1):
            args = [P] * 3
            args[i] = bad
            assert lib.fh_embedding_fwd(r, *args, None) == INVALID, (i, bad)
    need = lib.fh_embedding_grad_workspace(r)
    assert need > 0
    assert lib.fh_embedding_grad(r, *[P] * 5, need - 1, None) == INVALID
    for i in range(5):  # dout, ids, base (which may be null), dtable, workspace
        for bad in (None, P + 1):
            if (i, bad) == (2, None):
                continue
            args = [P] * 5
            args[i] = bad
            assert lib.fh_embedding_grad(r, *args, need, None) == INVALID, (i, bad)
    four = ctypes.byref(table(dtype=F32))
    assert lib.fh_embedding_fwd(four, P + 2, P, P, None) == INVALID
    assert lib.fh_embedding_grad(r, P, P, None, P, P + 8, need, None) == INVALID


@pytest.mark.parametrize("over,code", [
    (dict(dtype=F32), UNIMPLEMENTED), (dict(dtype=16), UNIMPLEMENTED), (dict(loss_dtype=F16), INVALID), (dict(mean=2), INVALID),
    (dict(tokens=-1), INVALID), (dict(vocab=0), INVALID), (dict(dim=0), INVALID), (dict(dim=60), UNIMPLEMENTED),
    (dict(x_stride=56), INVALID), (dict(w_stride=68), INVALID), (dict(x_stride=2 ** 33), INVALID), (dict(tokens=2 ** 25), INVALID),
    (dict(vocab=2 ** 25), INVALID), (dict(dim=2 ** 21, x_stride=2 ** 21, w_stride=2 ** 21), INVALID),
    (dict(tokens=2 ** 24, vocab=2 ** 24), INVALID),
], ids=str)
def test_loss_sizes_are_refused(over, code):
    lib, r = abi.lib(), ctypes.byref(loss(**over))
    assert lib.fh_vocab_loss_workspace(r) == -1 and lib.fh_last_error()
    assert lib.fh_vocab_loss_grad_workspace(r) == -1 and lib.fh_vocab_loss_grad_least(r) == -1
    assert lib.fh_vocab_loss_fwd(r, *[P] * 7, 1 << 50, None) == code
    assert lib.fh_vocab_loss_grad(r, *[P] * 8, 1 << 50, None) == code


@pytest.mark.parametrize("what,over", [
    ("table", dict(tokens=2 ** 25 + 1)), ("table", dict(tokens=2 ** 25, dim=2048, row_stride=2048)),
    ("loss", dict(tokens=2 ** 24, vocab=2 ** 18)), ("loss", dict(vocab=2 ** 24, dim=2 ** 17, x_stride=2 ** 17, w_stride=2 ** 17)),
], ids=str)
def test_launches_of_2_to_the_32_threads_are_refused(what, over):
    lib, r = abi.lib(), ctypes.byref(table(**over) if what == "table" else loss(**over))
    if what == "table":
        assert lib.fh_embedding_fwd(r, P, P, P, None) == INVALID and lib.fh_embedding_grad_workspace(r) == -1
    else:
        assert lib.fh_vocab_loss_workspace(r) == -1 and lib.fh_vocab_loss_grad_workspace(r) == -1
    assert b"too large" in lib.fh_last_error()


def test_loss_pointers_are_refused():
    lib, r = abi.lib(), ctypes.byref(loss())
    assert lib.fh_vocab_loss_fwd(None, *[P] * 7, 1 << 50, None) == INVALID
    need, least, best = lib.fh_vocab_loss_workspace(r), lib.fh_vocab_loss_grad_least(r), lib.fh_vocab_loss_grad_workspace(r)
    assert 0 < least <= best
    assert lib.fh_vocab_loss_fwd(r, *[P] * 7, need - 1, None) == INVALID
    assert lib.fh_vocab_loss_grad(r, *[P] * 8, least - 1, None) == INVALID
    for i in range(7):  # x, w, targets, loss, row_loss (which may be null), lse, workspace
        for bad in (None, P + 2):
            if (i, bad) == (4, None):
                continue
            args = [P] * 7
            args[i] = bad
            assert lib.fh_vocab_loss_fwd(r, *args, need, None) == INVALID, (i, bad)
    for i in range(8):  # x, w, targets, lse, dloss, dx, dw (either of which may be null), workspace
        for bad in (None, P + 2):
            if bad is None and i in (5, 6):
                continue
            args = [P] * 8
            args[i] = bad
            assert lib.fh_vocab_loss_grad(r, *args, best, None) == INVALID, (i, bad)


def test_nothing_to_do_is_ok():
    lib = abi.lib()
    assert lib.fh_embedding_fwd(ctypes.byref(table(tokens=0)), None, None, None, None) == 0
    none = table(tokens=0)  # on top of itself: every row stays
    assert lib.fh_embedding_grad(ctypes.byref(none), None, None, P, P, None, 0, None) == 0
    r = ctypes.byref(loss())
    assert lib.fh_vocab_loss_grad(r, *[P] * 5, None, None, P, 0, None) == 0
    assert lib.fh_vocab_loss_grad(ctypes.byref(loss(tokens=0)), *[None] * 5, P, None, None, 0, None) == 0


def test_workspaces_grow_with_what_they_hold():
    lib = abi.lib()
    small, wide = loss(tokens=512, vocab=100000), loss(tokens=1 << 16, vocab=131072, dim=4096, x_stride=4096, w_stride=4096)
    for g in (small, wide):
        assert lib.fh_vocab_loss_grad_least(ctypes.byref(g)) < lib.fh_vocab_loss_grad_workspace(ctypes.byref(g))
    # the derivatives of 2^16 rows and the whole vocabulary would be 16 GiB
    assert lib.fh_vocab_loss_grad_workspace(ctypes.byref(wide)) < 3 << 30


def test_reference_gradients_are_differences():
    rng = np.random.default_rng(5)
    x, w = rng.normal(size=(5, 8)), rng.normal(size=(7, 8))
    targets = np.array([3, -1, 0, 7, 6])
    for mean in (True, False):
        (dx, _), (dw, _) = ref.Loss(x, w, targets, mean, BF16).gradients(1.5)
        for a, got in ((x, dx), (w, dw)):
            for i in np.ndindex(a.shape):
                at, h = a[i], 1e-5
                a[i] = at + h
                high = ref.Loss(x, w, targets, mean, BF16).loss
                a[i] = at - h
                low = ref.Loss(x, w, targets, mean, BF16).loss
                a[i] = at
                assert abs(1.5 * (high - low) / (2 * h) - got[i]) < 1e-8
    table_, ids, dout = rng.normal(size=(6, 3)), np.array([2, 2, 9, 0, -1]), rng.normal(size=(5, 3))
    got, _ = ref.embed_grad(dout, ids, 6, 0.5, None, F32)
    for i in np.ndindex(table_.shape):
        step = np.zeros_like(table_)
        step[i] = 1.0
        assert abs((ref.embed(step, ids, 0.5, F32)[0] * dout).sum() - got[i]) < 1e-12  # linear in the table
