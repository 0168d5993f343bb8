"""Softmax cross entropy over a vocabulary and its gradients against float64 (tests/language_ref.py, which derives the bounds)."""
import ctypes

import numpy as np
import pytest

import language_ref as ref
from frame_hip import synth

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 2, 3
KEEP = 0x5a5a
NAN = {F16: 0x7e00, BF16: 0x7fc0}


def say(msg):
    print(f"[case] {msg}", flush=True)


class Loss:
    def __init__(self, hip, dtype, tokens, vocab, dim, outside=0.0, mean=1, pad=0, loss_dtype=F32, seed=1, std=1.5, learned=True):
        """pad: elements between the rows of x and w (dx and dw) that belong to none. Rows without a target hold NaN."""
        self.hip, self.dtype, self.tokens, self.vocab, self.dim = hip, dtype, tokens, vocab, dim
        self.mean, self.ld, self.loss_dtype = mean, dim + pad, loss_dtype
        rng = np.random.default_rng(seed)
        self.targets = rng.integers(0, vocab, tokens).astype(np.int32)
        bad = rng.random(tokens) < outside
        self.targets[bad] = rng.choice([-1, -100, vocab, 2 ** 31 - 1, -2 ** 31], bad.sum())
        self.counted = (self.targets >= 0) & (self.targets < vocab)
        w = rng.normal(size=(vocab, dim)) * std / np.sqrt(dim)
        x = rng.normal(size=(tokens, dim))
        if learned:  # the target's logit raised, by 0 to 9
            mine = w[np.where(self.counted, self.targets, 0)]
            x += mine * (9 * rng.random((tokens, 1)) / np.maximum((mine ** 2).sum(1, keepdims=True), 1e-3))
        self.x, self.w = (synth.to_storage(a.astype(np.float32), dtype) for a in (x, w))
        self.x[~self.counted] = NAN[dtype]

    def want(self):
        return ref.Loss(ref.values(self.x, self.dtype), ref.values(self.w, self.dtype), self.targets.astype(np.int64), self.mean, self.dtype,
                        self.loss_dtype)

    def geom(self):
        return self.hip.VocabLoss(dtype=self.dtype, loss_dtype=self.loss_dtype, mean=self.mean, tokens=self.tokens, vocab=self.vocab,
                                  dim=self.dim, x_stride=self.ld, w_stride=self.ld)

    def up(self, a):
        whole = np.full((max(a.shape[0], 1), self.ld), KEEP, np.uint16)
        whole[:a.shape[0], :self.dim] = a
        return self.hip.to_device(whole)

    def down(self, buf, rows):
        whole = buf.download((rows, self.ld), np.uint16)
        assert (whole[:, self.dim:] == KEEP).all(), "the columns between rows were written"
        return whole[:, :self.dim]

    def room(self, need):
        return self.hip.to_device(np.full(need // 4 + 64, np.nan, np.float32))

    def intact(self, ws, need):
        assert np.isnan(ws.download((need // 4 + 64,), np.float32)[need // 4:]).all(), "written behind the workspace"

    def scalar(self, value):
        return self.hip.to_device(synth.to_storage(np.full(1, value, np.float32), self.loss_dtype))

    def forward(self, rows=True, stream=None):
        hip, lib, n = self.hip, self.hip.lib(), self.tokens
        x, w, t = self.up(self.x), self.up(self.w), hip.to_device(self.targets if n else np.zeros(1, np.int32))
        loss, row, lse = self.scalar(-7.0), hip.to_device(np.full(n + 1, -7, np.float32)), hip.to_device(np.full(n + 1, -7, np.float32))
        g = self.geom()
        need = lib.fh_vocab_loss_workspace(ctypes.byref(g))
        ws = self.room(need)
        hip.check(lib.fh_vocab_loss_fwd(ctypes.byref(g), x.value, w.value, t.value, loss.value, row.value if rows else None, lse.value,
                                        ws.value, need, stream))
        hip.check(lib.fh_device_synchronize())
        self.intact(ws, need)
        row, lse = (b.download((n + 1,), np.float32) for b in (row, lse))
        assert row[n] == -7 and lse[n] == -7
        loss = synth.to_float(loss.download((1,), np.float32 if self.loss_dtype == F32 else np.uint16), self.loss_dtype)
        return float(loss[0]), row[:n], lse[:n]

    def backward(self, lse, dloss=1.0, which="xw", columns=None, stream=None):
        """columns: of a piece, by the workspace that is given."""
        hip, lib, n = self.hip, self.hip.lib(), self.tokens
        x, w, t = self.up(self.x), self.up(self.w), hip.to_device(self.targets if n else np.zeros(1, np.int32))
        lse, d = hip.to_device(np.append(lse, 0).astype(np.float32)), self.scalar(dloss)
        dx, dw = (self.up(np.full((r, self.dim), KEEP, np.uint16)) for r in (n, self.vocab))
        g = self.geom()
        need = lib.fh_vocab_loss_grad_workspace(ctypes.byref(g))
        if columns is not None:
            need = lib.fh_vocab_loss_grad_least(ctypes.byref(g)) + (columns - 256) * 2 * (-(-n // 256) * 256)
        ws = self.room(need)
        hip.check(lib.fh_vocab_loss_grad(ctypes.byref(g), x.value, w.value, t.value, lse.value, d.value, dx.value if "x" in which else None,
                                         dw.value if "w" in which else None, ws.value, need, stream))
        hip.check(lib.fh_device_synchronize())
        self.intact(ws, need)
        return self.down(dx, n), self.down(dw, self.vocab)

    def check(self, dloss=1.0, columns=None):
        want = self.want()
        loss, row, lse = self.forward()
        ref.check(lse.astype(np.float64), want.lse, want.lse_tol, "lse")
        ref.check(row.astype(np.float64), want.row, want.row_tol, "row_loss")
        assert abs(loss - want.loss) <= want.loss_tol, (loss, want.loss, want.loss_tol)
        dx, dw = self.backward(lse, dloss, columns=columns)
        for name, got, (w, tol) in zip(("dx", "dw"), (dx, dw), want.gradients(dloss)):
            ref.check(ref.values(got, self.dtype), w, tol, name)
        return loss, row, lse, dx, dw


SHAPES = [  # tokens, vocab, dim, share of rows without a target, mean, pad
    (1, 1, 8, 0.0, 1, 0), (1, 2, 8, 0.0, 0, 0), (2, 7, 16, 0.0, 1, 8), (1, 5003, 64, 0.0, 1, 0), (15, 63, 40, 0.3, 1, 0),
    (64, 64, 64, 0.0, 0, 0), (65, 65, 72, 0.0, 1, 0), (33, 257, 24, 0.5, 0, 16), (130, 1000, 128, 0.1, 1, 0), (256, 256, 256, 0.0, 1, 0),
    (257, 511, 264, 0.0, 1, 0), (333, 2003, 200, 0.4, 1, 8), (700, 300, 96, 0.2, 0, 0), (16, 3001, 1000, 0.0, 1, 0), (600, 1500, 512, 0.0, 1, 0),
    (1100, 1025, 136, 0.9, 1, 0),
    # the larger tiles: of logits, of dx and dw, of both, and few rows of many columns
    (2048, 8197, 40, 0.1, 1, 0), (2100, 2051, 6152, 0.3, 1, 0), (300, 11003, 24, 0.0, 1, 0), (800, 900, 5000, 0.0, 1, 0),
    (60, 40000, 16, 0.0, 1, 0), (5, 70, 33000, 0.0, 1, 0),
    # where another kernel takes over: the joins' rows, the rows that workgroups list themselves, runs of the list
    (16, 300, 24, 0.3, 1, 0), (17, 300, 24, 0.3, 1, 0), (64, 300, 24, 0.3, 1, 0), (1024, 130, 24, 0.3, 1, 0), (1025, 130, 24, 0.3, 1, 0),
    (2049, 70, 16, 0.5, 0, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_and_gradients(hip, shape, dtype):
    tokens, vocab, dim, outside, mean, pad = shape
    say(f"vocabulary loss {shape} dtype={dtype}")
    Loss(hip, dtype, tokens, vocab, dim, outside, mean, pad).check(2.5)


@pytest.mark.parametrize("columns", [256, 512, 768, 2048])
def test_pieces_of_the_vocabulary(hip, columns):
    say(f"pieces of {columns} columns")
    Loss(hip, BF16, 300, 2003, 136, 0.2).check(1.0, columns)


@pytest.mark.parametrize("columns", [None, 256])
@pytest.mark.parametrize("shape", [(511, 900, 72, 0.4, 1, 8), (512, 900, 64, 0.4, 0, 0), (513, 900, 72, 0.4, 1, 0), (20, 8192, 1024, 0.2, 1, 0),
                                   (20, 8193, 1024, 0.2, 1, 0), (512, 700, 64, 2.0, 1, 0)], ids=str)
def test_where_fewer_launches_take_over(hip, shape, columns):
    say(f"rows listed beside the derivatives, both gradients in one launch: {shape}, pieces of {columns} columns")
    tokens, vocab, dim, outside, mean, pad = shape
    Loss(hip, BF16, tokens, vocab, dim, outside, mean, pad).check(1.5, columns)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_loss_in_the_tensors_type(hip, dtype):
    say(f"loss and its gradient as one value of dtype {dtype}")
    Loss(hip, dtype, 100, 700, 64, 0.1, loss_dtype=dtype).check(0.5)


@pytest.mark.parametrize("dloss", [2.0 ** -20, 2.0 ** 15, 0.0, -3.0])
def test_size_of_the_losses_gradient(hip, dloss):
    """f16: the derivatives keep their bits whatever the loss' gradient is; only the results are rounded after it."""
    say(f"dloss {dloss}")
    Loss(hip, F16, 200, 900, 64).check(dloss)


def test_rows_without_a_target_only(hip):
    say("no row has a target: a loss of 0, gradients of zeros")
    p = Loss(hip, BF16, 70, 300, 64, 2.0)
    assert not p.counted.any()
    loss, row, lse = p.forward()
    assert loss == 0.0 and not row.any() and not lse.any()
    dx, dw = p.backward(lse, float("nan"))
    assert not dx.any() and not dw.any()


def test_no_tokens(hip):
    say("no tokens")
    p = Loss(hip, BF16, 0, 300, 64)
    loss, _, _ = p.forward()
    assert loss == 0.0
    _, dw = p.backward(np.zeros(0))
    assert not dw.any()


def test_a_single_row_with_a_target_among_many(hip):
    say("one of 900 rows has a target")
    p = Loss(hip, BF16, 900, 400, 64, 2.0)
    p.targets[611], p.counted[611] = 399, True
    p.x[611] = synth.tensor(3, (64,), BF16, "normal")
    p.check()


def test_one_gradient_alone(hip):
    say("dx alone, dw alone")
    p = Loss(hip, BF16, 130, 600, 72, 0.1)
    _, _, lse, dx, dw = p.check()
    only_x, kept = p.backward(lse, which="x")
    assert np.array_equal(only_x, dx) and (kept == KEEP).all()
    kept, only_w = p.backward(lse, which="w")
    assert np.array_equal(only_w, dw) and (kept == KEEP).all()


def test_no_row_losses(hip):
    say("row_loss is NULL")
    p = Loss(hip, BF16, 100, 300, 64, 0.1)
    loss, _, lse = p.forward()
    again, untouched, lse2 = p.forward(rows=False)
    assert again == loss and np.array_equal(lse, lse2) and (untouched == -7).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_logits(hip, dtype):
    """Logits up to hundreds: one token takes it all, most others' probabilities are zero in 32 bits."""
    say(f"large logits dtype={dtype}")
    Loss(hip, dtype, 90, 800, 64, std=60.0, learned=False).check()


@pytest.mark.parametrize("shift", [-800.0, -150.0, 150.0, 800.0])
def test_logits_far_from_zero(hip, shift):
    """Exponentials of the logits themselves are zero or infinite in 32 bits."""
    say(f"logits around {shift}")
    p = Loss(hip, BF16, 70, 1000, 64)
    p.x[:, 0] = synth.to_storage(np.full(1, shift, np.float32), BF16)[0]
    p.w[:, 0] = 0x3f80  # 1.0
    p.check()


def test_every_logit_alike(hip):
    say("logits all zero: log(vocab), exact thirds")
    p = Loss(hip, BF16, 40, 3, 8)
    p.w[:] = 0
    loss, row, lse = p.forward()
    assert np.abs(lse - np.log(3)).max() < 2e-7 and np.abs(row - np.log(3)).max() < 2e-7 and abs(loss - np.log(3)) < 2e-7
    p.check()


def test_values_that_are_not_finite(hip):
    """A NaN in a row of x reaches that row's loss and dx and all of dw; one in a row of w every row's loss."""
    say("NaN in x, in w, infinite logits")
    p = Loss(hip, BF16, 70, 300, 64)
    _, _, lse0 = p.forward()
    p.x[5, 3] = NAN[BF16]
    loss, row, lse = p.forward()
    assert np.isnan(loss) and np.isnan(row[5]) and np.isnan(lse[5])
    others = np.arange(70) != 5
    assert np.array_equal(lse[others], lse0[others])
    dx, dw = (ref.values(a, BF16) for a in p.backward(lse))
    assert np.isnan(dx[5]).all() and np.isfinite(dx[others]).all() and np.isnan(dw).all()
    p = Loss(hip, BF16, 70, 300, 64)
    p.w[299, 63] = NAN[BF16]
    loss, row, lse = p.forward()
    assert np.isnan(loss) and np.isnan(row).all()
    # a logit of -infinity is a token of probability zero; it is nobody's target
    p = Loss(hip, BF16, 70, 300, 64)
    p.targets[p.targets == 299] = 0
    p.x[:, 0] = np.uint16(0x3f80)  # 1.0
    p.w[:, 0] = 0
    p.w[299, 0] = np.uint16(0xff80)  # -infinity
    loss, row, lse = p.forward()
    q = Loss(hip, BF16, 70, 299, 64)
    q.targets, q.x, q.w = p.targets, p.x, p.w[:299]
    want = q.want()
    ref.check(lse.astype(np.float64), want.lse, want.lse_tol, "lse")
    assert abs(loss - want.loss) <= want.loss_tol


def test_deterministic(hip):
    say("two calls give the same bits")
    p = Loss(hip, F16, 333, 2003, 200, 0.3)
    first, second = p.forward(), p.forward()
    assert first[0] == second[0] and all(np.array_equal(a, b) for a, b in zip(first[1:], second[1:]))
    for a, b in zip(p.backward(first[2]), p.backward(first[2])):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("n", [300, 1100])
def test_captured_and_replayed(hip, n):
    say("loss and gradients captured, targets changed between the replays")
    p = Loss(hip, BF16, n, 1300, 136, 0.2)
    p.x[~p.counted] = 0
    lib, g = hip.lib(), p.geom()
    r = ctypes.byref(g)
    need, need_grad = lib.fh_vocab_loss_workspace(r), lib.fh_vocab_loss_grad_workspace(r)
    x, w, t, d = p.up(p.x), p.up(p.w), hip.to_device(p.targets), p.scalar(1.0)
    loss, lse, dx, dw = p.scalar(0.0), hip.DeviceBuffer(4 * n), p.up(p.x), p.up(p.w)
    ws, stream, graph = hip.DeviceBuffer(max(need, need_grad)), hip.Stream(), ctypes.c_void_p()
    hip.check(lib.fh_device_synchronize())
    hip.check(lib.fh_graph_begin_capture(stream.ptr))
    hip.check(lib.fh_vocab_loss_fwd(r, x.value, w.value, t.value, loss.value, None, lse.value, ws.value, need, stream.ptr))
    hip.check(lib.fh_vocab_loss_grad(r, x.value, w.value, t.value, lse.value, d.value, dx.value, dw.value, ws.value, need_grad, stream.ptr))
    hip.check(lib.fh_graph_end_capture(stream.ptr, 1, ctypes.byref(graph)))
    rng = np.random.default_rng(9)
    for replay in range(4):
        p.targets = np.where(rng.random(n) < 0.3 * replay, -1, rng.integers(0, 1300, n)).astype(np.int32)
        p.counted = p.targets >= 0
        t.upload(p.targets)
        hip.check(lib.fh_graph_launch(graph, stream.ptr))
        stream.synchronize()
        want = p.forward()
        assert loss.download((1,), np.float32)[0] == np.float32(want[0]), replay
        assert np.array_equal(lse.download((n,), np.float32), want[2]), replay
        want = p.backward(want[2])
        assert np.array_equal(p.down(dx, n), want[0]) and np.array_equal(p.down(dw, 1300), want[1]), replay
    hip.check(lib.fh_graph_destroy(graph))


def test_two_streams_at_once(hip):
    say("two calls at once, each with its workspace")
    lib, runs = hip.lib(), []
    for i in range(2):
        p = Loss(hip, BF16, 500, 1500, 128, 0.1, seed=60 + i)
        lse, g = p.forward()[2], p.geom()
        need = lib.fh_vocab_loss_grad_workspace(ctypes.byref(g))
        runs.append((p, lse, g, need, [p.up(p.x), p.up(p.w), hip.to_device(p.targets), hip.to_device(lse), p.scalar(1.0), p.up(p.x), p.up(p.w),
                                       hip.DeviceBuffer(need)], hip.Stream()))
    hip.check(lib.fh_device_synchronize())
    for _ in range(3):
        for p, lse, g, need, bufs, st in runs:
            hip.check(lib.fh_vocab_loss_grad(ctypes.byref(g), *[b.value for b in bufs], need, st.ptr))
    for p, lse, g, need, bufs, st in runs:
        st.synchronize()
        dx, dw = p.backward(lse)
        assert np.array_equal(p.down(bufs[5], 500), dx) and np.array_equal(p.down(bufs[6], 1500), dw)
