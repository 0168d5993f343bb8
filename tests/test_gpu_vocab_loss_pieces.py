"""The vocabulary loss' gradients where the best workspace holds a piece of the vocabulary and dx' sums over a piece are split among workgroups,
tensors whose rows lie differently far apart, and offsets past 32 bits."""
import ctypes

import numpy as np
import pytest

from frame_hip import synth
from test_gpu_vocab_loss import KEEP, Loss, say

pytestmark = pytest.mark.gpu
F16, BF16 = 2, 3


@pytest.mark.parametrize("case", [
    # two pieces, four splits of 256 x 256 tiles: one stage is left to the last piece's, and none to three of its splits
    (BF16, 4096, 16400, 1024, 0.1),
    # eight splits of 128 x 128 tiles, four of them empty in the last piece; uneven columns
    (F16, 2048, 32800, 512, 0.2),
    # 64 x 64 tiles, rows listed by workgroups, the last piece's two products in one launch, uneven depth
    (BF16, 1000, 66000, 264, 0.1),
    # up to 512 rows, listed and gathered in the first piece's derivatives; splits of the last piece without a stage
    (BF16, 100, 262700, 72, 0.3),
], ids=str)
def test_split_sums_over_several_pieces(hip, case):
    dtype, tokens, vocab, dim, outside = case
    say(f"several pieces and splits at the best workspace: {case}")
    p = Loss(hip, dtype, tokens, vocab, dim, outside)
    p.targets[-1], p.counted[-1] = vocab - 1, True  # a target in the last piece
    p.x[-1] = synth.tensor(3, (dim,), dtype, "normal")
    p.check(2.0)


def strided(hip, a, ld):
    whole = np.full((a.shape[0], ld), KEEP, np.uint16)
    whole[:, :a.shape[1]] = a
    return hip.to_device(whole)


@pytest.mark.parametrize("strides", [(80, 144), (200, 72), (72, 2048)], ids=str)
@pytest.mark.parametrize("tokens", [90, 700, 1500])
def test_strides_of_x_and_w_are_their_own(hip, tokens, strides):
    say(f"rows of x and w {strides} elements apart, {tokens} tokens")
    vocab, dim, lib = 1300, 72, hip.lib()
    p = Loss(hip, BF16, tokens, vocab, dim, 0.2)
    loss0, row0, lse0 = p.check(2.0)[:3]
    dx0, dw0 = p.backward(lse0, 2.0)
    g = p.geom()
    g.x_stride, g.w_stride = strides
    r = ctypes.byref(g)
    x, w, t = strided(hip, p.x, strides[0]), strided(hip, p.w, strides[1]), hip.to_device(p.targets)
    dx, dw = strided(hip, np.full_like(p.x, 1), strides[0]), strided(hip, np.full_like(p.w, 1), strides[1])
    loss, lse, d = p.scalar(0.0), hip.DeviceBuffer(4 * tokens), p.scalar(2.0)
    need, need_grad = lib.fh_vocab_loss_workspace(r), lib.fh_vocab_loss_grad_workspace(r)
    ws = hip.DeviceBuffer(max(need, need_grad))
    hip.check(lib.fh_vocab_loss_fwd(r, x.value, w.value, t.value, loss.value, None, lse.value, ws.value, need, None))
    hip.check(lib.fh_vocab_loss_grad(r, x.value, w.value, t.value, lse.value, d.value, dx.value, dw.value, ws.value, need_grad, None))
    hip.check(lib.fh_device_synchronize())
    assert loss.download((1,), np.float32)[0] == np.float32(loss0) and np.array_equal(lse.download((tokens,), np.float32), lse0)
    for buf, n, ld, want in ((dx, tokens, strides[0], dx0), (dw, vocab, strides[1], dw0)):
        whole = buf.download((n, ld), np.uint16)
        assert np.array_equal(whole[:, :dim], want) and (whole[:, dim:] == KEEP).all()


def test_offsets_past_32_bits(hip):
    """Rows of w and dw 2^22 - 8 elements apart: 600 of them span 5 GB. Only their first 64 columns are written or read."""
    say("rows of w 8 MB apart, 600 of them")
    tokens, vocab, dim, ld, lib = 300, 600, 64, 2 ** 22 - 8, hip.lib()
    p = Loss(hip, BF16, tokens, vocab, dim, 0.1)
    loss0, _, lse0 = p.check()[:3]
    dx0, dw0 = p.backward(lse0)
    g = p.geom()
    g.w_stride = ld
    r = ctypes.byref(g)
    x, t, near = p.up(p.x), hip.to_device(p.targets), p.up(p.w)
    w, dw = (hip.DeviceBuffer(2 * (ld * (vocab - 1) + dim)) for _ in "ab")
    dx, loss, lse, d = p.up(p.x), p.scalar(0.0), hip.DeviceBuffer(4 * tokens), p.scalar(1.0)
    need, need_grad = lib.fh_vocab_loss_workspace(r), lib.fh_vocab_loss_grad_workspace(r)
    ws, back = hip.DeviceBuffer(max(need, need_grad)), p.up(p.w)
    row = 2 * dim
    hip.check(lib.fh_copy2d(w.value, 2 * ld, near.value, row, row, vocab, None))
    hip.check(lib.fh_vocab_loss_fwd(r, x.value, w.value, t.value, loss.value, None, lse.value, ws.value, need, None))
    hip.check(lib.fh_vocab_loss_grad(r, x.value, w.value, t.value, lse.value, d.value, dx.value, dw.value, ws.value, need_grad, None))
    hip.check(lib.fh_copy2d(back.value, row, dw.value, 2 * ld, row, vocab, None))
    hip.check(lib.fh_device_synchronize())
    assert loss.download((1,), np.float32)[0] == np.float32(loss0) and np.array_equal(lse.download((tokens,), np.float32), lse0)
    assert np.array_equal(p.down(dx, tokens), dx0) and np.array_equal(p.down(back, vocab), dw0)
