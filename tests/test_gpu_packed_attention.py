"""Attention over packed sequences, its gradients, the paged cache and attention over it, against float64 (tests/attention_ref.py,
which derives the bounds)."""
import ctypes

import numpy as np
import pytest

import attention_ref as ref
from frame_hip import synth

pytestmark = pytest.mark.gpu

F16, BF16 = 2, 3
E4M3 = 16
NAN = {F16: 0x7e00, BF16: 0x7fc0}
KEEP = 0x5a5a  # what rows that a call may not write hold before and after


def say(msg):
    print(f"[case] {msg}", flush=True)


def starts(lens, first=0):
    return np.cumsum([first] + list(lens)).astype(np.int32)


class Packed:
    """Packed tensors on the device: separate ones, or (fused) columns of one buffer with 8 values between rows that belong to none."""

    def __init__(self, hip, dtype, lens, heads, kv_heads, dh, causal, first=0, behind=0, fused=False, seed=1, std=1.0, scale=None):
        self.hip, self.dtype, self.lens, self.heads, self.kv_heads, self.dh = hip, dtype, list(lens), heads, kv_heads, dh
        self.cu = starts(lens, first)
        self.rows = int(self.cu[-1]) + behind
        self.scale = float(np.float32(1.0 / np.sqrt(dh) if scale is None else scale))
        self.causal = causal
        widths = [heads * dh, kv_heads * dh, kv_heads * dh]
        self.inside = np.zeros(self.rows, bool)
        self.inside[self.cu[0]:self.cu[-1]] = True
        self.x = {}
        for i, (name, w) in enumerate(zip("qkv", widths)):
            self.x[name] = synth.tensor(seed + i, (self.rows, w), dtype, "normal", std)
            self.x[name][~self.inside] = NAN[dtype]  # rows of no sequence are not read
        self.x["dout"] = synth.tensor(seed + 5, (self.rows, widths[0]), dtype, "normal")
        self.x["dout"][~self.inside] = NAN[dtype]
        self.ld = [sum(widths) + 8] * 3 if fused else widths
        self.at = [0, widths[0], widths[0] + widths[1]] if fused else [0, 0, 0]
        self.widths, self.fused = widths, fused

    def upload(self, arrays):
        """Three tensors q, k, v (or their gradients' room) -> buffers and addresses."""
        if not self.fused:
            bufs = [self.hip.to_device(a) for a in arrays]
            return bufs, [b.value for b in bufs]
        whole = np.full((self.rows, self.ld[0]), KEEP, np.uint16)
        for a, at, w in zip(arrays, self.at, self.widths):
            whole[:, at:at + w] = a
        buf = self.hip.to_device(whole)
        return [buf], [buf.value + 2 * at for at in self.at]

    def download(self, bufs):
        if not self.fused:
            return [b.download((self.rows, w), np.uint16) for b, w in zip(bufs, self.widths)]
        whole = bufs[0].download((self.rows, self.ld[0]), np.uint16)
        assert (whole[:, sum(self.widths):] == KEEP).all(), "the columns between rows were written"
        return [whole[:, at:at + w] for at, w in zip(self.at, self.widths)]

    def geom(self):
        return self.hip.PackedAttention(dtype=self.dtype, causal=self.causal, tokens=self.rows, batch=len(self.lens),
                                        heads=self.heads, kv_heads=self.kv_heads, dh=self.dh, q_stride=self.ld[0],
                                        k_stride=self.ld[1], v_stride=self.ld[2], out_stride=self.widths[0], scale=self.scale)

    def heads_of(self):
        """(rows, head, key head, q, k, v, dout, mask) per sequence and head, in float64."""
        group = self.heads // self.kv_heads
        for b, n in enumerate(self.lens):
            rows = slice(self.cu[b], self.cu[b + 1])
            seen = np.tril(np.ones((n, n), bool)) if self.causal else np.ones((n, n), bool)
            for h in range(self.heads if n else 0):
                j = h // group
                mine, shared = slice(h * self.dh, (h + 1) * self.dh), slice(j * self.dh, (j + 1) * self.dh)
                yield (rows, h, mine, shared, *(ref.values(self.x[t][rows, c], self.dtype)
                                                for t, c in (("q", mine), ("k", shared), ("v", shared), ("dout", mine))), seen)

    def want(self):
        out, tol = np.zeros((2, self.rows, self.widths[0]))
        lse, lse_tol = np.zeros((2, self.rows, self.heads))
        for rows, h, mine, _, q, k, v, _, seen in self.heads_of():
            out[rows, mine], tol[rows, mine], _, lse[rows, h], lse_tol[rows, h] = ref.attend(q, k, v, seen, self.scale, self.dtype)
        return out, tol, lse, lse_tol

    def forward(self, stream=None, keep=None):
        hip = self.hip
        bufs, ptrs = self.upload([self.x[t] for t in "qkv"])
        cu = hip.to_device(self.cu)
        out = hip.to_device(np.full((self.rows, self.widths[0]), KEEP, np.uint16))
        lse = hip.to_device(np.full((self.rows, self.heads), -7.0, np.float32))
        g = self.geom()
        hip.check(hip.lib().fh_attention_packed_fwd(ctypes.byref(g), *ptrs, cu.value, out.value, lse.value, stream))
        hip.check(hip.lib().fh_device_synchronize())
        return out.download((self.rows, self.widths[0]), np.uint16), lse.download((self.rows, self.heads), np.float32)

    def check_forward(self, out, lse, what):
        assert (out[~self.inside] == KEEP).all() and (lse[~self.inside] == -7.0).all(), "rows of no sequence were written"
        want, tol, want_lse, lse_tol = self.want()
        i = self.inside
        ref.check(ref.values(out, self.dtype)[i], want[i], tol[i], what + " out")
        ref.check(lse.astype(np.float64)[i], want_lse[i], lse_tol[i], what + " lse")

    def backward(self, out_bits, lse):
        hip = self.hip
        bufs, ptrs = self.upload([self.x[t] for t in "qkv"])
        cu, out, dout, stats = (hip.to_device(a) for a in (self.cu, out_bits, self.x["dout"], lse))
        grads, gptrs = self.upload([np.full((self.rows, w), KEEP, np.uint16) for w in self.widths])
        g = self.geom()
        need = hip.lib().fh_attention_packed_grad_workspace(ctypes.byref(g))
        ws = hip.to_device(np.full(need // 4, np.nan, np.float32))
        hip.check(hip.lib().fh_attention_packed_grad(ctypes.byref(g), *ptrs, cu.value, out.value, stats.value, dout.value, *gptrs,
                                                     ws.value, need, None))
        hip.check(hip.lib().fh_device_synchronize())
        return self.download(grads)

    def want_grads(self):
        total = [np.zeros((self.rows, w)) for w in self.widths]
        tol = [np.zeros((self.rows, w)) for w in self.widths]
        for rows, h, mine, shared, q, k, v, dout, seen in self.heads_of():
            out, _, p, _, _ = ref.attend(q, k, v, seen, self.scale, self.dtype)
            for i, (g, t) in enumerate(ref.gradients(q, k, v, dout, out, p, self.scale, self.dtype)):
                at = (rows, mine if i == 0 else shared)
                total[i][at] += g
                tol[i][at] += t
        return total, tol

    def stored_forward(self):
        """out rounded to the storage type and lse as fp32, from float64; NaN in rows of no sequence."""
        out, _, lse, _ = self.want()
        bits = synth.to_storage(out.astype(np.float32), self.dtype)
        bits[~self.inside] = NAN[self.dtype]
        lse = lse.astype(np.float32)
        lse[~self.inside] = np.nan
        return bits, lse


# dtype, lengths, heads, kv_heads, dh, causal, first row, rows behind, fused
PACKED = [
    (BF16, [64], 1, 1, 64, 1, 0, 0, False),
    (BF16, [1], 4, 4, 64, 1, 0, 0, False),                          # one token
    (F16, [0, 1, 63, 0, 64, 65, 0], 4, 2, 64, 1, 0, 3, True),       # empty sequences at both ends, block edges
    (BF16, [127, 128, 129, 2], 6, 2, 128, 1, 5, 2, True),           # group of 3: tiles cross tokens
    (BF16, [200, 33, 301], 8, 1, 64, 1, 0, 0, False),               # all heads share one key head
    (F16, [130, 70], 5, 5, 128, 0, 0, 1, False),                    # not causal
    (BF16, [257], 2, 2, 80, 1, 0, 0, True),                         # head dims between tile sizes
    (F16, [97, 31], 3, 1, 96, 0, 3, 0, False),
    (BF16, [90, 5, 18], 2, 1, 8, 1, 0, 0, False),
    (F16, [40, 77], 4, 4, 40, 1, 0, 6, True),
    (BF16, [1] * 70 + [3, 0, 200] + [2] * 70, 2, 1, 64, 1, 0, 0, False),  # more than 64 sequences: the lookup's second step
    (BF16, [700, 45], 16, 2, 128, 1, 0, 0, True),
    (F16, [513], 14, 2, 64, 1, 0, 0, False),                        # group of 7
]


def packed_id(c):
    return f"{'f16' if c[0] == F16 else 'bf16'}-{len(c[1])}x{max(c[1])}-h{c[2]}k{c[3]}d{c[4]}{'c' if c[5] else ''}"


@pytest.mark.parametrize("case", PACKED, ids=packed_id)
def test_packed_forward(hip, case):
    say(f"packed forward {case}")
    p = Packed(hip, *case)
    p.check_forward(*p.forward(), "packed")


@pytest.mark.parametrize("case", PACKED, ids=packed_id)
def test_packed_gradients(hip, case):
    say(f"packed gradients {case}")
    p = Packed(hip, *case)
    out, lse = p.stored_forward()
    got = p.backward(out, lse)
    for name, g, total, tol in zip("qkv", got, *p.want_grads()):
        assert (g[~p.inside] == KEEP).all(), f"d{name}: rows of no sequence were written"
        ref.check(ref.values(g, p.dtype)[p.inside], total[p.inside], ref.rounded(total, tol, p.dtype)[p.inside], "d" + name)


@pytest.mark.parametrize("dtype,dh", [(BF16, 128), (F16, 64)])
def test_packed_gradients_of_single_tokens(hip, dtype, dh):
    # a softmax over one key has no derivative: dq and dk are zeros, not the noise of dp - D
    say(f"packed gradients of single tokens dtype={dtype} dh={dh}")
    p = Packed(hip, dtype, [1, 1, 0, 1], 4, 2, dh, 1)
    dq, dk, dv = p.backward(*p.forward())
    assert not (dq & 0x7fff).any() and not (dk & 0x7fff).any()
    total, tol = p.want_grads()
    ref.check(ref.values(dv, dtype), total[2], ref.rounded(total[2], tol[2], dtype), "dv")


@pytest.mark.parametrize("std,scale", [(4.0, 0.125), (1.0, 1e-6), (0.01, 3.0)])
def test_packed_score_ranges(hip, std, scale):
    # wide scores (most probabilities vanish, the running maximum moves often), all but equal ones, tiny inputs
    say(f"packed ranges std={std} scale={scale}")
    p = Packed(hip, BF16, [300, 41], 4, 2, 64, 1, std=std, scale=scale)
    p.check_forward(*p.forward(), "packed")


def test_packed_rising_scores(hip):
    # every block's scores exceed the last block's by far: each one scales the sums again
    say("packed rising scores")
    p = Packed(hip, BF16, [400], 1, 1, 64, 0)
    ramp = np.zeros((400, 64), np.float32)
    ramp[:, 0] = np.arange(400) // 16 * 8
    p.x["k"] = synth.to_storage(ramp, BF16)
    one = np.zeros((400, 64), np.float32)
    one[:, 0] = 4.0
    p.x["q"] = synth.to_storage(one, BF16)
    p.check_forward(*p.forward(), "rising")


def test_packed_lse_is_optional_and_other_streams(hip):
    say("packed without lse, on a stream")
    p = Packed(hip, BF16, [100, 3], 4, 2, 64, 1)
    want, _ = p.forward()
    bufs, ptrs = p.upload([p.x[t] for t in "qkv"])
    cu, out, g = hip.to_device(p.cu), hip.to_device(np.zeros_like(want)), p.geom()
    stream = hip.Stream()
    hip.check(hip.lib().fh_attention_packed_fwd(ctypes.byref(g), *ptrs, cu.value, out.value, None, stream.ptr))
    stream.synchronize()
    assert np.array_equal(out.download(want.shape, np.uint16), want)


def test_packed_not_finite_values_stay_in_their_sequence(hip):
    # a sequence that holds NaN and infinities next to ones that do not: the others are what they are without it
    say("packed NaN isolation")
    p = Packed(hip, BF16, [70, 50, 130], 4, 2, 64, 1)
    bad = slice(p.cu[1], p.cu[2])
    for t in "qkv":
        p.x[t][bad] = NAN[BF16]
    p.x["v"][p.cu[1] + 1] = 0x7f80  # +inf
    out, lse = p.forward()
    assert np.isnan(ref.values(out[bad], BF16)).all()
    clean = np.ones(p.rows, bool)
    clean[bad] = False
    want, tol, want_lse, lse_tol = p.want()
    ref.check(ref.values(out, BF16)[clean], want[clean], tol[clean], "out")
    ref.check(lse.astype(np.float64)[clean], want_lse[clean], lse_tol[clean], "lse")


INF = {F16: 0x7c00, BF16: 0x7f80}


@pytest.mark.parametrize("dtype,heads,kv_heads,dh", [(BF16, 4, 2, 64), (F16, 2, 2, 128), (BF16, 3, 1, 40)])
@pytest.mark.parametrize("t", [0, 5, 64, 130, 298])
def test_packed_not_finite_values_reach_the_rows_that_see_them(hip, dtype, heads, kv_heads, dh, t):
    check_not_finite(hip, dtype, heads, kv_heads, dh, t, [70, 300])


# batches of more tiles than CUs, which the kernels cut otherwise than small ones
MANY = [70, 300, 0, 1, 129] + [17, 64, 100, 95] * 15


@pytest.mark.parametrize("t", [5, 130])
@pytest.mark.parametrize("dtype,heads,kv_heads,dh", [(BF16, 16, 16, 64), (BF16, 32, 8, 128)])
def test_packed_not_finite_values_among_many_sequences(hip, dtype, heads, kv_heads, dh, t):
    check_not_finite(hip, dtype, heads, kv_heads, dh, t, MANY)


@pytest.mark.parametrize("case", [(BF16, MANY, 16, 16, 64, 1, 0, 5, True), (F16, MANY, 32, 8, 128, 1, 3, 0, False),
                                  (BF16, MANY, 16, 16, 80, 0, 0, 0, False), (F16, MANY, 28, 14, 40, 1, 0, 2, True)], ids=packed_id)
def test_packed_many_sequences(hip, case):
    say(f"packed, many sequences {case}")
    p = Packed(hip, *case)
    p.check_forward(*p.forward(), "many")
    got = p.backward(*p.stored_forward())
    for name, g, total, tol in zip("qkv", got, *p.want_grads()):
        assert (g[~p.inside] == KEEP).all(), f"d{name}: rows of no sequence were written"
        ref.check(ref.values(g, p.dtype)[p.inside], total[p.inside], ref.rounded(total, tol, p.dtype)[p.inside], "d" + name)


def check_not_finite(hip, dtype, heads, kv_heads, dh, t, lens):
    # token t of the second sequence holds values that are not finite, one tensor at a time: rows that do not see it keep every bit
    say(f"packed NaN at token {t}, {heads} heads over {kv_heads} of {dh}")
    p = Packed(hip, dtype, lens, heads, kv_heads, dh, 1)
    group, at = heads // kv_heads, int(p.cu[1]) + t
    clean_out, clean_lse = p.forward()
    clean = p.backward(clean_out, clean_lse)
    later = np.zeros(p.rows, bool)
    later[at:p.cu[2]] = True
    mine = np.arange(heads * dh) // dh < group  # the heads of key head 0
    value = lambda a: ref.values(a, dtype)

    def with_bad(name, row, col, bits):
        kept = p.x[name].copy()
        p.x[name][row, col] = bits
        out, lse = p.forward()
        grads = p.backward(out, lse)
        p.x[name] = kept
        return out, lse, grads

    def check(got, want, affected, test, what):
        assert np.array_equal(got[~affected], want[~affected]), what + ": changed where nothing sees the value"
        assert test(value(got[affected])).all(), what

    # a value: its column, and no score
    for bits, test in ((NAN[dtype], np.isnan), (INF[dtype], np.isposinf), (INF[dtype] | 0x8000, np.isneginf)):
        out, lse, grads = with_bad("v", at, 3, bits)
        check(out, clean_out, later[:, None] & mine & (np.arange(heads * dh) % dh == 3), test, "out of v")
        assert np.array_equal(lse, clean_lse)
        # (rows that see key t alone have a derivative of zero times its value)
        check(grads[0], clean[0], later[:, None] & mine, lambda y: ~np.isfinite(y), "dq of v")
    # infinities of both signs, the second one token on
    kept = p.x["v"].copy()
    p.x["v"][at, 3], p.x["v"][at + 1, 3] = INF[dtype], INF[dtype] | 0x8000
    out, _ = p.forward()
    p.x["v"] = kept
    assert np.isposinf(value(out[at:at + 1, 3])).all() and np.isnan(value(out[at + 1:p.cu[2], 3])).all()
    assert np.array_equal(out[:at], clean_out[:at]) and np.array_equal(out[p.cu[2]:], clean_out[p.cu[2]:])
    # a key: all of its rows' scores
    out, lse, grads = with_bad("k", at, 3, NAN[dtype])
    check(out, clean_out, later[:, None] & mine, np.isnan, "out of k")
    check(grads[0], clean[0], later[:, None] & mine, np.isnan, "dq of k")
    assert np.isnan(lse[at:p.cu[2], :group]).all() and np.array_equal(lse[:at], clean_lse[:at])
    # a row of q: itself, and the keys that it sees
    shared = np.arange(kv_heads * dh) < dh
    seen = np.zeros(p.rows, bool)
    seen[p.cu[1]:at + 1] = True
    this = np.zeros(p.rows, bool)
    this[at] = True
    first = np.arange(heads * dh) < dh
    out, lse, grads = with_bad("q", at, 3, NAN[dtype])
    check(out, clean_out, this[:, None] & first, np.isnan, "out of q")
    for i, rows, cols in ((0, this, first), (1, seen, shared), (2, seen, shared)):
        check(grads[i], clean[i], rows[:, None] & cols, np.isnan, f"d{'qkv'[i]} of q")
    # an output's gradient: its column of dv, all of dk
    kept = p.x["dout"].copy()
    p.x["dout"][at, 3] = NAN[dtype]
    grads = p.backward(clean_out, clean_lse)
    p.x["dout"] = kept
    for i, rows, cols in ((0, this, first), (1, seen, shared), (2, seen, shared & (np.arange(kv_heads * dh) % dh == 3))):
        check(grads[i], clean[i], rows[:, None] & cols, np.isnan, f"d{'qkv'[i]} of dout")


def test_packed_bad_lengths_stay_in_bounds(hip):
    # cu_seqlens out of range or decreasing: values are taken into [0, tokens] and no memory outside is touched
    say("packed lengths out of range")
    p = Packed(hip, BF16, [100, 60], 2, 2, 64, 1)
    want, _ = p.forward()
    p.cu = np.array([-5, 100, 1 << 30], np.int32)  # 0 .. 100 .. tokens
    got, _ = p.forward()
    assert np.array_equal(got, want)
    p.cu = np.array([100, 60, 160], np.int32)  # the first sequence is empty; what the second holds is its own affair
    got, lse = p.forward()
    assert (got[:60] == KEEP).all()


def test_packed_decreasing_lengths_stay_in_bounds(hip):
    # a sequence behind one that begins further on: slots of tiles then find the latter, whose tiles begin behind them. Causal rows 0 .. 9
    # are the same in both sequences that hold them, so every row is either right or untouched.
    say("packed decreasing lengths")
    p = Packed(hip, BF16, [500], 2, 2, 64, 1)
    want, lse = p.forward()
    grads = p.backward(want, lse)
    p.cu, p.lens = np.array([0, 500, 0, 10], np.int32), [500, 0, 10]
    got, _ = p.forward()
    right, untouched = (got == want).all(axis=1), (got == KEEP).all(axis=1)
    assert (right | untouched).all() and right[:128].all()
    dq = p.backward(want, lse)[0]
    right, untouched = (dq == grads[0]).all(axis=1), (dq == KEEP).all(axis=1)
    assert (right | untouched).all() and right[:128].all()


def test_packed_gradients_are_deterministic_and_replay(hip):
    say("packed forward and gradients captured and replayed")
    p = Packed(hip, BF16, [150, 0, 47], 4, 2, 64, 1, fused=True)
    lib = hip.lib()
    out_bits, lse_host = p.forward()
    want = p.backward(out_bits, lse_host)
    again = p.backward(out_bits, lse_host)
    assert all(np.array_equal(a, b) for a, b in zip(want, again))
    bufs, ptrs = p.upload([p.x[t] for t in "qkv"])
    cu, dout = hip.to_device(p.cu), hip.to_device(p.x["dout"])
    out, lse = hip.to_device(np.full_like(out_bits, KEEP)), hip.to_device(np.full_like(lse_host, -7.0))
    room = [np.full((p.rows, w), KEEP, np.uint16) for w in p.widths]
    grads, gptrs = p.upload(room)
    g = p.geom()
    need = lib.fh_attention_packed_grad_workspace(ctypes.byref(g))
    ws, stream, graph = hip.DeviceBuffer(need), hip.Stream(), ctypes.c_void_p()
    hip.check(lib.fh_graph_begin_capture(stream.ptr))
    hip.check(lib.fh_attention_packed_fwd(ctypes.byref(g), *ptrs, cu.value, out.value, lse.value, stream.ptr))
    hip.check(lib.fh_attention_packed_grad(ctypes.byref(g), *ptrs, cu.value, out.value, lse.value, dout.value, *gptrs, ws.value,
                                           need, stream.ptr))
    hip.check(lib.fh_graph_end_capture(stream.ptr, 1, ctypes.byref(graph)))
    for replay in range(4):
        blank = np.full((p.rows, p.ld[0]), KEEP, np.uint16)
        grads[0].upload(blank)
        out.upload(np.full_like(out_bits, KEEP))
        hip.check(lib.fh_graph_launch(graph, stream.ptr))
        stream.synchronize()
        for name, a, b in zip("qkv", p.download(grads), want):
            assert np.array_equal(a, b), f"replay {replay}: d{name}"
        assert np.array_equal(p.forward()[0], out_bits)  # eager work between the replays
    hip.check(lib.fh_graph_destroy(graph))


# ---- the paged cache --------------------------------------------------------------------------------------------

class Paged:
    def __init__(self, hip, dtype, cache_dtype, past, new, heads, kv_heads, dh, page, behind=0, seed=1, bad_page=None, spare=2):
        self.hip, self.dtype, self.cache_dtype = hip, dtype, cache_dtype
        self.past, self.new, self.heads, self.kv_heads, self.dh, self.page = list(past), list(new), heads, kv_heads, dh, page
        self.cached = np.array([a + b for a, b in zip(past, new)], np.int32)
        rng = np.random.default_rng(seed)
        used = [-(-int(max(n, 0)) // page) for n in self.cached]
        self.pages = sum(used) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(used), max(used + [1])), -1, np.int32)  # entries past a sequence's length name no page
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        if bad_page is not None:  # (sequence, place in its table, number): a page that does not exist
            self.table[bad_page[0], bad_page[1]] = bad_page[2]
        self.cu = starts(new)
        self.rows = int(self.cu[-1]) + behind
        self.k, self.v = (synth.tensor(seed + 20 + i, (self.rows, kv_heads * dh), dtype, "normal") for i in range(2))
        self.q = synth.tensor(seed + 22, (self.rows, heads * dh), dtype, "normal")
        # every byte of the cache starts as a NaN's: rows that are not written never count
        shape = (self.pages, page, kv_heads, dh)
        item = np.uint8 if cache_dtype == E4M3 else np.uint16
        self.kc, self.vc = (np.full(shape, 0x7f if cache_dtype == E4M3 else NAN[dtype], item) for _ in range(2))
        self.ks, self.vs = (np.full(shape[:3], 0xff, np.uint8) for _ in range(2))

    def slot(self, b, position):
        page = int(self.table[b, position // self.page])
        return (page, position % self.page) if 0 <= page < self.pages else None

    def fill_past(self, seed=50):
        """Values for the positions before the new tokens, in the cache's own form."""
        for b, n in enumerate(self.past):
            for x, c, s, i in ((0, self.kc, self.ks, 0), (1, self.vc, self.vs, 1)):
                rows = synth.tensor(seed + 2 * b + i, (max(n, 1), self.kv_heads * self.dh), self.dtype, "normal")[:max(n, 0)]
                self.put(c, s, b, 0, rows)

    def put(self, c, s, b, first, rows):
        v = ref.values(rows, self.dtype).reshape(-1, self.kv_heads, self.dh)
        if self.cache_dtype == E4M3:
            y, scale = ref.quantise(v)
            bits = np.zeros(y.shape, np.uint8)
            grid = ref.e4m3_values(np.arange(127))
            bits = np.searchsorted(grid, np.abs(y)).astype(np.uint8) | (np.signbit(y) << 7).astype(np.uint8)
        for i in range(v.shape[0]):
            if first + i < 0 or (at := self.slot(b, first + i)) is None:
                continue
            if self.cache_dtype == E4M3:
                c[at], s[at] = bits[i], scale[i]
            else:
                c[at] = rows[i].reshape(self.kv_heads, self.dh)

    def put_new(self):
        for b, n in enumerate(self.new):
            rows = slice(self.cu[b], self.cu[b + 1])
            self.put(self.kc, self.ks, b, self.past[b], self.k[rows])
            self.put(self.vc, self.vs, b, self.past[b], self.v[rows])

    def row(self, c, s, at):
        """A cache row [kv_heads, dh] in float64, as the storage type holds it."""
        if self.cache_dtype != E4M3:
            return ref.values(c[at], self.dtype)
        v = ref.e4m3_values(c[at]) * (2.0 ** (s[at].astype(np.float64) - 127))[:, None]
        return ref.values(synth.to_storage(v.astype(np.float32), self.dtype), self.dtype)

    def upload(self):
        hip = self.hip
        self.dev = {n: hip.to_device(getattr(self, n)) for n in ("kc", "vc", "ks", "vs", "table", "cached", "cu", "q", "k", "v")}
        d = self.dev
        self.desc = hip.PagedCache(dtype=self.dtype, cache_dtype=self.cache_dtype, pages=self.pages, page_size=self.page,
                                   kv_heads=self.kv_heads, dh=self.dh, k=d["kc"].value, v=d["vc"].value, k_scale=d["ks"].value,
                                   v_scale=d["vs"].value, batch=len(self.new), block_table=d["table"].value,
                                   table_stride=self.table.shape[1], kv_lens=d["cached"].value)
        return ctypes.byref(self.desc)

    def attend(self, max_new=None, max_keys=None, stream=None):
        hip, d, r = self.hip, self.dev, ctypes.byref(self.desc)
        new = max(self.new) if max_new is None else max_new
        keys = int(max(self.cached)) if max_keys is None else max_keys
        need = hip.lib().fh_attention_paged_workspace(r, self.rows, self.heads, new, keys)
        assert need >= 0
        ws = hip.to_device(np.full(max(need // 4, 1), np.nan, np.float32))
        out = hip.to_device(np.full((self.rows, self.heads * self.dh), KEEP, np.uint16))
        hip.check(hip.lib().fh_attention_paged(r, d["q"].value, self.heads * self.dh, out.value, self.heads * self.dh, self.rows,
                                               self.heads, d["cu"].value, float(np.float32(1 / np.sqrt(self.dh))), new, keys,
                                               ws.value if need else None, need, stream))
        hip.check(hip.lib().fh_device_synchronize())
        return out.download((self.rows, self.heads * self.dh), np.uint16), need

    def check_attend(self, out, what):
        scale, group = float(np.float32(1 / np.sqrt(self.dh))), self.heads // self.kv_heads
        assert (out[self.cu[-1]:] == KEEP).all(), "rows behind the last sequence were written"
        for b, n in enumerate(self.new):
            total = int(self.cached[b])
            slots = [self.slot(b, p) for p in range(max(total, 0))]
            there = np.array([s is not None for s in slots], bool)
            empty = np.zeros((self.kv_heads, self.dh))
            keys, vals = (np.array([self.row(c, scales, s) if s else empty for s in slots]).reshape(-1, self.kv_heads, self.dh)
                          for c, scales in ((self.kc, self.ks), (self.vc, self.vs)))
            seen = (np.arange(total)[None, :] <= total - n + np.arange(n)[:, None]) & there[None, :]
            rows = slice(self.cu[b], self.cu[b + 1])
            for h in range(self.heads if n else 0):
                mine = slice(h * self.dh, (h + 1) * self.dh)
                q = ref.values(self.q[rows, mine], self.dtype)
                want, tol, *_ = ref.attend(q, keys[:, h // group], vals[:, h // group], seen, scale, self.dtype)
                # parts joined in fp32 add a few roundings of the sums
                ref.check(ref.values(out[rows, mine], self.dtype), want, tol + 2.0 ** -20 * np.abs(want), f"{what} sequence {b} head {h}")


# dtype, cache, past, new, heads, kv_heads, dh, page, rows behind
PAGED = [
    (BF16, BF16, [0], [1], 1, 1, 64, 16, 0),                              # a first token over itself
    (BF16, BF16, [100, 0, 63, 64], [1, 1, 1, 1], 8, 2, 128, 16, 0),       # a decoding step
    (BF16, E4M3, [100, 0, 63, 64], [1, 1, 1, 1], 8, 2, 128, 16, 3),
    (F16, F16, [33, 5, 0], [7, 0, 40], 4, 4, 64, 8, 2),                   # chunks, an empty one, pages of 8
    (F16, E4M3, [33, 5, 0], [7, 0, 40], 6, 2, 64, 1, 0),                  # pages of one row
    (BF16, E4M3, [250, 1], [90, 130], 6, 1, 80, 64, 0),                   # head dim between tile sizes
    (BF16, BF16, [2000], [1], 4, 1, 128, 32, 0),                          # keys cut into parts
    (BF16, E4M3, [3001, 17, 700], [1, 1, 1], 4, 2, 64, 128, 0),
    (F16, F16, [1500, 900], [3, 20], 16, 2, 96, 256, 4),
    (BF16, BF16, [0, 10] * 40, [1] * 80, 2, 1, 64, 16, 0),                # more than 64 sequences
    (F16, E4M3, [500], [260], 2, 2, 128, 64, 0),
    (BF16, E4M3, [70, 900], [1, 5], 40, 1, 32, 16, 0),                    # a group of 40
]


def paged_id(c):
    return (f"{'f16' if c[0] == F16 else 'bf16'}-{'e4m3' if c[1] == E4M3 else '16bit'}-{len(c[2])}x{max(c[2])}+{max(c[3])}-"
            f"h{c[4]}k{c[5]}d{c[6]}p{c[7]}")


@pytest.mark.parametrize("case", PAGED, ids=paged_id)
def test_paged_attention(hip, case):
    say(f"paged attention {case}")
    p = Paged(hip, *case)
    p.fill_past()
    p.put_new()
    p.upload()
    out, _ = p.attend()
    p.check_attend(out, "paged")
    # the expected lengths choose the cut and nothing else: none, and ones that the sequences exceed or fall short of
    for new, keys in ((1, 1), (1, 1 << 20), (4096, 300)):
        p.check_attend(p.attend(new, keys)[0], f"paged, cut for {new} x {keys}")


def test_paged_rows_that_see_nothing(hip):
    # more new tokens than cached positions: the first ones stand before position 0; and a sequence without a cache
    say("paged rows that see nothing")
    for cache_dtype in (BF16, E4M3):
        p = Paged(hip, BF16, cache_dtype, [0, -3, 0], [2, 6, 5], 4, 2, 64, 16)
        p.cached[2] = 0
        p.put_new()
        p.upload()
        for keys in (3, 1 << 20):
            out, _ = p.attend(max_keys=keys)
            p.check_attend(out, "empty rows")
            assert (out[p.cu[1]:p.cu[1] + 3] == 0).all() and (out[p.cu[2]:] == 0).all()


@pytest.mark.parametrize("dtype,cache_dtype,dh", [(BF16, BF16, 128), (F16, E4M3, 64)])
def test_paged_many_chunks(hip, dtype, cache_dtype, dh):
    # more tiles than CUs
    say(f"paged, many chunks, dh {dh}, cache {cache_dtype}")
    p = Paged(hip, dtype, cache_dtype, [0, 100, 33, 7] * 15, [40, 33, 20, 70] * 15, 32, 8, dh, 16)
    p.fill_past()
    p.put_new()
    p.upload()
    p.check_attend(p.attend()[0], "many chunks")


@pytest.mark.parametrize("number", [-1, 1 << 30])
def test_paged_pages_that_do_not_exist(hip, number):
    say(f"paged page number {number}")
    for cache_dtype in (F16, E4M3):
        p = Paged(hip, F16, cache_dtype, [200, 90], [1, 30], 4, 2, 64, 32, bad_page=(0, 2, number))
        p.fill_past()
        p.put_new()
        p.upload()
        for keys in (64, 1 << 20):
            p.check_attend(p.attend(max_keys=keys)[0], "missing page")


@pytest.mark.parametrize("cache_dtype", [BF16, E4M3])
@pytest.mark.parametrize("past,new,bad", [(70, 5, 3), (0, 4, 2), (2000, 6, 5), (61, 90, 40), (1500, 130, 1)])
def test_paged_not_finite_values_reach_the_rows_that_see_them(hip, cache_dtype, past, new, bad):
    say(f"paged NaN at new token {bad} of {new} behind {past}, cache {cache_dtype}")
    p = Paged(hip, BF16, cache_dtype, [past], [new], 4, 2, 64, 16)
    p.fill_past()
    p.put_new()
    p.upload()
    for keys in (64, 1 << 20):
        clean, _ = p.attend(max_keys=keys)
        at, nan = p.slot(0, past + bad), 0x7f if cache_dtype == E4M3 else NAN[BF16]
        kept = p.vc[at + (0, 3)]
        p.vc[at + (0, 3)] = nan
        p.dev["vc"].upload(p.vc)
        out, _ = p.attend(max_keys=keys)
        p.vc[at + (0, 3)] = kept
        p.dev["vc"].upload(p.vc)
        affected = (np.arange(new)[:, None] >= bad) & (np.arange(256) < 128) & (np.arange(256) % 64 == 3)
        assert np.array_equal(out[~affected], clean[~affected])
        assert np.isnan(ref.values(out[affected], BF16)).all()


def test_paged_lengths_past_the_table(hip):
    # lengths are taken as what the block table can hold, negative ones as none
    say("paged lengths past the table")
    p = Paged(hip, BF16, BF16, [60, 16], [4, 2], 2, 1, 64, 16)
    p.fill_past()
    p.put_new()
    p.upload()
    full = np.array([p.table.shape[1] * 16, -7], np.int32)
    p.dev["cached"].upload(np.array([1 << 30, -7], np.int32))
    out, _ = p.attend()
    p.cached = np.maximum(full, 0)
    p.check_attend(out, "past the table")


@pytest.mark.parametrize("case", PAGED, ids=paged_id)
def test_cache_write_and_read(hip, case):
    say(f"cache write and read {case}")
    p = Paged(hip, *case)
    p.fill_past()
    r = p.upload()
    lib, d, ld = hip.lib(), p.dev, p.kv_heads * p.dh
    hip.check(lib.fh_kv_cache_write(r, d["k"].value, ld, d["v"].value, ld, p.rows, d["cu"].value, None))
    p.put_new()
    names = ["kc", "vc"] + (["ks", "vs"] if p.cache_dtype == E4M3 else [])
    for n in names:
        want = getattr(p, n)
        assert np.array_equal(d[n].download(want.shape, want.dtype), want), n
    # everything back, with one position more than is cached per sequence: it reads as zeros
    lens = [int(n) + 1 for n in p.cached]
    cu = starts(lens, 2)
    rows = int(cu[-1]) + 3
    back = [hip.to_device(np.full((rows, ld + 8), KEEP, np.uint16)) for _ in range(2)]
    dcu = hip.to_device(cu)
    hip.check(lib.fh_kv_cache_read(r, back[0].value, ld + 8, back[1].value, ld + 8, rows, dcu.value, None))
    for buf, c, s in ((back[0], p.kc, p.ks), (back[1], p.vc, p.vs)):
        got = buf.download((rows, ld + 8), np.uint16)
        want = np.full((rows, ld + 8), KEEP, np.uint16)
        for b, n in enumerate(lens):
            for i in range(n):
                at = p.slot(b, i) if i < n - 1 else None
                value = p.row(c, s, at).ravel() if at else np.zeros(ld)
                want[cu[b] + i, :ld] = synth.to_storage(value.astype(np.float32), p.dtype)
        same = (got == want) | ((got | 0x8000) == 0x8000) & ((want | 0x8000) == 0x8000)  # zeros of either sign
        assert same.all(), np.argwhere(~same)[:3]


def special_rows(dtype):
    """Rows whose quantisation has edges: ties, the largest quotient, powers of two, zeros, subnormals, values that are not finite."""
    tiny = 2.0 ** -24 if dtype == F16 else 2.0 ** -133
    big = 65504.0 if dtype == F16 else 3.0e38
    rows = np.zeros((12, 64), np.float64)
    rows[0] = np.linspace(-1, 1, 64)
    rows[1, :4] = [448, 447, -448, 1]              # just within
    rows[2, :4] = [450, 28, 29, -30]               # just past: the next power of two
    rows[3] = [2.0 ** (i - 40) if dtype == BF16 else 2.0 ** (i % 30 - 20) for i in range(64)]
    rows[4, 5] = -0.0
    rows[5, :3] = [tiny, -tiny, 3 * tiny]
    rows[6, :3] = [big, -big / 3, 1.0]
    rows[7] = 1.0 + np.arange(64) / 64.0           # ties between neighbours of the 3-bit fraction
    rows[8, :4] = [np.nan, 1.0, -2.0, 0.5]
    rows[9, :4] = [np.inf, 1.0, -np.inf, 0.5]
    rows[10] = np.nan
    rows[11] = 2.0 ** -10 * (1 + np.arange(64) / 7.0)
    return synth.to_storage(rows.astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_quantised_values(hip, dtype):
    say(f"e4m3 edges dtype={dtype}")
    rows = special_rows(dtype)
    p = Paged(hip, dtype, E4M3, [0], [len(rows)], 1, 1, 64, 16)
    p.k, p.v = rows, rows[::-1].copy()
    r = p.upload()
    d = p.dev
    hip.check(hip.lib().fh_kv_cache_write(r, d["k"].value, 64, d["v"].value, 64, p.rows, d["cu"].value, None))
    for src, c, s in ((p.k, "kc", "ks"), (p.v, "vc", "vs")):
        got, scale = d[c].download(p.kc.shape, np.uint8), d[s].download(p.ks.shape, np.uint8)
        want, want_scale = ref.quantise(ref.values(src, dtype))
        for i in range(len(rows)):
            at = p.slot(0, i)
            assert scale[at][0] == want_scale[i], (c, i)
            assert np.array_equal(ref.e4m3_values(got[at][0]), want[i], equal_nan=True), (c, i)


def test_write_skips_what_has_no_place(hip):
    # positions before 0, rows of no sequence and pages that do not exist are skipped
    say("cache write without a place")
    p = Paged(hip, BF16, E4M3, [-2, 20], [5, 30], 2, 2, 64, 16, behind=4, bad_page=(1, 2, 99999))
    r = p.upload()
    d = p.dev
    hip.check(hip.lib().fh_kv_cache_write(r, d["k"].value, 128, d["v"].value, 128, p.rows, d["cu"].value, None))
    p.put_new()
    for n in ("kc", "vc", "ks", "vs"):
        want = getattr(p, n)
        assert np.array_equal(d[n].download(want.shape, want.dtype), want), n


@pytest.mark.parametrize("cache_dtype", [BF16, E4M3])
def test_offsets_past_32_bits(hip, cache_dtype):
    # 2^32 elements and more in front of the pages: the same results as in a small cache
    say(f"a cache of more than 2^32 elements, cache {cache_dtype}")
    total, new, heads, dh, page = 603, 3, 4, 128, 256
    k, v = (synth.tensor(70 + i, (total, dh), BF16, "normal") for i in range(2))
    q = synth.tensor(72, (new, heads * dh), BF16, "normal")
    lib, item = hip.lib(), 1 if cache_dtype == E4M3 else 2
    dk, dv, dq = (hip.to_device(x) for x in (k, v, q))
    lens, cu_all, cu_new = hip.to_device(np.array([total], np.int32)), hip.to_device(starts([total])), hip.to_device(starts([new]))
    got = []
    for pages in (3, (1 << 17) + 3):
        kc, vc = (hip.DeviceBuffer(pages * page * dh * item) for _ in range(2))
        ks, vs = (hip.DeviceBuffer(pages * page) for _ in range(2))
        table = hip.to_device(np.array([[pages - 1, 0, pages - 2]], np.int32))
        c = hip.PagedCache(dtype=BF16, cache_dtype=cache_dtype, pages=pages, page_size=page, kv_heads=1, dh=dh, k=kc.value, v=vc.value,
                           k_scale=ks.value, v_scale=vs.value, batch=1, block_table=table.value, table_stride=3, kv_lens=lens.value)
        r = ctypes.byref(c)
        hip.check(lib.fh_kv_cache_write(r, dk.value, dh, dv.value, dh, total, cu_all.value, None))
        back = [hip.to_device(np.zeros((total, dh), np.uint16)) for _ in range(2)]
        hip.check(lib.fh_kv_cache_read(r, back[0].value, dh, back[1].value, dh, total, cu_all.value, None))
        got.append([b.download((total, dh), np.uint16) for b in back])
        out = hip.to_device(np.zeros((new, heads * dh), np.uint16))
        for max_new in (new, 64):  # both forms
            need = lib.fh_attention_paged_workspace(r, new, heads, max_new, total)
            ws = hip.DeviceBuffer(max(need, 16))
            hip.check(lib.fh_attention_paged(r, dq.value, heads * dh, out.value, heads * dh, new, heads, cu_new.value,
                                             float(np.float32(1 / np.sqrt(dh))), max_new, total, ws.value, need, None))
            hip.check(lib.fh_device_synchronize())
            got[-1].append(out.download((new, heads * dh), np.uint16))
        for b in (kc, vc):
            b.free()
    for a, b in zip(*got):
        assert a.any() and np.array_equal(a, b)
    if cache_dtype == BF16:
        assert np.array_equal(got[0][0], k) and np.array_equal(got[0][1], v)


def test_a_prompt_then_tokens_one_by_one(hip):
    """A run as a server makes it: the prompt's keys and values into an e4m3 cache, then steps that write one token each and attend
    over the cache, every step captured once and replayed, against the packed forward over what the cache reads back as."""
    say("prompt, then decoding steps")
    lens, steps, heads, kv_heads, dh, page = [130, 1, 64], 6, 8, 2, 64, 16
    p = Paged(hip, BF16, E4M3, lens, [steps] * 3, heads, kv_heads, dh, page)
    lib, ld = hip.lib(), kv_heads * dh
    total = p.cached.copy()
    p.upload()
    d, r = p.dev, ctypes.byref(p.desc)
    prompt = [synth.tensor(90 + i, (sum(lens), ld), BF16, "normal") for i in range(2)]
    dev_prompt, pcu = [hip.to_device(x) for x in prompt], hip.to_device(starts(lens))
    d["cached"].upload(np.array(lens, np.int32))
    hip.check(lib.fh_kv_cache_write(r, dev_prompt[0].value, ld, dev_prompt[1].value, ld, sum(lens), pcu.value, None))
    step_cu = hip.to_device(starts([1, 1, 1]))
    k1, v1, q1, o1 = (hip.DeviceBuffer(3 * w * 2) for w in (ld, ld, heads * dh, heads * dh))
    scale = float(np.float32(1 / np.sqrt(dh)))
    need = lib.fh_attention_paged_workspace(r, 3, heads, 1, int(total.max()))
    ws, stream, graph = hip.DeviceBuffer(max(need, 16)), hip.Stream(), ctypes.c_void_p()
    hip.check(lib.fh_device_synchronize())
    hip.check(lib.fh_graph_begin_capture(stream.ptr))
    hip.check(lib.fh_kv_cache_write(r, k1.value, ld, v1.value, ld, 3, step_cu.value, stream.ptr))
    hip.check(lib.fh_attention_paged(r, q1.value, heads * dh, o1.value, heads * dh, 3, heads, step_cu.value, scale, 1,
                                     int(total.max()), ws.value, need, stream.ptr))
    hip.check(lib.fh_graph_end_capture(stream.ptr, 1, ctypes.byref(graph)))
    outs = []
    for i in range(steps):
        at = [int(p.cu[b]) + i for b in range(3)]
        k1.upload(p.k[at])
        v1.upload(p.v[at])
        q1.upload(p.q[at])
        d["cached"].upload(np.array(lens, np.int32) + i + 1)
        hip.check(lib.fh_graph_launch(graph, stream.ptr))
        stream.synchronize()
        outs.append(o1.download((3, heads * dh), np.uint16))
    hip.check(lib.fh_graph_destroy(graph))
    # the whole sequences from the cache, and the packed forward over them: its last rows are the steps'
    whole = Packed(hip, BF16, list(total), heads, kv_heads, dh, 1)
    cu = hip.to_device(whole.cu)
    back = [hip.DeviceBuffer(whole.rows * ld * 2) for _ in range(2)]
    hip.check(lib.fh_kv_cache_read(r, back[0].value, ld, back[1].value, ld, whole.rows, cu.value, None))
    whole.x["k"], whole.x["v"] = (b.download((whole.rows, ld), np.uint16) for b in back)
    for b in range(3):
        for i in range(steps):
            whole.x["q"][whole.cu[b] + lens[b] + i] = p.q[p.cu[b] + i]
    want, tol, _, _ = whole.want()
    for i in range(steps):
        rows = [int(whole.cu[b]) + lens[b] + i for b in range(3)]
        ref.check(ref.values(outs[i], BF16), want[rows], tol[rows] + 2.0 ** -20 * np.abs(want[rows]), f"step {i}")
    out, lse = whole.forward()
    whole.check_forward(out, lse, "packed over the cache's rows")
