"""Token embedding and its table's gradient against float64 (tests/language_ref.py, which derives the bounds)."""
import ctypes

import numpy as np
import pytest

import language_ref as ref
from frame_hip import synth

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 2, 3
KEEP = {F32: np.float32(-77.0), F16: np.uint16(0x5a5a), BF16: np.uint16(0x5a5a)}


def say(msg):
    print(f"[case] {msg}", flush=True)


def text_ids(tokens, vocab, seed, outside=0.0):
    """Ids as frequent as words, some of them outside the vocabulary on either side."""
    rng = np.random.default_rng(seed)
    ids = np.minimum(np.exp(rng.random(tokens) * np.log(vocab + 1)).astype(np.int64) - 1, vocab - 1)
    bad = rng.random(tokens) < outside
    ids[bad] = rng.choice([-1, vocab, 2 ** 31 - 1, -2 ** 31], bad.sum())
    return ids.astype(np.int32)


class Embedding:
    def __init__(self, hip, dtype, tokens, vocab, dim, ids, scale=1.0, pad=0, shift=0, seed=1):
        """pad: elements between rows of out and dout that belong to none. shift: elements that every tensor begins behind 16 bytes."""
        self.hip, self.dtype, self.tokens, self.vocab, self.dim = hip, dtype, tokens, vocab, dim
        self.ids, self.scale, self.ld, self.shift, self.seed = np.asarray(ids, np.int32), float(np.float32(scale)), dim + pad, shift, seed
        self.size = 4 if dtype == F32 else 2

    def up(self, array):
        flat = np.concatenate([np.full(self.shift, KEEP[self.dtype]), np.ascontiguousarray(array).ravel(), np.full(8, KEEP[self.dtype])])
        buf = self.hip.to_device(flat)
        return buf, buf.value + self.shift * self.size

    def down(self, buf, shape):
        flat = buf.download((self.shift + int(np.prod(shape)) + 8,), KEEP[self.dtype].dtype)
        assert (flat[:self.shift] == KEEP[self.dtype]).all() and (flat[-8:] == KEEP[self.dtype]).all(), "written outside the tensor"
        return flat[self.shift:-8].reshape(shape)

    def geom(self):
        return self.hip.TokenEmbedding(dtype=self.dtype, tokens=self.tokens, vocab=self.vocab, dim=self.dim, row_stride=self.ld,
                                       scale=self.scale)

    def rows(self, array):
        """[tokens, dim] into rows of the stride."""
        whole = np.full((self.tokens, self.ld), KEEP[self.dtype])
        whole[:, :self.dim] = array
        return whole

    def forward(self, table, stream=None):
        hip = self.hip
        tb, tp = self.up(table)
        ids = hip.to_device(self.ids if self.tokens else np.zeros(1, np.int32))
        ob, op = self.up(np.full((self.tokens, self.ld), KEEP[self.dtype]))
        hip.check(hip.lib().fh_embedding_fwd(ctypes.byref(self.geom()), tp, ids.value, op, stream))
        hip.check(hip.lib().fh_device_synchronize())
        out = self.down(ob, (self.tokens, self.ld))
        assert (out[:, self.dim:] == KEEP[self.dtype]).all(), "the columns between rows were written"
        return out[:, :self.dim]

    def backward(self, dout, base=None, in_place=False, stream=None):
        hip, lib = self.hip, self.hip.lib()
        db, dp = self.up(self.rows(dout))
        ids = hip.to_device(self.ids if self.tokens else np.zeros(1, np.int32))
        bb, bp = self.up(base) if base is not None else (None, None)
        gb, gp = (bb, bp) if in_place else self.up(np.full((self.vocab, self.dim), KEEP[self.dtype]))
        g = self.geom()
        need = lib.fh_embedding_grad_workspace(ctypes.byref(g))
        ws = hip.to_device(np.full(need // 4 + 4, np.nan, np.float32))
        hip.check(lib.fh_embedding_grad(ctypes.byref(g), dp, ids.value, bp, gp, ws.value, need, stream))
        hip.check(lib.fh_device_synchronize())
        assert np.isnan(ws.download((need // 4 + 4,), np.float32)[need // 4:]).all(), "written behind the workspace"
        return self.down(gb, (self.vocab, self.dim))


SHAPES = [  # tokens, vocab, dim, scale, pad, shift, share of ids outside
    (1, 1, 1, 1.0, 0, 0, 0.0), (1, 7, 64, 1.0, 0, 0, 0.0), (2, 3, 3, 0.5, 0, 1, 0.0), (17, 5, 8, 1.0, 0, 0, 0.3),
    (64, 1000, 128, 11.3125, 0, 0, 0.1), (300, 40, 333, 1.0, 3, 1, 0.2), (257, 1, 72, 1.0, 8, 0, 0.0), (500, 65536, 40, 1.0, 0, 0, 0.05),
    (33, 511, 1000, -2.0, 24, 0, 0.0), (100, 512, 1001, 1.0, 0, 3, 0.0), (3000, 300, 96, 1.0, 0, 0, 0.1), (9, 12, 4100, 0.25, 0, 0, 0.5),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(hip, shape, dtype):
    tokens, vocab, dim, scale, pad, shift, outside = shape
    say(f"embedding {shape} dtype={dtype}")
    e = Embedding(hip, dtype, tokens, vocab, dim, text_ids(tokens, vocab, 3, outside), scale, pad, shift)
    table = synth.tensor(11, (vocab, dim), dtype, "normal")
    want, tol = ref.embed(ref.values(table, dtype), e.ids.astype(np.int64), e.scale, dtype)
    ref.check(ref.values(e.forward(table), dtype), want, tol, "out")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("base", ["none", "other", "same"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradient(hip, shape, base, dtype):
    tokens, vocab, dim, scale, pad, shift, outside = shape
    say(f"embedding gradient {shape} base={base} dtype={dtype}")
    e = Embedding(hip, dtype, tokens, vocab, dim, text_ids(tokens, vocab, 3, outside), scale, pad, shift)
    dout = synth.tensor(12, (tokens, dim), dtype, "normal")
    other = None if base == "none" else synth.tensor(13, (vocab, dim), dtype, "normal")
    want, tol = ref.embed_grad(ref.values(dout, dtype), e.ids.astype(np.int64), vocab, e.scale,
                               None if other is None else ref.values(other, dtype), dtype)
    got = e.backward(dout, other, base == "same")
    ref.check(ref.values(got, dtype), want, tol, "dtable")
    assert np.array_equal(got, e.backward(dout, other, base == "same")), "two calls differ"


PATTERNS = {  # where ids' runs begin and end in the sorted list
    "one id": lambda n: np.zeros(n), "each once": lambda n: np.arange(n)[::-1], "runs of 16": lambda n: np.arange(n) // 16,
    "runs of 15": lambda n: np.arange(n) // 15, "runs of 17": lambda n: np.arange(n) // 17, "two halves": lambda n: np.arange(n) * 2 // n,
    "all outside": lambda n: np.full(n, -5), "one inside": lambda n: np.where(np.arange(n) == n // 2, 4, -1),
    "alternating": lambda n: np.arange(n) % 2, "one behind a run": lambda n: np.where(np.arange(n) == 16, 1, 0),
}


@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 32, 33, 1000, 2048, 2049, 20000])
@pytest.mark.parametrize("pattern", sorted(PATTERNS))
def test_gradient_runs(hip, pattern, tokens):
    """Whole numbers: every sum is exact, whatever its order."""
    say(f"embedding gradient, {pattern}, {tokens} tokens")
    ids, vocab, dim = PATTERNS[pattern](tokens).astype(np.int32), tokens + 1, 24
    e = Embedding(hip, F32, tokens, vocab, dim, ids)
    dout = np.random.default_rng(1).integers(-8, 9, (tokens, dim)).astype(np.float32)
    want = np.zeros((vocab, dim))
    named = (ids >= 0) & (ids < vocab)
    np.add.at(want, ids[named], dout[named].astype(np.float64))
    assert np.array_equal(e.backward(dout).astype(np.float64), want)


@pytest.mark.parametrize("tokens", [1024, 1025, 4096, 4097, 16384, 16385])
def test_gradient_where_another_sort_takes_over(hip, tokens):
    say(f"embedding gradient, {tokens} tokens of 700 ids")
    vocab, dim = 700, 16
    ids = text_ids(tokens, vocab, 17, 0.1)
    e = Embedding(hip, F32, tokens, vocab, dim, ids)
    dout = np.random.default_rng(2).integers(-8, 9, (tokens, dim)).astype(np.float32)
    want = np.zeros((vocab, dim))
    named = (ids >= 0) & (ids < vocab)
    np.add.at(want, ids[named], dout[named].astype(np.float64))
    assert np.array_equal(e.backward(dout).astype(np.float64), want)


@pytest.mark.parametrize("dim,shift", [(1, 0), (8, 0), (24, 1), (333, 0), (1200, 0), (2056, 0)])
@pytest.mark.parametrize("tokens", [255, 256, 257, 511, 512, 513, 700, 1023, 1024, 1025])
def test_gradient_of_few_tokens(hip, tokens, dim, shift):
    """The first, the last and an id of most tokens; rows shorter and longer than what a workgroup writes, some of them not whole vectors."""
    say(f"embedding gradient, {tokens} tokens of 600 x {dim}, {shift} elements behind 16 bytes")
    vocab, rng = 600, np.random.default_rng(tokens)
    ids = np.where(rng.random(tokens) < 0.6, 77, rng.integers(-1, vocab + 1, tokens)).astype(np.int32)
    ids[0], ids[-1], ids[5] = vocab - 1, 0, vocab - 1
    e = Embedding(hip, F32, tokens, vocab, dim, ids, shift=shift)
    dout = rng.integers(-8, 9, (tokens, dim)).astype(np.float32)
    base = rng.integers(-8, 9, (vocab, dim)).astype(np.float32)
    want = np.zeros((vocab, dim))
    named = (ids >= 0) & (ids < vocab)
    np.add.at(want, ids[named], dout[named].astype(np.float64))
    assert np.array_equal(e.backward(dout).astype(np.float64), want)
    assert np.array_equal(e.backward(dout, base).astype(np.float64), want + base)
    assert np.array_equal(e.backward(dout, base, True).astype(np.float64), want + base)


@pytest.mark.parametrize("vocab", [8192, 8193])
def test_gradient_where_the_writing_takes_longer_than_a_sort(hip, vocab):
    say(f"embedding gradient, 40 tokens of {vocab} x 2,048 f32")
    dim, rng = 2048, np.random.default_rng(3)
    ids = rng.integers(0, vocab, 40).astype(np.int32)
    ids[3], ids[7] = vocab - 1, ids[30]
    dout = rng.integers(-8, 9, (40, dim)).astype(np.float32)
    want = np.zeros((vocab, dim), np.float32)
    np.add.at(want, ids, dout)
    assert np.array_equal(Embedding(hip, F32, 40, vocab, dim, ids).backward(dout), want)


@pytest.mark.parametrize("vocab", [1, 2, 510, 511, 512, 513, 262143, 262144])
def test_gradient_of_any_number_of_digits(hip, vocab):
    """The ids outside the vocabulary sort behind all others: their key is the vocabulary's size, which may need one bit more."""
    say(f"embedding gradient, {vocab} ids")
    tokens, dim = 3000, 8
    ids = np.random.default_rng(vocab).integers(0, vocab, tokens).astype(np.int32)
    ids[::7], ids[1], ids[-1] = -1, vocab - 1, vocab - 1
    dout = np.random.default_rng(2).integers(-8, 9, (tokens, dim)).astype(np.float32)
    want = np.zeros((vocab, dim))
    np.add.at(want, ids[ids >= 0], dout[ids >= 0].astype(np.float64))
    assert np.array_equal(Embedding(hip, F32, tokens, vocab, dim, ids).backward(dout).astype(np.float64), want)


def test_many_tokens_and_a_large_vocabulary(hip):
    say("70,000 tokens of 300,000 ids")
    tokens, vocab, dim = 70000, 300000, 8
    rng = np.random.default_rng(4)
    ids = np.where(rng.random(tokens) < 0.5, rng.integers(0, vocab, tokens), text_ids(tokens, vocab, 5)).astype(np.int32)
    dout = rng.integers(-4, 5, (tokens, dim)).astype(np.float32)
    want = np.zeros((vocab, dim))
    np.add.at(want, ids, dout.astype(np.float64))
    assert np.array_equal(Embedding(hip, F32, tokens, vocab, dim, ids).backward(dout).astype(np.float64), want)


def test_rows_outside_the_vocabulary_reach_nothing(hip):
    say("NaN in rows that name nothing")
    tokens, vocab, dim = 100, 9, 64
    ids = text_ids(tokens, vocab, 6, 0.5)
    dout = synth.tensor(14, (tokens, dim), BF16, "normal")
    named = (ids >= 0) & (ids < vocab)
    dout[~named] = 0x7fc0
    got = ref.values(Embedding(hip, BF16, tokens, vocab, dim, ids).backward(dout), BF16)
    clean = np.where(named[:, None], ref.values(dout, BF16), 0.0)
    want, tol = ref.embed_grad(clean, ids.astype(np.int64), vocab, 1.0, None, BF16)
    ref.check(got, want, tol, "dtable")


def test_values_that_are_not_finite_stay_with_their_id(hip):
    say("infinity and NaN in one token's row")
    dout = synth.tensor(15, (40, 64), F16, "normal")
    dout[7, 3], dout[7, 4] = 0x7c00, 0x7e00
    ids = (np.arange(40) % 10).astype(np.int32)
    got = ref.values(Embedding(hip, F16, 40, 10, 64, ids).backward(dout), F16)
    assert np.isposinf(got[7, 3]) and np.isnan(got[7, 4])
    got[7, 3] = got[7, 4] = 0.0
    assert np.isfinite(got).all()


def test_no_tokens(hip):
    say("no tokens: zeros, base, and base left alone")
    e = Embedding(hip, BF16, 0, 5, 16, [])
    none = np.zeros((0, 16), np.uint16)
    base = synth.tensor(16, (5, 16), BF16, "normal")
    assert e.forward(base).shape == (0, 16)
    assert not e.backward(none).any()
    assert np.array_equal(e.backward(none, base), base) and np.array_equal(e.backward(none, base, True), base)


def test_table_past_32_bits(hip):
    """A table of more than 2^32 bytes: the last rows, and their gradients on top of themselves."""
    vocab, dim, tokens = 2 ** 21 + 5, 1024, 6
    say(f"table of {vocab * dim * 2} bytes")
    ids = np.array([0, vocab - 1, 2 ** 21, vocab - 1, vocab, 2 ** 20 + 3], np.int32)
    lib = hip.lib()
    table, out = hip.DeviceBuffer(vocab * dim * 2), hip.DeviceBuffer(tokens * dim * 2)
    hip.check(lib.fh_fill(table.value, 2, 0x3f80, vocab * dim, None))  # ones
    rows = {int(i): synth.tensor(20 + n, (dim,), BF16, "normal") for n, i in enumerate(sorted(set(ids[ids < vocab])))}
    for i, r in rows.items():
        hip.check(lib.fh_memcpy(table.value + i * dim * 2, r.ctypes.data, r.nbytes, hip.H2D, None))
    g = hip.TokenEmbedding(dtype=BF16, tokens=tokens, vocab=vocab, dim=dim, row_stride=dim, scale=1.0)
    dev_ids = hip.to_device(ids)
    hip.check(lib.fh_embedding_fwd(ctypes.byref(g), table.value, dev_ids.value, out.value, None))
    got = out.download((tokens, dim), np.uint16)
    for t, i in enumerate(ids):
        assert np.array_equal(got[t], rows[int(i)] if i < vocab else np.zeros(dim, np.uint16))
    need = lib.fh_embedding_grad_workspace(ctypes.byref(g))
    ws = hip.DeviceBuffer(need)
    hip.check(lib.fh_embedding_grad(ctypes.byref(g), out.value, dev_ids.value, table.value, table.value, ws.value, need, None))
    hip.check(lib.fh_device_synchronize())
    for i, r in rows.items():
        now = np.empty(dim, np.uint16)
        hip.check(lib.fh_memcpy(now.ctypes.data, table.value + i * dim * 2, now.nbytes, hip.D2H, None))
        want = ref.values(r, BF16) * (1 + (ids == i).sum())
        ref.check(ref.values(now, BF16), want, ref.rounded(want, 0.0, BF16), f"row {i}")
    near = np.empty(dim, np.uint16)
    hip.check(lib.fh_memcpy(near.ctypes.data, table.value + (vocab - 2) * dim * 2, near.nbytes, hip.D2H, None))
    assert (near == 0x3f80).all()


def test_table_of_more_elements_than_a_launch_writes(hip):
    """Elements that are written one by one (the table begins behind 2 bytes), more than 2^31 of them: in two launches."""
    vocab, dim, tokens = 2 ** 21 + 5, 1029, 5
    say(f"table of {vocab * dim} elements behind 2 bytes")
    ids = np.array([1, vocab - 1, 1, vocab // 2, -1], np.int32)
    lib = hip.lib()
    dout = synth.tensor(27, (tokens, dim), BF16, "normal")
    table = hip.DeviceBuffer((vocab * dim + 8) * 2)
    hip.check(lib.fh_fill(table.value, 2, 0x3f80, vocab * dim + 8, None))
    g = hip.TokenEmbedding(dtype=BF16, tokens=tokens, vocab=vocab, dim=dim, row_stride=dim, scale=1.0)
    need = lib.fh_embedding_grad_workspace(ctypes.byref(g))
    ws, dev_ids, dev_dout = hip.DeviceBuffer(need), hip.to_device(ids), hip.to_device(dout)
    hip.check(lib.fh_embedding_grad(ctypes.byref(g), dev_dout.value, dev_ids.value, None, table.value + 2, ws.value, need, None))
    hip.check(lib.fh_device_synchronize())

    def elements(first, n):
        got = np.empty(n, np.uint16)
        hip.check(lib.fh_memcpy(got.ctypes.data, table.value + 2 + first * 2, got.nbytes, hip.D2H, None))
        return got

    assert elements(-1, 1)[0] == 0x3f80 and (elements(vocab * dim, 7) == 0x3f80).all(), "written outside the tensor"
    named = {1: ref.values(dout[0], BF16) + ref.values(dout[2], BF16), vocab - 1: ref.values(dout[1], BF16), vocab // 2: ref.values(dout[3], BF16)}
    middle = vocab * dim // 2 // dim  # where the second launch takes over
    rows = {0, 2, middle - 1, middle, middle + 1, 2 ** 31 // dim - 1, 2 ** 31 // dim, 2 ** 31 // dim + 1, vocab - 2}
    rows |= set(np.random.default_rng(28).integers(0, vocab, 200).tolist())
    for v in sorted(rows | set(named)):
        want = named.get(v, np.zeros(dim))
        ref.check(ref.values(elements(v * dim, dim), BF16), want, ref.rounded(want, 0.0, BF16), f"row {v}")


@pytest.mark.parametrize("tokens", [700, 3000, 20000])
def test_captured_and_replayed(hip, tokens):
    say("embedding and its gradient captured, ids changed between the replays")
    vocab, dim = 90, 136
    lib, e = hip.lib(), Embedding(hip, BF16, tokens, vocab, dim, text_ids(tokens, vocab, 8, 0.1))
    table, dout = synth.tensor(21, (vocab, dim), BF16, "normal"), synth.tensor(22, (tokens, dim), BF16, "normal")
    g = e.geom()
    need = lib.fh_embedding_grad_workspace(ctypes.byref(g))
    d = {n: hip.to_device(x) for n, x in dict(ids=e.ids, table=table, dout=dout, out=np.zeros_like(dout), grad=np.zeros_like(table)).items()}
    ws, stream, graph = hip.DeviceBuffer(need), hip.Stream(), ctypes.c_void_p()
    hip.check(lib.fh_device_synchronize())
    hip.check(lib.fh_graph_begin_capture(stream.ptr))
    hip.check(lib.fh_embedding_fwd(ctypes.byref(g), d["table"].value, d["ids"].value, d["out"].value, stream.ptr))
    hip.check(lib.fh_embedding_grad(ctypes.byref(g), d["dout"].value, d["ids"].value, None, d["grad"].value, ws.value, need, stream.ptr))
    hip.check(lib.fh_graph_end_capture(stream.ptr, 1, ctypes.byref(graph)))
    for replay in range(4):
        e.ids = text_ids(tokens, vocab, 30 + replay, 0.2 * replay)
        d["ids"].upload(e.ids)
        hip.check(lib.fh_graph_launch(graph, stream.ptr))
        stream.synchronize()
        assert np.array_equal(d["out"].download((tokens, dim), np.uint16), e.forward(table)), replay
        assert np.array_equal(d["grad"].download((vocab, dim), np.uint16), e.backward(dout)), replay
    hip.check(lib.fh_graph_destroy(graph))


def test_two_streams_at_once(hip):
    say("two calls at once, each with its workspace")
    lib, runs = hip.lib(), []
    for i in range(2):
        e = Embedding(hip, F32, 5000, 700, 64, text_ids(5000, 700, 40 + i))
        dout = synth.tensor(50 + i, (5000, 64), F32, "normal")
        g = e.geom()
        need = lib.fh_embedding_grad_workspace(ctypes.byref(g))
        runs.append((e, dout, g, need, hip.to_device(dout), hip.to_device(e.ids), hip.DeviceBuffer(700 * 64 * 4), hip.DeviceBuffer(need), hip.Stream()))
    hip.check(lib.fh_device_synchronize())
    for _ in range(3):
        for e, _, g, need, dd, di, dg, ws, st in runs:
            hip.check(lib.fh_embedding_grad(ctypes.byref(g), dd.value, di.value, None, dg.value, ws.value, need, st.ptr))
    for e, dout, g, need, dd, di, dg, ws, st in runs:
        st.synchronize()
        assert np.array_equal(dg.download((700, 64), np.float32), e.backward(dout))
