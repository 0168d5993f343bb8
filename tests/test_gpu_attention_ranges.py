"""Attention where its numbers reach far: scores that rise and fall from block to block, derivatives that f16 cannot hold as they are.
Against float64 (tests/attention_ref.py, which derives the bounds)."""
import numpy as np
import pytest

import attention_ref as ref
from frame_hip import synth
from test_gpu_packed_attention import BF16, E4M3, F16, NAN, Packed, Paged, say

pytestmark = pytest.mark.gpu


def levels(shape, n):
    """How high the scores of position 0 .. n - 1 lie: steps of 24 (e^24 > 2^34) from one block of 32 to the next."""
    block = np.arange(n) // 32
    return 24.0 * {"rising": block, "falling": block[::-1], "zigzag": block * 7 % 5}[shape]


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (BF16, E4M3), (F16, F16), (F16, E4M3)])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("shape", ["rising", "falling", "zigzag"])
def test_paged_scores_that_move_between_blocks(hip, dtype, cache_dtype, dh, shape):
    # every block of keys that every row sees moves the running maximum, or leaves it far above: decoding steps and chunks, whole and in parts
    say(f"paged {shape} scores, dtype {dtype}, cache {cache_dtype}, dh {dh}")
    for new in ([1, 1, 2], [40, 70, 1]):
        p = Paged(hip, dtype, cache_dtype, [640, 64, 300], new, 8, 2, dh, 16)
        scale = 1 / np.sqrt(dh)
        for b, n in enumerate(p.cached):
            rows = [synth.to_float(synth.tensor(300 + 2 * b + i, (int(n), p.kv_heads * dh), dtype, "normal", 0.25), dtype) for i in range(2)]
            rows[0][:, ::dh] = (levels(shape, int(n)) / (4.0 * scale))[:, None]  # q holds 4 there
            for rows, c, s in ((rows[0], p.kc, p.ks), (rows[1], p.vc, p.vs)):
                p.put(c, s, b, 0, synth.to_storage(rows.astype(np.float32), dtype))
        q = synth.to_float(p.q, dtype).copy()
        q[:, ::dh] = 4.0
        p.q = synth.to_storage(q.astype(np.float32), dtype)
        p.upload()
        for keys in (64, None, 1 << 20):
            p.check_attend(p.attend(max_keys=keys)[0], f"{shape}, cut for {keys}")


# dtype, tokens, heads, key heads, dims, size of dout, of v, causal
SPANS = [
    (F16, [3000], 2, 1, 64, 2.0 ** -12, 1.0, 1),    # ds about 2^-25: nothing of it is a normal f16 value, most is below the smallest one
    (F16, [1500, 700], 4, 2, 128, 2.0 ** -12, 1.0, 1),
    (F16, [2100], 1, 1, 64, 1.0, 2.0 ** -14, 0),
    (F16, [513, 1500], 3, 3, 80, 2.0 ** -9, 2.0 ** -6, 0),
    (F16, [1000, 900], 2, 1, 64, 2.0 ** 8, 2.0 ** 7, 1),    # first rows: ds up to 2^18, past the largest f16 value, gradients too
    (F16, [600, 40, 1], 2, 2, 128, 2.0 ** 8, 1.0, 1),
    (F16, [400, 64] * 30, 8, 4, 64, 2.0 ** -12, 1.0, 1),    # more tiles than CUs
    (F16, [400, 64] * 30, 32, 8, 128, 2.0 ** -12, 1.0, 1),
    (BF16, [1500], 2, 1, 64, 2.0 ** -30, 1.0, 1),
    (BF16, [700], 2, 1, 128, 2.0 ** 30, 2.0 ** 10, 0),
]


def spans_id(c):
    return f"{'f16' if c[0] == F16 else 'bf16'}-{len(c[1])}x{max(c[1])}-h{c[2]}k{c[3]}d{c[4]}-dout{c[5]:.0e}-v{c[6]:.0e}{'c' if c[7] else ''}"


@pytest.mark.parametrize("case", SPANS, ids=spans_id)
def test_packed_gradients_hold_small_and_large_derivatives(hip, case):
    # A derivative keeps its bits whatever its size: each is off by half a step of its own (ref.U), plus for f16 2^-34 of the largest one
    # that it is summed with (a power of two takes the largest to 2^10 or more, and 2^-25 there is the least step's half: 2^-35, twice).
    dtype, lens, heads, kv_heads, dh, dout, v, causal = case
    say(f"packed gradients, dout {dout:g}, v {v:g}: {case}")
    p = Packed(hip, dtype, lens, heads, kv_heads, dh, causal)
    for name, size in (("dout", dout), ("v", v)):
        p.x[name] = synth.to_storage((synth.to_float(p.x[name], dtype) * np.float32(size)).astype(np.float32), dtype)
    got = p.backward(*p.stored_forward())
    total = [np.zeros((p.rows, w)) for w in p.widths]
    tol = [np.zeros((p.rows, w)) for w in p.widths]
    u, out_step = ref.U[dtype], ref.TINY[dtype]
    for rows, h, mine, shared, q, k, vh, g, seen in p.heads_of():
        out, _, prob, _, _ = ref.attend(q, k, vh, seen, p.scale, dtype)
        dp = g @ vh.T
        ds = prob * (dp - (prob * dp).sum(1, keepdims=True))
        E = ref.softmax_error(q, k, p.scale) + (k.shape[0] + 64) * 2.0 ** -24
        # D from the stored output (off by its rounding, at least f16's least step) and from fp32 sums
        off_d = ((u + 140 * 2.0 ** -24) * np.abs(g * out) + out_step * np.abs(g)).sum(1, keepdims=True)
        off_ds = 1.02 * u * np.abs(ds) + prob * (1.02 * off_d + 140 * 2.0 ** -24 * (np.abs(g) @ np.abs(vh).T)) + 2 * E * np.abs(ds)
        off_p = 1.02 * u * prob + 2 * E * prob
        for i, (value, off, operand, factor) in enumerate(((ds, off_ds, k, p.scale), (ds.T, off_ds.T, q, p.scale),
                                                          (prob.T, off_p.T, g, 1.0))):
            off = off + 2.0 ** -34 * np.abs(value).max(1, keepdims=True) * (seen if i == 0 else seen.T)
            at = (rows, mine if i == 0 else shared)
            total[i][at] += factor * (value @ operand)
            tol[i][at] += factor * (off + (value.shape[1] + 4) * 2.0 ** -24 * np.abs(value)) @ np.abs(operand)
    for i, name in enumerate("qkv"):
        bound = ref.rounded(total[i], tol[i], dtype)
        want, have = total[i].copy(), ref.values(got[i], dtype)
        if dtype == F16:  # past the largest value: infinite, next to it either
            high = np.abs(want) > 65504
            near = np.abs(np.abs(want) - 65520) <= bound
            have[near & np.isinf(have)] = want[near & np.isinf(have)]
            want[high & ~near] = np.inf * np.sign(want[high & ~near])
        with np.errstate(invalid="ignore"):  # infinite minus infinite
            ref.check(have, want, bound, "d" + name)


INF = {F16: 0x7c00, BF16: 0x7f80}


@pytest.mark.parametrize("dtype,heads,kv_heads,dh", [(BF16, 4, 2, 64), (F16, 2, 2, 128)])
@pytest.mark.parametrize("lens", [[70, 300], [70, 300, 100] * 30])
def test_packed_rows_whose_scores_are_all_minus_infinity(hip, dtype, heads, kv_heads, dh, lens):
    # an infinite value of q against keys of the other sign: 0 / 0 in the row's softmax, and nothing for any other row
    say(f"packed scores of minus infinity, {heads} heads over {kv_heads} of {dh}, {len(lens)} sequences")
    p = Packed(hip, dtype, lens, heads, kv_heads, dh, 1)
    p.x["k"][:, 3] |= 0x8000
    clean, _ = p.forward()
    kept = p.x["q"].copy()
    for t in (0, 1, 64, 299):
        at = int(p.cu[1]) + t
        p.x["q"][at, 3] = INF[dtype]
        out, lse = p.forward()
        p.x["q"] = kept.copy()
        hit = np.zeros(out.shape, bool)
        hit[at, :dh] = True
        assert np.isnan(ref.values(out[hit], dtype)).all() and np.array_equal(out[~hit], clean[~hit])
        assert not np.isfinite(lse[at, 0])


@pytest.mark.parametrize("dtype,cache_dtype,dh", [(BF16, BF16, 64), (F16, E4M3, 128)])
@pytest.mark.parametrize("past,new", [(70, 2), (1900, 3), (0, 1), (40, 90), (1500, 130)])
def test_paged_rows_whose_scores_are_all_minus_infinity(hip, dtype, cache_dtype, dh, past, new):
    say(f"paged scores of minus infinity, {new} tokens behind {past}, cache {cache_dtype}")
    p = Paged(hip, dtype, cache_dtype, [past], [new], 4, 2, dh, 16)
    p.fill_past()
    p.put_new()
    p.kc[..., 0, 3] |= 0x80 if cache_dtype == E4M3 else 0x8000  # key head 0's keys are negative there
    p.upload()
    row = new // 2
    for keys in (64, 1 << 20):
        clean, _ = p.attend(max_keys=keys)
        p.check_attend(clean, "finite")
        kept = p.q.copy()
        p.q[row, 3] = INF[dtype]
        p.dev["q"].upload(p.q)
        out, _ = p.attend(max_keys=keys)
        hit = np.zeros(out.shape, bool)
        hit[row, :dh] = True
        assert np.isnan(ref.values(out[hit], dtype)).all() and np.array_equal(out[~hit], clean[~hit])
        # the same row over pages that do not exist sees nothing, and is zeros
        p.dev["table"].upload(np.full_like(p.table, -1))
        out, _ = p.attend(max_keys=keys)
        assert not (out & 0x7fff).any()
        p.dev["table"].upload(p.table)
        p.q = kept
        p.dev["q"].upload(p.q)


@pytest.mark.parametrize("dtype,dh", [(BF16, 64), (F16, 128)])
@pytest.mark.parametrize("past,new", [(1900, 3), (1500, 130), (100, 40)])
def test_paged_keys_at_minus_infinity_weigh_nothing(hip, dtype, dh, past, new):
    # whole parts of the context at minus infinity beside finite ones: the others' result
    say(f"paged keys at minus infinity, {new} tokens behind {past}")
    p = Paged(hip, dtype, dtype, [past], [new], 4, 2, dh, 16)
    p.fill_past()
    p.put_new()
    p.q[:, 3::dh] &= 0x7fff  # positive there
    finite = past * 2 // 3
    for i in range(finite):
        p.kc[p.slot(0, i)][:, 3] = INF[dtype] | 0x8000
    p.upload()
    slots = [p.slot(0, i) for i in range(past + new)]
    keys, vals = (np.array([p.row(c, None, s) for s in slots]) for c in (p.kc, p.vc))
    keys[:finite] = 0.0
    seen = (np.arange(past + new)[None, :] <= past + np.arange(new)[:, None]) & (np.arange(past + new) >= finite)
    for max_keys in (64, 1 << 20):
        out, _ = p.attend(max_keys=max_keys)
        for h in range(p.heads):
            mine = slice(h * dh, (h + 1) * dh)
            want, tol, *_ = ref.attend(ref.values(p.q[:, mine], dtype), keys[:, h // 2], vals[:, h // 2], seen,
                                       float(np.float32(1 / np.sqrt(dh))), dtype)
            ref.check(ref.values(out[:, mine], dtype), want, tol + 2.0 ** -20 * np.abs(want), f"head {h}")


@pytest.mark.parametrize("dtype,dh", [(F16, 64), (F16, 128), (BF16, 64), (BF16, 128)])
def test_e4m3_cache_keeps_the_largest_values_finite(hip, dtype, dh):
    # The largest values of a type are nearest to 256 times their row's scale, which is past it (f16: 65536; bf16: 2^128): they come back as the largest
    # there is, and attention over them is finite.
    say(f"e4m3 cache of the largest values, dtype {dtype}, dh {dh}")
    top = 0x7bff if dtype == F16 else 0x7f7f
    rows = 40
    bits = np.random.default_rng(5).integers(top - 3, top + 1, (rows, dh)).astype(np.uint16)
    bits[:, ::2] |= 0x8000
    bits[0, 1] = NAN[dtype]
    # (bf16: over one row; the fp32 sum of more has no room for them)
    for past, new in ((0, [rows]), (rows - 1, [1]), (rows - 6, [6])) if dtype == F16 else ((0, [1]),):
        rows = past + sum(new)
        bits = bits[:rows]
        p = Paged(hip, dtype, E4M3, [past], new, 2, 1, dh, 16)
        p.k[:] = 0
        for c, s, all_rows in ((p.kc, p.ks, np.zeros_like(bits)), (p.vc, p.vs, bits)):
            p.put(c, s, 0, 0, all_rows)
        r = p.upload()
        back = [hip.to_device(np.zeros((rows, dh), np.uint16)) for _ in range(2)]
        cu = hip.to_device(np.array([0, rows], np.int32))
        hip.check(hip.lib().fh_kv_cache_read(r, back[0].value, dh, back[1].value, dh, rows, cu.value, None))
        got = back[1].download((rows, dh), np.uint16)
        nan = (bits & 0x7fff) == NAN[dtype]
        assert np.array_equal(got[~nan], top | (bits[~nan] & 0x8000)) and np.isnan(ref.values(got[nan], dtype)).all()
        for max_new in (1, 64):  # both forms; equal scores, so the mean of the values
            out, _ = p.attend(max_new=max_new)
            out = ref.values(out, dtype)
            want = np.where(np.arange(dh) % 2, 1.0, -1.0) * float(ref.values(np.array([top], np.uint16), dtype)[0])
            keep = np.arange(2 * dh) % dh != 1
            assert np.allclose(out[:, keep], np.tile(want, 2)[keep], rtol=4 * ref.U[dtype], atol=0)
            assert np.isnan(out[:, ~keep]).all()
