"""What the packed and paged attention entry points refuse, decided on the host before any launch (no GPU needed), and the float64
reference's own gradients against differences."""
import ctypes

import numpy as np
import pytest

import attention_ref as ref
from frame_hip import abi

F32, F16, BF16 = 0, 2, 3
P = 4096  # an aligned address that nothing reads: every call here is refused, or has nothing to do


def geom(**over):
    f = dict(dtype=BF16, causal=1, tokens=64, batch=2, heads=4, kv_heads=2, dh=64, q_stride=256, k_stride=128, v_stride=128,
             out_stride=256, scale=0.125)
    f.update(over)
    return abi.PackedAttention(**f)


def cache(**over):
    f = dict(dtype=BF16, cache_dtype=abi.E4M3, pages=8, page_size=16, kv_heads=2, dh=64, k=P, v=P, k_scale=P, v_scale=P, batch=2,
             block_table=P, table_stride=4, kv_lens=P)
    f.update(over)
    return abi.PagedCache(**f)


INVALID, UNIMPLEMENTED = 1, 4
BAD_GEOM = [
    (dict(dtype=F32), UNIMPLEMENTED), (dict(dh=60), UNIMPLEMENTED), (dict(dh=136, q_stride=1024, out_stride=1024, k_stride=512,
     v_stride=512), UNIMPLEMENTED), (dict(dh=0), UNIMPLEMENTED), (dict(tokens=-1), INVALID), (dict(batch=-1), INVALID),
    (dict(heads=3), INVALID), (dict(kv_heads=0), INVALID), (dict(causal=2), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(q_stride=248), INVALID), (dict(k_stride=120), INVALID), (dict(v_stride=0), INVALID), (dict(out_stride=260), INVALID),
    (dict(tokens=2 ** 31), INVALID), (dict(tokens=2 ** 30), INVALID),
]


@pytest.mark.parametrize("over,code", BAD_GEOM, ids=lambda x: str(x))
def test_packed_geometry_is_refused(over, code):
    lib, g = abi.lib(), geom(**over)
    assert lib.fh_attention_packed_fwd(ctypes.byref(g), P, P, P, P, P, P, None) == code
    assert abi.lib().fh_last_error()
    assert lib.fh_attention_packed_grad_workspace(ctypes.byref(g)) == -1
    assert lib.fh_attention_packed_grad(ctypes.byref(g), *[P] * 11, 1 << 40, None) == code


def test_packed_pointers_are_refused():
    lib, g = abi.lib(), geom()
    r = ctypes.byref(g)
    assert lib.fh_attention_packed_fwd(None, P, P, P, P, P, P, None) == INVALID
    for i in range(5):  # q, k, v, cu_seqlens, out
        for bad in (None, P + 2):
            args = [P] * 5
            args[i] = bad
            assert lib.fh_attention_packed_fwd(r, *args, None, None) == INVALID, (i, bad)
    assert lib.fh_attention_packed_fwd(r, P, P, P, P, P, P + 2, None) == INVALID  # lse
    need = lib.fh_attention_packed_grad_workspace(r)
    assert need > 0
    assert lib.fh_attention_packed_grad(r, *[P] * 11, need - 1, None) == INVALID
    for i in range(11):
        for bad in (None, P + 2):
            args = [P] * 11
            args[i] = bad
            assert lib.fh_attention_packed_grad(r, *args, need, None) == INVALID, (i, bad)


def test_nothing_to_do_is_ok():
    lib = abi.lib()
    for over in (dict(tokens=0), dict(batch=0)):
        g = geom(**over)
        assert lib.fh_attention_packed_fwd(ctypes.byref(g), None, None, None, None, None, None, None) == 0
        assert lib.fh_attention_packed_grad(ctypes.byref(g), *[None] * 11, 0, None) == 0
    c = cache()
    assert lib.fh_kv_cache_write(ctypes.byref(c), None, 128, None, 128, 0, None, None) == 0
    c = cache(batch=0, block_table=None, kv_lens=None)
    assert lib.fh_kv_cache_read(ctypes.byref(c), None, 128, None, 128, 5, None, None) == 0
    assert lib.fh_attention_paged(ctypes.byref(c), None, 256, None, 256, 5, 4, None, 0.125, 1, 64, None, 0, None) == 0


BAD_CACHE = [
    (dict(dtype=F32), UNIMPLEMENTED), (dict(cache_dtype=F16), UNIMPLEMENTED), (dict(cache_dtype=8), UNIMPLEMENTED),
    (dict(dh=4), UNIMPLEMENTED), (dict(dh=192), UNIMPLEMENTED), (dict(page_size=24), UNIMPLEMENTED),
    (dict(page_size=0), UNIMPLEMENTED), (dict(page_size=1 << 17), UNIMPLEMENTED), (dict(kv_heads=0), INVALID),
    (dict(batch=-1), INVALID), (dict(pages=-1), INVALID), (dict(table_stride=-1), INVALID), (dict(table_stride=1 << 28), INVALID),
    (dict(kv_lens=None), INVALID), (dict(block_table=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(k_scale=None), INVALID), (dict(v_scale=None), INVALID), (dict(k=P + 8), INVALID), (dict(kv_lens=P + 1), INVALID),
]


@pytest.mark.parametrize("over,code", BAD_CACHE, ids=lambda x: str(x))
def test_cache_descriptor_is_refused(over, code):
    lib, c = abi.lib(), cache(**over)
    r = ctypes.byref(c)
    assert lib.fh_kv_cache_write(r, P, 1024, P, 1024, 4, P, None) == code
    assert lib.fh_kv_cache_read(r, P, 1024, P, 1024, 4, P, None) == code
    assert lib.fh_attention_paged_workspace(r, 4, 4, 1, 64) == -1
    assert lib.fh_attention_paged(r, P, 1024, P, 1024, 4, 4, P, 0.125, 1, 64, P, 1 << 40, None) == code


def test_cache_calls_are_refused():
    lib, c = abi.lib(), cache()
    r = ctypes.byref(c)
    for fn in (lib.fh_kv_cache_write, lib.fh_kv_cache_read):
        assert fn(None, P, 128, P, 128, 4, P, None) == INVALID
        for args in ((None, 128, P, 128, 4, P), (P, 128, None, 128, 4, P), (P, 128, P, 128, 4, None), (P + 8, 128, P, 128, 4, P),
                     (P, 120, P, 128, 4, P), (P, 128, P, 132, 4, P), (P, 128, P, 128, -1, P), (P, 128, P, 128, 1 << 31, P),
                     (P, 128, P, 128, 4, P + 2)):
            assert fn(r, *args, None) == INVALID, args

    def paged(q=P, qs=256, out=P, os=256, tokens=4, heads=4, cu=P, scale=0.125, new=1, keys=64, ws=P, n=1 << 40):
        return lib.fh_attention_paged(r, q, qs, out, os, tokens, heads, cu, scale, new, keys, ws, n, None)

    for bad in (dict(q=None), dict(out=None), dict(cu=None), dict(q=P + 8), dict(out=P + 8), dict(cu=P + 2), dict(qs=248),
                dict(os=260), dict(tokens=-1), dict(heads=3), dict(heads=0), dict(scale=0.0), dict(scale=float("nan")),
                dict(new=-1), dict(keys=-1), dict(tokens=1 << 31)):
        assert paged(**bad) == INVALID, bad
    c = cache(table_stride=1 << 16)
    r = ctypes.byref(c)
    need = lib.fh_attention_paged_workspace(r, 4, 4, 1, 1 << 20)
    assert need > 0  # few rows over a long context: the keys are cut into parts
    assert paged(keys=1 << 20, n=need - 1) == INVALID
    assert paged(keys=1 << 20, ws=None, n=need) == INVALID
    assert paged(keys=1 << 20, ws=P + 8, n=need) == INVALID


def test_positions_fit_32_bits():
    lib = abi.lib()
    c = cache(table_stride=0x7fff0000 // 16)
    assert lib.fh_attention_paged_workspace(ctypes.byref(c), 1, 2, 1, 1) >= 0
    c.table_stride += 1
    assert lib.fh_attention_paged_workspace(ctypes.byref(c), 1, 2, 1, 1) == -1


def test_reference_gradients_are_the_differences():
    rng = np.random.default_rng(3)
    n, dh, scale = 7, 8, 0.4
    q, k, v, dout = (rng.standard_normal((n, dh)) for _ in range(4))
    seen = np.tril(np.ones((n, n), bool))

    def loss(q, k, v):
        return float((ref.attend(q, k, v, seen, scale, BF16)[0] * dout).sum())

    out, _, p, _, _ = ref.attend(q, k, v, seen, scale, BF16)
    grads = [g for g, _ in ref.gradients(q, k, v, dout, out, p, scale, BF16)]
    h = 1e-5  # the differences are off by about h^2 + 1e-16 / h
    for which, g in enumerate(grads):
        for i in np.ndindex(n, dh):
            args = [q.copy(), k.copy(), v.copy()]
            args[which][i] += h
            up = loss(*args)
            args[which][i] -= 2 * h
            assert abs((up - loss(*args)) / (2 * h) - g[i]) < 1e-7
