"""Graphs of packed_attention that the CPU and the GPU tests share."""
from __future__ import annotations

import numpy as np

import attention_ref as ref
from frame_hip import graphs, synth


def attention_graph(dtype, tokens, batch, heads, kv_heads, dh, causal=True, device="cpu", loss=False, **attrs):
    """out = packed_attention(q, k, v, cu_seqlens); loss: sum(out * w) over everything, w the fifth input."""
    g = graphs.Graph(device)
    q, k, v = (g.input(dtype, (tokens, h * dh)) for h in (heads, kv_heads, kv_heads))
    out = g.packed_attention(q, k, v, g.input(graphs.I32, (batch + 1,)), heads, kv_heads, causal, **attrs)
    if loss:
        w = g.input(dtype, out.shape)
        g.output(g.op("sum", [g.mul(out, w)], (), {"axes": []}))
    else:
        g.output(out)
    return g


def inputs(dtype, cu, tokens, heads, kv_heads, dh, seed=1):
    """q, k, v, cu_seqlens and dout (the loss's w)."""
    arrays = [synth.tensor(seed + i, (tokens, h * dh), dtype, "normal") for i, h in enumerate((heads, kv_heads, kv_heads, heads))]
    return arrays[:3] + [np.asarray(cu, np.int32), arrays[3]]


def check(outs, ins, dtype, heads, kv_heads, dh, causal, scale=None):
    """outs: [out] or [out, dq, dk, dv] against float64 (tests/attention_ref.py); rows outside the sequences are zeros."""
    q, k, v, cu, dout = ins
    scale = 1.0 / np.sqrt(dh) if scale is None else scale
    shapes = [q.shape, q.shape, k.shape, k.shape]
    total, tol = ([np.zeros(s) for s in shapes] for _ in range(2))
    for b in range(len(cu) - 1):
        rows, n = slice(cu[b], cu[b + 1]), cu[b + 1] - cu[b]
        seen = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
        for h in range(heads if n else 0):
            j = h // (heads // kv_heads)
            mine, shared = slice(h * dh, (h + 1) * dh), slice(j * dh, (j + 1) * dh)
            qh, kh, vh, gh = (ref.values(t[rows, c], dtype) for t, c in ((q, mine), (k, shared), (v, shared), (dout, mine)))
            out, off, p, _, _ = ref.attend(qh, kh, vh, seen, scale, dtype)
            total[0][rows, mine], tol[0][rows, mine] = out, off
            for i, (g, t) in enumerate(ref.gradients(qh, kh, vh, gh, out, p, scale, dtype)):
                at = (rows, mine if i == 0 else shared)
                total[1 + i][at] += g
                tol[1 + i][at] += t
    for i in range(len(outs)):
        bound = tol[i] if i == 0 else ref.rounded(total[i], tol[i], dtype)
        ref.check(ref.values(outs[i], dtype), total[i], bound, ("out", "dq", "dk", "dv")[i])
        assert not (outs[i][cu[-1]:] & 0x7fff).any() and not (outs[i][:cu[0]] & 0x7fff).any()


def decoder_inputs(shapes, cu, tokens, d_model, dtype, seed=701, train=False):
    arrays = [synth.tensor(seed, (tokens, d_model), dtype, "normal"), np.asarray(cu, np.int32)]
    for i, s in enumerate(shapes):
        if len(s) == 1:  # layer-norm gamma = 1 + noise, beta = noise
            noise = synth.tensor(seed + 1 + i, s, 0, "normal", 0.02)
            arrays.append(synth.to_storage((noise + (1.0 if i in (0, 6) else 0.0)).astype(np.float32), dtype))
        else:
            arrays.append(synth.tensor(seed + 1 + i, s, dtype, "normal", 0.02))
    if train:
        arrays.append(synth.tensor(seed + 50, (tokens, d_model), dtype, "normal"))
    return arrays
