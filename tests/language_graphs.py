"""Graphs of embedding and vocab_loss that the CPU and the GPU tests share."""
from __future__ import annotations

import numpy as np

import language_ref as ref
from frame_hip import graphs, host, synth


def loss_graph(dtype, tokens, vocab, dim, mean=True, device="cpu"):
    g = graphs.Graph(device)
    x, w, t = g.input(dtype, (tokens, dim)), g.input(dtype, (vocab, dim)), g.input(graphs.I32, (tokens,))
    g.output(g.vocab_loss(x, w, t, mean))
    return g


def embedding_graph(dtype, tokens, vocab, dim, scale=1.0, device="cpu", loss=False):
    """out = embedding(table, ids); loss: sum(out * w), w the third input."""
    g = graphs.Graph(device)
    out = g.embedding(g.input(dtype, (vocab, dim)), g.input(graphs.I32, (tokens,)), scale)
    g.output(g.op("sum", [g.mul(out, g.input(dtype, out.shape))], (), {"axes": []}) if loss else out)
    return g


def tied_graph(dtype, tokens, vocab, dim, device="cpu"):
    """vocab_loss(embedding(table, ids), table, targets): both gradients of one table."""
    g = graphs.Graph(device)
    table, ids, t = g.input(dtype, (vocab, dim)), g.input(graphs.I32, (tokens,)), g.input(graphs.I32, (tokens,))
    g.output(g.vocab_loss(g.embedding(table, ids, 2.0), table, t))
    return g


def ids(rng, tokens, vocab, outside):
    out = rng.integers(0, vocab, tokens)
    bad = rng.random(tokens) < outside
    out[bad] = rng.choice([-1, vocab, 2 ** 31 - 1], bad.sum())
    return out.astype(np.int32)


def loss_inputs(dtype, tokens, vocab, dim, seed=1, outside=0.2):
    return [synth.tensor(seed, (tokens, dim), dtype, "normal"), synth.tensor(seed + 1, (vocab, dim), dtype, "normal", 1.5 / np.sqrt(dim)),
            ids(np.random.default_rng(seed), tokens, vocab, outside)]


def check_loss(outs, ins, dtype, mean):
    """outs: [loss] or [loss, dx, dw] (of a loss' gradient of 1) against float64."""
    x, w, targets = ins
    want = ref.Loss(ref.values(x, dtype), ref.values(w, dtype), targets.astype(np.int64), mean, dtype, dtype)
    assert abs(float(ref.values(outs[0], dtype).reshape(())) - want.loss) <= want.loss_tol
    for name, got, (total, tol) in zip(("dx", "dw"), outs[1:], want.gradients(1.0)):
        ref.check(ref.values(got, dtype), total, tol, name)


def check_embedding(outs, ins, dtype, scale):
    """outs: [out] or [out, dtable] against float64."""
    table, which, w = ins
    want, tol = ref.embed(ref.values(table, dtype), which.astype(np.int64), scale, dtype)
    ref.check(ref.values(outs[0], dtype), want, tol, "out")
    if len(outs) > 1:
        total, tol = ref.embed_grad(ref.values(w, dtype), which.astype(np.int64), table.shape[0], scale, None, dtype)
        ref.check(ref.values(outs[1], dtype), total, tol, "dtable")


def embedding_inputs(dtype, tokens, vocab, dim, seed=1, outside=0.2):
    return [synth.tensor(seed, (vocab, dim), dtype, "normal"), ids(np.random.default_rng(seed), tokens, vocab, outside),
            synth.tensor(seed + 2, (tokens, dim), dtype, "normal")]


def model_inputs(shapes, cu, tokens, vocab, dtype, seed=901):
    """ids, cu_seqlens, targets (the next token of the same sequence, none for the last), then the parameters."""
    rng = np.random.default_rng(seed)
    which = rng.integers(0, vocab, tokens).astype(np.int32)
    targets = np.full(tokens, -1, np.int32)
    for b, e in zip(cu[:-1], cu[1:]):
        targets[b:max(e - 1, b)] = which[b + 1:e]
    arrays = [which, np.asarray(cu, np.int32), targets]
    for i, s in enumerate(shapes):
        std = 1.0 if len(s) == 2 and s[0] == vocab else 0.05
        noise = synth.tensor(seed + 1 + i, s, 0, "normal", 0.02 if len(s) == 1 else std / (np.sqrt(s[1]) if std == 1.0 else 1.0))
        first = len(s) == 1 and (i == 0 or len(shapes[i - 1]) != 1)  # a norm's gamma stands before its beta
        arrays.append(synth.to_storage((noise + (1.0 if first else 0.0)).astype(np.float32), dtype))
    return arrays


def backward(g, wrt):
    return host.backward(g.text(), 0, wrt)
