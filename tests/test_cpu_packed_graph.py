"""packed_attention as a graph op, on the CPU: its contract, the training graph that differentiates it, what the hip backend plans for
it, and the oracle's kernels against float64."""
import numpy as np
import pytest

import oracle_lib as orc
import packed_graphs as pg
from frame_hip import graphs, host

F32, F16, BF16 = 0, 2, 3


@pytest.fixture(scope="module", autouse=True)
def cpu_backend():
    orc.load_cpu_backend()


CASES = [(BF16, [0, 5, 5, 13], 15, 4, 2, 8, True), (F16, [2, 9, 10], 10, 2, 2, 16, False), (BF16, [0, 1], 1, 3, 1, 8, True)]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_oracle_matches_float64(case):
    dtype, cu, tokens, heads, kv_heads, dh, causal = case
    ins = pg.inputs(dtype, cu, tokens, heads, kv_heads, dh)
    (out,) = orc.run_graph_cpu(pg.attention_graph(dtype, tokens, len(cu) - 1, heads, kv_heads, dh, causal), ins[:4])
    loss = pg.attention_graph(dtype, tokens, len(cu) - 1, heads, kv_heads, dh, causal, loss=True)
    grads = orc.run_graph_cpu(host.backward(loss.text(), 0, [0, 1, 2]), ins)[1:]
    pg.check([out, *grads], ins, dtype, heads, kv_heads, dh, causal)


def test_gradient_is_one_node_and_integer_inputs_have_none():
    text = pg.attention_graph(BF16, 12, 2, 4, 2, 8, loss=True).text()
    back = host.backward(text, 0, [0, 1, 2])
    assert back.count(" packed_attention_grad_internal(") == 1 and back.count(" packed_attention(") == 1
    assert host.roundtrip(back) == back
    with pytest.raises(host.FrameError, match="not of a floating-point type"):
        host.backward(text, 0, [0, 3])


def test_two_attentions_share_one_cu_seqlens():
    g = graphs.Graph("cpu")
    q, k, v = (g.input(BF16, (6, 16)) for _ in range(3))
    cu, w = g.input(graphs.I32, (3,)), g.input(BF16, (6, 16))
    y = g.packed_attention(g.packed_attention(q, k, v, cu, 2, 2), k, v, cu, 2, 2)
    g.output(g.op("sum", [g.mul(y, w)], (), {"axes": []}))
    back = host.backward(g.text(), 0, [0, 1, 2])
    assert back.count(" packed_attention_grad_internal(") == 2
    ins = pg.inputs(BF16, [0, 4, 6], 6, 2, 2, 8)
    assert len(orc.run_graph_cpu(back, ins)) == 4
    low = host.hip_lowered(back.replace("@cpu:0", "@hip:0"))
    assert low.count(" hip_packed_attention_internal(") == 2 and low.count(" hip_packed_attention_grad_internal(") == 2


@pytest.mark.parametrize("opt", [0, 1])
def test_hip_plans_the_gradient_with_the_forwards_statistics(opt):
    text = pg.attention_graph(BF16, 300, 2, 4, 2, 64, device="hip", loss=True).text()
    low = host.hip_lowered(host.backward(text, 0, [0, 1, 2]), opt)
    assert low.count(" hip_packed_attention_internal(") == 1 and low.count(" hip_packed_attention_grad_internal(") == 1
    assert " packed_attention(" not in low and "float32[300,4]" in low
    assert " packed_attention(" in host.hip_lowered(text, opt)  # a forward graph keeps no statistics


@pytest.mark.parametrize("change,message", [
    (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=3), "multiple of kv_heads"), (dict(scale=0.0), "must be positive"),
    (dict(scale=-1.0), "must be positive"), (dict(heads=0), "multiple of kv_heads"),
])
def test_attributes_are_checked(change, message):
    args = dict(heads=4, kv_heads=2, scale=0.5)
    args.update(change)
    g = graphs.Graph("cpu")
    q, k = g.input(BF16, (6, 32)), g.input(BF16, (6, 16))
    g.output(g.packed_attention(q, k, k, g.input(graphs.I32, (2,)), args["heads"] or 4, args["kv_heads"], True, args["scale"]))
    text = g.text().replace("heads=4,", "heads=0,") if args["heads"] == 0 else g.text()
    with pytest.raises(host.FrameError, match=message):
        host.backward(loss_of(text), 0, [0])


def loss_of(text):
    """The graph's output summed, so that differentiating it runs the op's own checks."""
    lines = text.strip().splitlines()
    last = lines[-2].split(" = ")[0]
    shape = lines[-2].rsplit(": ", 1)[1]
    n = int(last[1:])
    dtype = shape.split("[")[0]
    lines[-1] = f"%{n + 1} = sum({last}) {{axes=[]}} : {dtype}[]@cpu:0"
    return "\n".join(lines + [f"graph_output(%{n + 1})"]) + "\n"


@pytest.mark.parametrize("shapes,message", [
    (((6, 32), (6, 16), (5, 16), (2,)), "requires k and v to be"), (((6, 32), (6, 8), (6, 8), (2,)), "requires k and v to be"),
    (((6, 33), (6, 16), (6, 16), (2,)), "multiple of heads"), (((6, 32), (6, 16), (6, 16), (2, 1)), "cu_seqlens"),
    (((6, 32), (6, 16), (6, 16), (0,)), "cu_seqlens"), (((192,), (6, 16), (6, 16), (2,)), "rank-2"),
])
def test_shapes_are_checked(shapes, message):
    g = graphs.Graph("cpu")
    vals = [g.input(graphs.I32 if i == 3 else BF16, s) for i, s in enumerate(shapes)]
    g.output(g.op("packed_attention", vals, shapes[0], {"heads": 4, "kv_heads": 2, "causal": True, "scale": 0.5}))
    with pytest.raises(host.FrameError, match=message):
        host.backward(loss_of(g.text()), 0, [0])


def test_cu_seqlens_is_int32():
    g = graphs.Graph("cpu")
    q, k, cu = g.input(BF16, (6, 32)), g.input(BF16, (6, 16)), g.input(BF16, (2,))
    g.output(g.packed_attention(q, k, k, cu, 4, 2))
    with pytest.raises(host.FrameError, match="int32"):
        host.backward(loss_of(g.text()), 0, [0])


def test_decoder_block_trains_on_the_oracle():
    tokens, d, cu = 20, 32, [0, 7, 7, 20]
    g, shapes = graphs.decoder_block(tokens, 3, d_model=d, heads=4, kv_heads=2, ffn=48, dtype=BF16, device="cpu", train=True)
    back = host.backward(g.text(), 0, list(range(2, 2 + len(shapes))))
    outs = orc.run_graph_cpu(back, pg.decoder_inputs(shapes, cu, tokens, d, BF16, train=True))
    assert len(outs) == 1 + len(shapes) and [o.shape for o in outs[1:]] == shapes
    from frame_hip import synth
    assert all(np.isfinite(synth.to_float(o, BF16)).all() and synth.to_float(o, BF16).any() for o in outs)
