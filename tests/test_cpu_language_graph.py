"""embedding and vocab_loss as graph ops, on the CPU: their contracts, the training graphs that differentiate them, what the hip backend
plans for them, and the oracle's kernels against float64."""
import numpy as np
import pytest

import language_graphs as lg
import oracle_lib as orc
from frame_hip import graphs, host, synth
from test_cpu_packed_graph import loss_of

F32, F16, BF16 = 0, 2, 3


@pytest.fixture(scope="module", autouse=True)
def cpu_backend():
    orc.load_cpu_backend()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("mean", [True, False])
def test_oracle_loss_matches_float64(dtype, mean):
    ins = lg.loss_inputs(dtype, 9, 13, 8)
    g = lg.loss_graph(dtype, 9, 13, 8, mean)
    (loss,) = orc.run_graph_cpu(g, ins)
    grads = orc.run_graph_cpu(lg.backward(g, [0, 1]), ins)[1:]
    lg.check_loss([loss, *grads], ins, dtype, mean)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_oracle_embedding_matches_float64(dtype):
    ins = lg.embedding_inputs(dtype, 11, 5, 7)
    (out,) = orc.run_graph_cpu(lg.embedding_graph(dtype, 11, 5, 7, 0.5), ins[:2])
    (grad,) = orc.run_graph_cpu(lg.backward(lg.embedding_graph(dtype, 11, 5, 7, 0.5, loss=True), [0]), ins)[1:]
    lg.check_embedding([out, grad], ins, dtype, 0.5)


def test_gradients_are_one_node_and_integer_inputs_have_none():
    back = lg.backward(lg.loss_graph(BF16, 6, 9, 8), [0, 1])
    assert back.count(" vocab_loss_grad_internal(") == 1 and host.roundtrip(back) == back
    back = lg.backward(lg.embedding_graph(BF16, 6, 9, 8, loss=True), [0])
    assert back.count(" embedding_grad_internal(") == 1 and host.roundtrip(back) == back
    for g, integer in ((lg.loss_graph(BF16, 6, 9, 8), 2), (lg.embedding_graph(BF16, 6, 9, 8, loss=True), 1)):
        with pytest.raises(host.FrameError, match="not of a floating-point type"):
            lg.backward(g, [0, integer])


@pytest.mark.parametrize("opt", [0, 1])
def test_hip_plans_workspaces_and_hands_the_gradient_the_rows_log_sum_exps(opt):
    low = host.hip_lowered(lg.backward(lg.loss_graph(BF16, 300, 1000, 64, device="hip"), [0, 1]), opt)
    assert low.count(" hip_vocab_loss_internal(") == 1 and low.count(" hip_vocab_loss_grad_internal(") == 1 and "float32[300]" in low
    assert " vocab_loss(" not in low and " vocab_loss_grad_internal(" not in low
    assert low.count(" hip_vocab_loss_internal(") == host.hip_lowered(lg.loss_graph(BF16, 300, 1000, 64, device="hip").text(), opt).count(
        " hip_vocab_loss_internal(")
    low = host.hip_lowered(lg.backward(lg.embedding_graph(F32, 300, 1000, 64, device="hip", loss=True), [0]), opt)
    assert low.count(" hip_embedding_grad_internal(") == 1 and " embedding_grad_internal(" not in low


GRADIENT_ALONE = ("%0 = graph_input() : bfloat16[40,64]@hip:0\n%1 = graph_input() : bfloat16[90,64]@hip:0\n%2 = graph_input() : int32[40]@hip:0\n"
                  "%3 = graph_input() : bfloat16[]@hip:0\n%4 = graph_input() : bfloat16[]@hip:0\n"
                  "%5, %6 = vocab_loss_grad_internal(%0, %1, %2, %3, %4) {mean=true} : bfloat16[40,64]@hip:0, bfloat16[90,64]@hip:0\n"
                  "graph_output(%5)\ngraph_output(%6)\n")


def test_hip_forms_the_log_sum_exps_of_a_gradient_without_its_forward():
    low = host.hip_lowered(GRADIENT_ALONE, 1)
    assert low.count(" hip_vocab_loss_internal(") == 1 and low.count(" hip_vocab_loss_grad_internal(") == 1 and "float32[40]" in low


def test_hip_sums_a_tied_tables_gradients_in_one():
    back = lg.backward(lg.tied_graph(BF16, 300, 1000, 64, device="hip"), [0])
    assert back.count(" add(") == 1
    low = host.hip_lowered(back, 1)
    assert " add(" not in low and low.count(" hip_embedding_grad_internal(") == 1
    line = next(x for x in low.splitlines() if " hip_embedding_grad_internal(" in x)
    assert line.split("hip_embedding_grad_internal(")[1].split(")")[0].count("%") == 3
    assert host.hip_lowered(back, 0).count(" add(") == 1
    # a gradient that is an output as well keeps its add
    text = ("%0 = graph_input() : bfloat16[6,8]@hip:0\n%1 = graph_input() : int32[6]@hip:0\n%2 = graph_input() : bfloat16[9,8]@hip:0\n"
            "%3 = embedding_grad_internal(%0, %1) {scale=1.0, table_shape=shape[9,8]} : bfloat16[9,8]@hip:0\n"
            "%4 = add(%2, %3) : bfloat16[9,8]@hip:0\ngraph_output(%4)\n")
    assert " add(" not in host.hip_lowered(text, 1)
    assert host.hip_lowered(text + "graph_output(%3)\n", 1).count(" add(") == 1


def test_two_embeddings_of_one_table():
    g = graphs.Graph("cpu")
    table, a, b = g.input(BF16, (9, 8)), g.input(graphs.I32, (5,)), g.input(graphs.I32, (5,))
    y = g.add(g.embedding(table, a), g.embedding(table, b, 0.5))
    g.output(g.op("sum", [g.mul(y, g.input(BF16, (5, 8)))], (), {"axes": []}))
    back = lg.backward(g, [0])
    assert back.count(" embedding_grad_internal(") == 2
    low = host.hip_lowered(back.replace("@cpu:0", "@hip:0"), 1)
    # one on top of the other
    calls = [x.split("hip_embedding_grad_internal(")[1].split(")")[0].count("%") for x in low.splitlines() if " hip_embedding_grad_internal(" in x]
    assert sorted(calls) == [2, 3]


@pytest.mark.parametrize("shapes,types,message", [
    (((6, 8), (9, 16), (6,)), (BF16, BF16, graphs.I32), "same second dimension"), (((6, 8), (9, 8), (5,)), (BF16, BF16, graphs.I32), "int32"),
    (((6, 8), (9, 8), (6,)), (BF16, BF16, BF16), "int32"), (((6, 8), (9, 8), (6,)), (BF16, F16, graphs.I32), "same dtype"),
    (((48,), (9, 8), (6,)), (BF16, BF16, graphs.I32), "rank-2"), (((6, 8), (9, 8), (6, 1)), (BF16, BF16, graphs.I32), "int32"),
])
def test_loss_shapes_are_checked(shapes, types, message):
    g = graphs.Graph("cpu")
    g.output(g.op("vocab_loss", [g.input(t, s) for t, s in zip(types, shapes)], (), {"mean": True}))
    with pytest.raises(host.FrameError, match=message):
        lg.backward(g, [0])


@pytest.mark.parametrize("shapes,types,attrs,message", [
    (((9, 8), (6, 1)), (BF16, graphs.I32), {"scale": 1.0}, "int32"), (((9, 8), (6,)), (BF16, BF16), {"scale": 1.0}, "int32"),
    (((72,), (6,)), (BF16, graphs.I32), {"scale": 1.0}, "rank-2"), (((9, 8), (6,)), (BF16, graphs.I32), {}, "scale"),
])
def test_embedding_shapes_are_checked(shapes, types, attrs, message):
    g = graphs.Graph("cpu")
    g.output(g.op("embedding", [g.input(t, s) for t, s in zip(types, shapes)], (6, 8), attrs))
    with pytest.raises(host.FrameError, match=message):
        host.backward(loss_of(g.text()), 0, [0])


@pytest.mark.parametrize("tied", [True, False])
def test_language_model_trains_on_the_oracle(tied):
    tokens, vocab, d, cu = 20, 37, 32, [0, 7, 7, 20]
    g, shapes = graphs.language_model(tokens, 3, vocab, d_model=d, heads=4, kv_heads=2, ffn=48, layers=2, tied=tied, device="cpu")
    outs = orc.run_graph_cpu(lg.backward(g, list(range(3, 3 + len(shapes)))), lg.model_inputs(shapes, cu, tokens, vocab, BF16))
    assert len(outs) == 1 + len(shapes) and [o.shape for o in outs[1:]] == shapes
    assert all(np.isfinite(synth.to_float(o, BF16)).all() and synth.to_float(o, BF16).any() for o in outs)


def test_language_models_gradient_is_the_losses_slope():
    """float32 on the oracle: the loss along a parameter's gradient, against differences."""
    tokens, vocab, d, cu = 12, 19, 16, [0, 5, 12]
    g, shapes = graphs.language_model(tokens, 2, vocab, d_model=d, heads=2, kv_heads=1, ffn=24, dtype=F32, device="cpu")
    ins = lg.model_inputs(shapes, cu, tokens, vocab, F32)
    grads = orc.run_graph_cpu(lg.backward(g, list(range(3, 3 + len(shapes)))), ins)[1:]
    for i in (0, 3, len(shapes) - 1):  # the tied table, wq, the last norm's beta
        way = grads[i].astype(np.float64) / np.sqrt((grads[i].astype(np.float64) ** 2).sum())
        ends = []
        for h in (1e-2, -1e-2):
            moved = list(ins)
            moved[3 + i] = (ins[3 + i] + h * way).astype(np.float32)
            ends.append(float(orc.run_graph_cpu(g, moved)[0].reshape(())))
        slope = float((grads[i] * way).sum())
        # the differences' own error: third derivatives of order the slope times h^2, and a loss of about 3 rounded to float32 over 2 h
        assert abs((ends[0] - ends[1]) / 2e-2 - slope) <= 0.02 * abs(slope) + 4 * 3.0 * 2.0 ** -24 / 2e-2
