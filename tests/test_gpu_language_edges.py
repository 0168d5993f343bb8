"""embedding and vocab_loss at the ends of what they take, through graphs: no tokens, tensors that start inside a block, one gradient wanted of two,
two losses on one table, logits that are infinite."""
import numpy as np
import pytest

import language_graphs as lg
import language_ref as ref
import oracle_lib as orc
from frame_hip import graphs, host, synth
from test_gpu_vocab_loss import Loss, say

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 2, 3


@pytest.fixture(scope="module", autouse=True)
def dev():
    assert host.device_count("hip") >= 1, "no hip device"
    orc.load_cpu_backend()


@pytest.mark.parametrize("opt", [0, 1])
def test_no_tokens(opt):
    say(f"no tokens opt={opt}")
    ins = lg.loss_inputs(BF16, 0, 90, 64)
    loss, dx, dw = host.compile(lg.backward(lg.loss_graph(BF16, 0, 90, 64, device="hip"), [0, 1]), "hip", opt).run(ins)
    assert not synth.to_float(loss, BF16).any() and dx.shape == (0, 64) and dw.shape == (90, 64) and not dw.any()
    for dtype in (F32, BF16):
        ins = lg.embedding_inputs(dtype, 0, 50, 24)
        (out,) = host.compile(lg.embedding_graph(dtype, 0, 50, 24, device="hip"), "hip", opt).run(ins[:2])
        assert out.shape == (0, 24)
        name = graphs.DTYPE_NAME[dtype]
        text = (f"%0 = graph_input() : {name}[0,24]@hip:0\n%1 = graph_input() : int32[0]@hip:0\n"
                f"%2 = embedding_grad_internal(%0, %1) {{scale=2.0, table_shape=shape[50,24]}} : {name}[50,24]@hip:0\ngraph_output(%2)\n")
        (grad,) = host.compile(text, "hip", opt).run([ins[2], ins[1]])
        assert grad.shape == (50, 24) and not grad.any()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tensors_that_start_inside_a_block(dtype):
    say(f"tensors one element into their blocks dtype={dtype}")
    size = {F32: 4, graphs.I32: 4, F16: 2, BF16: 2}

    def run(graph, ins):
        exe, stream = host.compile(graph, "hip", 1), host.Stream("hip")
        t_in = [host.Tensor.from_numpy("hip", d, a, byte_offset=size[d]) for a, (d, _) in zip(ins, exe.input_specs())]
        t_out = [host.Tensor("hip", d, shape, byte_offset=size[d]) for d, shape in exe.output_specs()]
        exe.run_tensors(t_in, t_out, stream)
        stream.synchronize()
        return [t.numpy() for t in t_out], exe.run(ins)

    for graph, ins in ((lg.backward(lg.loss_graph(dtype, 60, 300, 72, device="hip"), [0, 1]), lg.loss_inputs(dtype, 60, 300, 72)),
                       (lg.embedding_graph(dtype, 60, 300, 72, 2.0, "hip"), lg.embedding_inputs(dtype, 60, 300, 72)[:2])):
        got, want = run(graph, ins)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("wrt", [[0], [1]])
@pytest.mark.parametrize("opt", [0, 1])
def test_one_gradient_of_the_loss(wrt, opt):
    say(f"gradient of input {wrt[0]} alone opt={opt}")
    ins = lg.loss_inputs(BF16, 220, 1000, 64)
    g = lg.loss_graph(BF16, 220, 1000, 64, device="hip")
    both = host.compile(lg.backward(g, [0, 1]), "hip", opt).run(ins)
    one = host.compile(lg.backward(g, wrt), "hip", opt).run(ins)
    assert np.array_equal(one[0], both[0]) and np.array_equal(one[1], both[1 + wrt[0]])


def test_two_losses_on_one_table():
    """Their gradients of the table are added by the graph; each loss hands its own log-sum-exps on."""
    say("two losses on one table")
    tokens, vocab, dim = (90, 130), 400, 64
    a, b = (lg.loss_inputs(BF16, n, vocab, dim, seed=s) for n, s in zip(tokens, (1, 7)))
    g = graphs.Graph("hip")
    w = g.input(BF16, (vocab, dim))
    x = [g.input(BF16, (n, dim)) for n in tokens]
    t = [g.input(graphs.I32, (n,)) for n in tokens]
    g.output(g.add(g.vocab_loss(x[0], w, t[0]), g.vocab_loss(x[1], w, t[1], mean=False)))
    _, dw, dx0, dx1 = host.compile(lg.backward(g, [0, 1, 2]), "hip", 1).run([a[1], a[0], b[0], a[2], b[2]])
    want = [ref.Loss(ref.values(i[0], BF16), ref.values(a[1], BF16), i[2].astype(np.int64), mean, BF16) for i, mean in ((a, True), (b, False))]
    (x0, x0_tol), (w0, w0_tol) = want[0].gradients(1.0)
    (x1, x1_tol), (w1, w1_tol) = want[1].gradients(1.0)
    ref.check(ref.values(dx0, BF16), x0, x0_tol, "dx of the first")
    ref.check(ref.values(dx1, BF16), x1, x1_tol, "dx of the second")
    ref.check(ref.values(dw, BF16), w0 + w1, ref.rounded(w0 + w1, w0_tol + w1_tol, BF16), "dw")


@pytest.mark.parametrize("tokens", [70, 600])
def test_infinite_logits(hip, tokens):
    """A logit of +infinity makes its row NaN; a row of -infinity alone has no probabilities."""
    say(f"infinite logits, {tokens} rows")
    p = Loss(hip, BF16, tokens, 300, 64)
    p.x[:, 0], p.w[:, 0] = 0, 0x3f80  # 1.0
    _, row0, lse0 = p.forward()
    up, others = 5, np.arange(tokens) != 5
    p.x[up, 0] = 0x7f80  # +infinity
    loss, row, lse = p.forward()
    assert np.isnan(row[up]) and np.isnan(lse[up]) and np.isnan(loss)
    assert np.array_equal(row[others], row0[others]) and np.array_equal(lse[others], lse0[others])
    dx, _ = p.backward(lse)
    dx = ref.values(dx, BF16)
    assert np.isnan(dx[up]).all() and np.isfinite(dx[others]).all()
    p.x[up, 0] = 0xff80  # every logit of the row -infinity
    _, row, lse = p.forward()
    assert np.isnan(row[up]) and lse[up] == -np.inf
    assert np.array_equal(row[others], row0[others]) and np.array_equal(lse[others], lse0[others])
