"""packed_attention through the compiled-graph path on the MI355X: forward and training graphs against float64, node by node through
Backend::launch, and the decoder block against the oracle's cpu backend."""
import numpy as np
import pytest

import oracle_lib as orc
import packed_graphs as pg
from frame_hip import graphs, host, synth
from tolerance import assert_close, assert_deep_lowp

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 2, 3


def say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.fixture(scope="module", autouse=True)
def dev():
    assert host.device_count("hip") >= 1, "no hip device"
    orc.load_cpu_backend()


CASES = [(BF16, [0, 70, 70, 213], 220, 4, 2, 64, True), (F16, [3, 130, 131], 131, 6, 3, 40, False), (BF16, [0, 1], 1, 3, 1, 128, True),
         (BF16, [0, 513], 513, 16, 2, 64, True)]


@pytest.mark.parametrize("opt", [0, 1])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_graphs_match_float64(case, opt):
    dtype, cu, tokens, heads, kv_heads, dh, causal = case
    say(f"packed graph {case} opt={opt}")
    args = (dtype, tokens, len(cu) - 1, heads, kv_heads, dh, causal, "hip")
    ins = pg.inputs(dtype, cu, tokens, heads, kv_heads, dh)
    (out,) = host.compile(pg.attention_graph(*args), "hip", opt).run(ins[:4])
    back = host.backward(pg.attention_graph(*args, loss=True).text(), 0, [0, 1, 2])
    exe = host.compile(back, "hip", opt)
    grads = exe.run(ins)[1:]
    pg.check([out, *grads], ins, dtype, heads, kv_heads, dh, causal)
    assert all(np.array_equal(a, b) for a, b in zip(grads, exe.run(ins)[1:]))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_nodes_launched_by_themselves(case):
    dtype, cu, tokens, heads, kv_heads, dh, causal = case
    say(f"packed eager {case}")
    ins = pg.inputs(dtype, cu, tokens, heads, kv_heads, dh)
    q, k, v, c, dout = (host.Tensor.from_numpy("hip", d, a) for d, a in zip((dtype, dtype, dtype, 6, dtype), ins))
    attrs = {"heads": heads, "kv_heads": kv_heads, "causal": causal, "scale": 1.0 / np.sqrt(dh)}
    y = host.Tensor("hip", dtype, ins[0].shape)
    g = graphs.Graph("hip")
    vals = [g.input(graphs.I32 if i == 3 else dtype, a.shape) for i, a in enumerate(ins[:4])]
    g.output(g.op("packed_attention", vals, ins[0].shape, attrs))
    host.launch(g.text(), "hip", [q, k, v, c], [y])
    grads = [host.Tensor("hip", dtype, a.shape) for a in ins[:3]] + [host.Tensor("hip", dtype, (tokens, 4 * heads))]
    t = [f"{graphs.DTYPE_NAME[dtype]}[{s[0]},{s[1]}]@hip:0" for s in (x.shape for x in grads)]
    text = "".join(f"%{i} = graph_input() : {graphs.DTYPE_NAME[6 if i == 3 else dtype]}[{','.join(map(str, s))}]@hip:0\n"
                   for i, s in enumerate([a.shape for a in ins[:4]] + [ins[0].shape] * 2))
    show = ", ".join(f"{n}={graphs._fmt_attr(attrs[n])}" for n in sorted(attrs))
    text += f"%6, %7, %8, %9 = packed_attention_grad_internal(%0, %1, %2, %3, %4, %5) {{{show}}} : {', '.join(t)}\ngraph_output(%6)\n"
    host.launch(text, "hip", [q, k, v, c, y, dout], grads)
    pg.check([y.numpy(), *(x.numpy() for x in grads[:3])], ins, dtype, heads, kv_heads, dh, causal)


def test_float32_is_refused():
    say("packed graph f32")
    g = pg.attention_graph(F32, 8, 1, 2, 1, 8, device="hip")
    ins = pg.inputs(F32, [0, 8], 8, 2, 1, 8)
    with pytest.raises(host.FrameError, match="bf16 or f16"):
        host.compile(g, "hip", 1).run(ins[:4])


def test_decoder_block_forward(dev):
    say("decoder block bf16")
    tokens, d, cu = 300, 256, [0, 100, 100, 101, 290]
    args = dict(d_model=d, heads=4, kv_heads=2, ffn=512)
    g, shapes = graphs.decoder_block(tokens, 4, dtype=BF16, device="hip", **args)
    ins = pg.decoder_inputs(shapes, cu, tokens, d, BF16)
    (got,) = host.compile(g, "hip", 1).run(ins)
    (want,) = orc.run_graph_cpu(g.text().replace("@hip:0", "@cpu:0"), ins)
    assert_close(got, want, BF16, what="decoder block")


def test_decoder_block_training_step(dev):
    """The whole training graph (several roundings deep) against the oracle's own bf16 result, both measured from float32."""
    say("decoder block bf16 training step")
    tokens, d, cu = 200, 128, [0, 60, 61, 61, 195]
    args = dict(d_model=d, heads=2, kv_heads=1, ffn=256, train=True)
    g, shapes = graphs.decoder_block(tokens, 4, dtype=BF16, device="hip", **args)
    wrt = list(range(2, 2 + len(shapes)))
    ins = pg.decoder_inputs(shapes, cu, tokens, d, BF16, train=True)
    back = host.backward(g.text(), 0, wrt)
    got = host.compile(back, "hip", 1).run(ins)
    want = orc.run_graph_cpu(back.replace("@hip:0", "@cpu:0"), ins)
    g32, _ = graphs.decoder_block(tokens, 4, dtype=F32, device="cpu", **args)
    exact = orc.run_graph_cpu(host.backward(g32.text(), 0, wrt),
                              [a if a.dtype == np.int32 else synth.to_float(a, BF16).reshape(a.shape) for a in ins])
    for i in range(len(shapes)):
        # mean_slack: the attention's gradients round p and ds, which the oracle's double evaluation does not: 3 roundings' variance to 1
        assert_deep_lowp(got[1 + i], want[1 + i], exact[1 + i], BF16, mean_slack=1.75, max_slack=3.0, what=f"gradient {i}")
