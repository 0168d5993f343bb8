"""embedding and vocab_loss through the compiled-graph path on the MI355X: forward and training graphs against float64, node by node
through Backend::launch, and a language model's training step against the oracle's cpu backend."""
import numpy as np
import pytest

import language_graphs as lg
import language_ref as ref
import oracle_lib as orc
from frame_hip import graphs, host, synth
from test_cpu_language_graph import GRADIENT_ALONE
from tolerance import assert_deep_lowp

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 2, 3


def say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.fixture(scope="module", autouse=True)
def dev():
    assert host.device_count("hip") >= 1, "no hip device"
    orc.load_cpu_backend()


LOSSES = [(BF16, 220, 1000, 64, True), (F16, 131, 513, 40, False), (BF16, 1, 5003, 128, True), (BF16, 700, 300, 256, True)]


@pytest.mark.parametrize("opt", [0, 1])
@pytest.mark.parametrize("case", LOSSES, ids=str)
def test_loss_graphs_match_float64(case, opt):
    dtype, tokens, vocab, dim, mean = case
    say(f"vocab_loss graph {case} opt={opt}")
    ins = lg.loss_inputs(dtype, tokens, vocab, dim, outside=0.0 if tokens == 1 else 0.2)
    g = lg.loss_graph(dtype, tokens, vocab, dim, mean, "hip")
    (loss,) = host.compile(g, "hip", opt).run(ins)
    exe = host.compile(lg.backward(g, [0, 1]), "hip", opt)
    outs = exe.run(ins)
    assert np.array_equal(outs[0], loss)
    lg.check_loss(outs, ins, dtype, mean)
    assert all(np.array_equal(a, b) for a, b in zip(outs, exe.run(ins)))


@pytest.mark.parametrize("opt", [0, 1])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_embedding_graphs_match_float64(dtype, opt):
    say(f"embedding graph dtype={dtype} opt={opt}")
    ins = lg.embedding_inputs(dtype, 333, 50, 72)
    (out,) = host.compile(lg.embedding_graph(dtype, 333, 50, 72, 8.0, "hip"), "hip", opt).run(ins[:2])
    (grad,) = host.compile(lg.backward(lg.embedding_graph(dtype, 333, 50, 72, 8.0, "hip", loss=True), [0]), "hip", opt).run(ins)[1:]
    lg.check_embedding([out, grad], ins, dtype, 8.0)


def eager(op, attrs, ins, types, shapes):
    """One node by itself; its outputs' arrays."""
    tensors = [host.Tensor.from_numpy("hip", t, a) for t, a in zip(types, ins)]
    outs = [host.Tensor("hip", types[0], s) for s in shapes]
    name = graphs.DTYPE_NAME
    text = "".join(f"%{i} = graph_input() : {name[t]}[{','.join(map(str, a.shape))}]@hip:0\n" for i, (t, a) in enumerate(zip(types, ins)))
    n = len(ins)
    text += (", ".join(f"%{n + i}" for i in range(len(shapes))) + f" = {op}({', '.join(f'%{i}' for i in range(n))}) {{{attrs}}} : "
             + ", ".join(f"{name[types[0]]}[{','.join(map(str, s))}]@hip:0" for s in shapes) + f"\ngraph_output(%{n})\n")
    host.launch(text, "hip", tensors, outs)
    return [o.numpy() for o in outs]


@pytest.mark.parametrize("case", LOSSES, ids=str)
def test_loss_nodes_launched_by_themselves(case):
    dtype, tokens, vocab, dim, mean = case
    say(f"vocab_loss eager {case}")
    ins = lg.loss_inputs(dtype, tokens, vocab, dim, outside=0.0 if tokens == 1 else 0.2)
    attrs, types = f"mean={'true' if mean else 'false'}", [dtype, dtype, graphs.I32]
    (loss,) = eager("vocab_loss", attrs, ins, types, [()])
    one = synth.to_storage(np.ones((), np.float32), dtype).reshape(())
    grads = eager("vocab_loss_grad_internal", attrs, ins + [loss, one], types + [dtype, dtype], [ins[0].shape, ins[1].shape])
    lg.check_loss([loss, *grads], ins, dtype, mean)


def test_a_compiled_gradient_without_its_forward():
    say("vocab_loss gradient compiled by itself")
    ins = lg.loss_inputs(BF16, 40, 90, 64)
    zero, one = (synth.to_storage(np.full((), v, np.float32), BF16).reshape(()) for v in (0.0, 1.0))
    grads = host.compile(GRADIENT_ALONE, "hip", 1).run(ins + [zero, one])
    (loss,) = host.compile(lg.loss_graph(BF16, 40, 90, 64, device="hip"), "hip", 1).run(ins)
    lg.check_loss([loss, *grads], ins, BF16, True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_embedding_nodes_launched_by_themselves(dtype):
    say(f"embedding eager dtype={dtype}")
    ins = lg.embedding_inputs(dtype, 100, 30, 24)
    (out,) = eager("embedding", "scale=0.5", ins[:2], [dtype, graphs.I32], [(100, 24)])
    (grad,) = eager("embedding_grad_internal", "scale=0.5, table_shape=shape[30,24]", [ins[2], ins[1]], [dtype, graphs.I32], [(30, 24)])
    lg.check_embedding([out, grad], ins, dtype, 0.5)


def test_a_float32_loss_is_refused():
    say("vocab_loss graph f32")
    with pytest.raises(host.FrameError, match="bf16 or f16"):
        host.compile(lg.loss_graph(F32, 8, 16, 8, device="hip"), "hip", 1).run(lg.loss_inputs(F32, 8, 16, 8))


@pytest.mark.parametrize("opt", [0, 1])
def test_a_tied_table_gets_both_gradients(opt):
    """d/dtable of vocab_loss(2 table[ids], table, targets): at opt 1 the sum is rounded once, at opt 0 after each."""
    say(f"tied table opt={opt}")
    tokens, vocab, dim = 300, 70, 64
    rng = np.random.default_rng(3)
    table = synth.tensor(1, (vocab, dim), BF16, "normal", 0.2)
    which, targets = lg.ids(rng, tokens, vocab, 0.1), lg.ids(rng, tokens, vocab, 0.3)
    _, got = host.compile(lg.backward(lg.tied_graph(BF16, tokens, vocab, dim, "hip"), [0]), "hip", opt).run([table, which, targets])
    t64 = ref.values(table, BF16)
    x, _ = ref.embed(t64, which.astype(np.int64), 2.0, BF16)
    x = ref.values(synth.to_storage(x.astype(np.float32), BF16), BF16)
    (dx, dx_tol), (dw, dw_tol) = ref.Loss(x, t64, targets.astype(np.int64), True, BF16).gradients(1.0)
    total, tol = ref.embed_grad(dx, which.astype(np.int64), vocab, 2.0, dw, BF16)
    more, _ = ref.embed_grad(dx_tol, which.astype(np.int64), vocab, 2.0, None, BF16)  # dx is rounded on the way
    first, _ = ref.embed_grad(dx, which.astype(np.int64), vocab, 2.0, None, BF16)
    tol = tol + 1.02 * (more + dw_tol) + ref.rounded(total, 0.0, BF16) + (ref.rounded(first, 0.0, BF16) if opt == 0 else 0.0)
    ref.check(ref.values(got, BF16), total, tol, "dtable")


@pytest.mark.parametrize("tied", [True, False])
def test_language_model_training_step(tied):
    """The whole training graph (many roundings deep) against the oracle's own bf16 result, both measured from float32."""
    say(f"language model bf16 training step tied={tied}")
    tokens, vocab, d, cu = 200, 300, 128, [0, 60, 61, 61, 195]
    args = dict(d_model=d, heads=2, kv_heads=1, ffn=256, layers=2, tied=tied)
    g, shapes = graphs.language_model(tokens, 4, vocab, device="hip", **args)
    wrt = list(range(3, 3 + len(shapes)))
    ins = lg.model_inputs(shapes, cu, tokens, vocab, BF16)
    back = lg.backward(g, wrt)
    exe = host.compile(back, "hip", 1)
    got = exe.run(ins)
    assert all(np.array_equal(a, b) for a, b in zip(got, exe.run(ins)))
    want = orc.run_graph_cpu(back.replace("@hip:0", "@cpu:0"), ins)
    g32, _ = graphs.language_model(tokens, 4, vocab, dtype=F32, device="cpu", **args)
    exact = orc.run_graph_cpu(lg.backward(g32, wrt), [a if a.dtype == np.int32 else synth.to_float(a, BF16).reshape(a.shape) for a in ins])
    assert abs(float(synth.to_float(got[0], BF16).reshape(())) - float(exact[0].reshape(()))) <= 0.02 * float(exact[0].reshape(()))
    for i in range(len(shapes)):
        # mean_slack: the loss' and the attention's gradients round their operands, which the oracle's double evaluation does not
        assert_deep_lowp(got[1 + i], want[1 + i], exact[1 + i], BF16, mean_slack=1.75, max_slack=3.0, what=f"gradient {i} {shapes[i]}")


def test_language_model_step_replayed(monkeypatch):
    """The training step captured on its second run and replayed: other tokens, targets and parameters in the same tensors, eager work of the
    same ops and host synchronisation between the replays; every run equals a fresh eager one bit for bit."""
    say("language model step captured and replayed")
    monkeypatch.setenv("FRAME_HIP_GRAPHS", "1")  # replay is opt-in; restored however the test ends
    tokens, vocab, d, cu = 96, 130, 64, [0, 40, 96]
    g, shapes = graphs.language_model(tokens, 2, vocab, d_model=d, heads=1, kv_heads=1, ffn=128, device="hip")
    text = lg.backward(g, list(range(3, 3 + len(shapes))))
    exe, stream = host.compile(text, "hip", 1), host.Stream("hip")
    ins, outs = exe.upload_inputs(lg.model_inputs(shapes, cu, tokens, vocab, BF16)), exe.alloc_outputs()
    small = lg.loss_inputs(BF16, 50, 70, 64)
    for run in range(6):
        values = lg.model_inputs(shapes, cu, tokens, vocab, BF16, seed=901 + 50 * run)
        for t, a in zip(ins, values):
            host.check(host.lib().frame_tensor_upload(t.handle, np.ascontiguousarray(a).ctypes.data, a.nbytes))
        exe.run_tensors(ins, outs, stream)  # eager, capture and launch, then replays
        eager("vocab_loss", "mean=true", small, [BF16, BF16, graphs.I32], [()])
        stream.synchronize()
        want = host.compile(text, "hip", 1).run(values)  # a fresh executable: eager
        for i, (a, b) in enumerate(zip(outs, want)):
            assert np.array_equal(a.numpy(), b), f"run {run}, output {i}"
