"""Backend::compile of embedding and vocab_loss nodes that no pass has verified: wrong ranks, attributes and counts of inputs are named, when the
graph is compiled or when it runs, and end nothing."""
import numpy as np
import pytest

from frame_hip import graphs, host

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 3


def graph(node, *inputs):
    """One node of these inputs (dtype, shape); its first output is the graph's."""
    text = "".join(f"%{i} = graph_input() : {graphs.DTYPE_NAME[t]}[{','.join(map(str, s))}]@hip:0\n" for i, (t, s) in enumerate(inputs))
    return f"{text}%{node}\ngraph_output(%{node.split(' ')[0].rstrip(',')})\n"


X, W, T, ONE = (BF16, (6, 8)), (BF16, (9, 8)), (graphs.I32, (6,)), (BF16, ())
LOSS, GX, GW = "bfloat16[]@hip:0", "bfloat16[6,8]@hip:0", "bfloat16[9,8]@hip:0"
GRAD = "vocab_loss_grad_internal(%0, %1, %2, %3, %4)"
CASES = {
    "loss without mean": (graph(f"3 = vocab_loss(%0, %1, %2) : {LOSS}", X, W, T), [X, W, T]),
    "loss of x of one dimension": (graph(f"3 = vocab_loss(%0, %1, %2) {{mean=true}} : {LOSS}", (BF16, (6,)), W, T), [(BF16, (6,)), W, T]),
    "loss of w without dimensions": (graph(f"3 = vocab_loss(%0, %1, %2) {{mean=true}} : {LOSS}", X, ONE, T), [X, ONE, T]),
    "loss of two inputs": (graph(f"2 = vocab_loss(%0, %1) {{mean=true}} : {LOSS}", X, W), [X, W]),
    "gradient without mean": (graph(f"5, %6 = {GRAD} : {GX}, {GW}", X, W, T, ONE, ONE), [X, W, T, ONE, ONE]),
    "gradient of x of one dimension": (graph(f"5, %6 = {GRAD} {{mean=true}} : {GX}, {GW}", (BF16, (6,)), W, T, ONE, ONE),
                                       [(BF16, (6,)), W, T, ONE, ONE]),
    "gradient of one output": (graph(f"5 = {GRAD} {{mean=true}} : {GX}", X, W, T, ONE, ONE), [X, W, T, ONE, ONE]),
    "gradient of a table of one dimension": (graph("2 = embedding_grad_internal(%0, %1) {scale=1.0, table_shape=shape[9,8]} : bfloat16[9]@hip:0", X, T),
                                             [X, T]),
    "gradient of gy without dimensions": (graph(f"2 = embedding_grad_internal(%0, %1) {{scale=1.0, table_shape=shape[9,8]}} : {GW}", ONE, T), [ONE, T]),
    "gradient without scale": (graph(f"2 = embedding_grad_internal(%0, %1) {{table_shape=shape[9,8]}} : {GW}", X, T), [X, T]),
}


@pytest.mark.parametrize("opt", [0, 1])
@pytest.mark.parametrize("name", list(CASES))
def test_nodes_that_no_schema_takes_are_named(name, opt):
    print(f"[case] {name} opt={opt}", flush=True)
    text, inputs = CASES[name]
    with pytest.raises(host.FrameError, match="vocab_loss|embedding"):
        host.backend_compile(text, "hip", opt).run([np.zeros(s, np.int32 if t == graphs.I32 else np.uint16) for t, s in inputs])


def test_a_gradient_whose_forward_is_no_loss():
    """y comes from a vocab_loss of two inputs: it cannot hand over log-sum-exps."""
    print("[case] gradient behind a loss of two inputs", flush=True)
    text = ("%0 = graph_input() : bfloat16[6,8]@hip:0\n%1 = graph_input() : bfloat16[9,8]@hip:0\n%2 = graph_input() : int32[6]@hip:0\n"
            "%3 = graph_input() : bfloat16[]@hip:0\n%4 = vocab_loss(%0, %1) {mean=true} : bfloat16[]@hip:0\n"
            "%5, %6 = vocab_loss_grad_internal(%0, %1, %2, %4, %3) {mean=true} : bfloat16[6,8]@hip:0, bfloat16[9,8]@hip:0\ngraph_output(%5)\n")
    with pytest.raises(host.FrameError, match="vocab_loss"):
        host.backend_compile(text, "hip", 1).run([np.zeros(s, np.int32 if t == graphs.I32 else np.uint16) for t, s in (X, W, T, ONE)])
