"""Training graphs with integer tensors: graphs of nothing else, inputs that an op gives no gradient to, and what computes those."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import oracle_lib as orc
import packed_graphs as pg
from frame_hip import graphs, host

BF16, I32 = 3, graphs.I32
PACKAGE = os.path.dirname(os.path.dirname(os.path.abspath(host.__file__)))


@pytest.fixture(scope="module", autouse=True)
def cpu_backend():
    orc.load_cpu_backend()


def total(g, x):
    return g.op("sum", [x], (), {"axes": []})


@pytest.mark.parametrize("wrt", [[0], [1], [0, 1]])
def test_a_graph_of_integers_is_differentiated(wrt):
    g = graphs.Graph("cpu")
    a, b = g.input(I32, (3,)), g.input(I32, (3,))
    g.output(total(g, g.mul(a, b)))
    back = host.backward(g.text(), 0, wrt)
    assert host.roundtrip(back) == back
    # d sum(a b) / da = the sum's gradient times b, and the other way round; all of it int32
    lines = back.splitlines()
    assert not any("float" in line for line in lines)
    outs = [line for line in lines if line.startswith("graph_output(")]
    assert len(outs) == 1 + len(wrt)
    for i, out in zip(wrt, outs[1:]):
        (made,) = [line for line in lines if line.startswith(out[len("graph_output("):-1] + " = ")]
        assert " mul(" in made and f"%{1 - i}" in made and made.endswith("int32[3]@cpu:0")


def test_an_integer_input_beside_the_loss_has_zeros():
    g = graphs.Graph("cpu")
    a, _ = g.input(I32, (3,)), g.input(I32, (2,))
    g.output(total(g, g.mul(a, a)))
    back = host.backward(g.text(), 0, [1])
    assert "int32[2]" in back.splitlines()[-3]


def attention(g, tokens, cu):
    q, k, v = (g.input(BF16, (tokens, 16)) for _ in range(3))
    return g.packed_attention(q, k, v, cu, 2, 2)


def test_cu_seqlens_may_be_computed():
    # a slice of a longer tensor: the nodes that make it lie on the way to the loss and have no gradient
    tokens, cu = 9, np.array([-3, 0, 4, 9, 7], np.int32)
    g = graphs.Graph("cpu")
    longer = g.input(I32, (5,))
    y = attention(g, tokens, g.slice(longer, 0, 1, 4))
    g.output(total(g, g.mul(y, g.input(BF16, (tokens, 16)))))
    back = host.backward(g.text(), 0, [1, 2, 3])
    assert back.count(" packed_attention_grad_internal(") == 1 and "slice_grad" not in back
    q, k, v, _, dout = pg.inputs(BF16, cu[1:4], tokens, 2, 2, 8)
    outs = orc.run_graph_cpu(back, [cu, q, k, v, dout])
    plain = host.backward(pg.attention_graph(BF16, tokens, 2, 2, 2, 8, loss=True).text(), 0, [0, 1, 2])
    for a, b in zip(outs, orc.run_graph_cpu(plain, [q, k, v, cu[1:4], dout])):
        assert np.array_equal(a, b)
    with pytest.raises(host.FrameError, match="not of a floating-point type"):
        host.backward(g.text(), 0, [0, 1])


def test_computed_cu_seqlens_through_several_nodes():
    tokens = 9
    g = graphs.Graph("cpu")
    parts = [g.input(I32, (n,)) for n in (2, 3)]
    cu = g.slice(g.concat(parts, 0), 0, 0, 3)
    y = attention(g, tokens, cu)
    g.output(total(g, g.mul(y, y)))
    back = host.backward(g.text(), 0, [2, 3, 4])
    assert back.count(" packed_attention_grad_internal(") == 1


PLUGIN = """
#include <frame/ops/op_registry.h>
#include <frame/ir/graph.h>
using namespace frame;
namespace {
Result<std::vector<Shape>> infer(const ops::NodeContext& c) { return std::vector<Shape>{c.input_types[0].shape}; }
// one gradient per input, the integer one's among them
Result<ir::Graph> gradient(const ops::NodeContext& c) {
  ir::Graph g{"two_gradients"};
  std::vector<ir::Value*> in;
  for (const ir::TensorType& t : {c.input_types[0], c.input_types[1], c.input_types[0], c.input_types[0]}) {
    Result<ir::Value*> v = g.add_graph_input(t);
    if (!v.is_ok()) return v.status();
    in.push_back(v.value());
  }
  if (Status s = g.mark_output(in[3]); !s.is_ok()) return s;
  if (Status s = g.mark_output(in[1]); !s.is_ok()) return s;
  return g;
}
}  // namespace
FRAME_REGISTER_OP("test_scaled_by_integer").input("x", "").input("n", "").output("y", "").shape_infer(&infer).gradient(&gradient);
"""


def test_an_op_may_give_its_integer_input_a_gradient(tmp_path):
    # a registered op whose gradient function has one output per input, as the contract of every op without such inputs says
    source, lib = tmp_path / "op.cpp", tmp_path / "libop.so"
    source.write_text(PLUGIN)
    subprocess.run(["g++", "-std=c++20", "-shared", "-fPIC", "-I", os.path.join(PACKAGE, "include"), str(source), "-o", str(lib),
                    "-L", os.path.join(PACKAGE, "lib"), "-lframe", "-Wl,-rpath," + os.path.join(PACKAGE, "lib")], check=True)
    host.lib()
    ctypes.CDLL(str(lib), mode=ctypes.RTLD_GLOBAL)
    g = graphs.Graph("cpu")
    x, n = g.input(BF16, (4,)), g.input(I32, (4,))
    g.output(total(g, g.op("test_scaled_by_integer", [x, n], (4,))))
    back = host.backward(g.text(), 0, [0, 1])
    assert back.splitlines()[-1] == f"graph_output(%{n.id})"
