"""packed_attention whose cu_seqlens other nodes of the graph compute, forward and training, on the MI355X."""
import numpy as np
import pytest

import oracle_lib as orc
import packed_graphs as pg
from frame_hip import graphs, host

pytestmark = pytest.mark.gpu
BF16 = 3


@pytest.mark.parametrize("opt", [0, 1])
def test_cu_seqlens_cut_from_a_longer_tensor(opt):
    print(f"[case] computed cu_seqlens, opt={opt}", flush=True)
    orc.load_cpu_backend()
    tokens, cu = 213, np.array([-3, 0, 70, 70, 200, 7], np.int32)
    ins = pg.inputs(BF16, cu[1:5], tokens, 4, 2, 64)
    plain = pg.attention_graph(BF16, tokens, 3, 4, 2, 64, device="hip", loss=True)
    want = host.compile(host.backward(plain.text(), 0, [0, 1, 2]), "hip", opt).run(ins)
    g = graphs.Graph("hip")
    q, k, v = (g.input(BF16, (tokens, h * 64)) for h in (4, 2, 2))
    lens = g.slice(g.input(graphs.I32, (6,)), 0, 1, 5)
    out = g.packed_attention(q, k, v, lens, 4, 2)
    g.output(g.op("sum", [g.mul(out, g.input(BF16, out.shape))], (), {"axes": []}))
    got = host.compile(host.backward(g.text(), 0, [0, 1, 2]), "hip", opt).run([*ins[:3], cu, ins[4]])
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
