"""Attention where its numbers reach far: scores that rise and fall from block to block, against float64 (tests/attention_ref.py, which
derives the bounds)."""
import numpy as np
import pytest

from frame_hip import synth
from test_gpu_packed_attention import BF16, E4M3, F16, Paged, say

pytestmark = pytest.mark.gpu


def levels(shape, n):
    """How high the scores of position 0 .. n - 1 lie: steps of 24 (e^24 > 2^34) from one block of 32 to the next."""
    block = np.arange(n) // 32
    return 24.0 * {"rising": block, "falling": block[::-1], "zigzag": block * 7 % 5}[shape]


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (BF16, E4M3), (F16, F16), (F16, E4M3)])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("shape", ["rising", "falling", "zigzag"])
def test_paged_scores_that_move_between_blocks(hip, dtype, cache_dtype, dh, shape):
    # every block of keys that every row sees moves the running maximum, or leaves it far above: decoding steps and chunks, whole and in parts
    say(f"paged {shape} scores, dtype {dtype}, cache {cache_dtype}, dh {dh}")
    for new in ([1, 1, 2], [40, 70, 1]):
        p = Paged(hip, dtype, cache_dtype, [640, 64, 300], new, 8, 2, dh, 16)
        scale = 1 / np.sqrt(dh)
        for b, n in enumerate(p.cached):
            rows = [synth.to_float(synth.tensor(300 + 2 * b + i, (int(n), p.kv_heads * dh), dtype, "normal", 0.25), dtype) for i in range(2)]
            rows[0][:, ::dh] = (levels(shape, int(n)) / (4.0 * scale))[:, None]  # q holds 4 there
            for rows, c, s in ((rows[0], p.kc, p.ks), (rows[1], p.vc, p.vs)):
                p.put(c, s, b, 0, synth.to_storage(rows.astype(np.float32), dtype))
        q = synth.to_float(p.q, dtype).copy()
        q[:, ::dh] = 4.0
        p.q = synth.to_storage(q.astype(np.float32), dtype)
        p.upload()
        for keys in (64, None, 1 << 20):
            p.check_attend(p.attend(max_keys=keys)[0], f"{shape}, cut for {keys}")
