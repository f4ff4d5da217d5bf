"""jv_server: what a pass that fails on the device leaves behind."""
from __future__ import annotations

import numpy as np
import pytest

import jevstral_b200 as jv
from small_model import SMALL_CFG
from test_gpu_server import ROWS, toks

pytestmark = pytest.mark.gpu


def _one_bad_token(src, path):
    """A copy of the model in which token 2000 alone has the first 32 channels of its embedding, and only those. The
    first layer takes them into keys and values some 1,000 times the others' and into queries outside fp16: the pass
    fails in the first rotation, with everything it appends finite."""
    import gguf

    raw = bytearray(open(src, "rb").read())
    tensors = {t.name: t for t in gguf.GGUFReader(src).tensors}
    row = SMALL_CFG.hidden // 32 * 34  # bytes of a Q8_0 row: blocks of an fp16 scale and 32 int8

    def scale_first_block(name, rows, factor):
        base = tensors[name].data_offset
        for r in rows:
            at = base + r * row
            d = np.frombuffer(bytes(raw[at:at + 2]), np.float16)[0]
            raw[at:at + 2] = np.float16(float(d) * factor).tobytes()

    scale_first_block("token_embd.weight", [r for r in range(SMALL_CFG.vocab) if r != 2000], 0.0)
    at = tensors["token_embd.weight"].data_offset + 2000 * row
    for b in range(34, row, 34):
        raw[at + b:at + b + 2] = b"\0\0"
    kv = SMALL_CFG.kv_heads * SMALL_CFG.head_dim
    scale_first_block("blk.0.attn_k.weight", range(kv), 1e3)
    scale_first_block("blk.0.attn_v.weight", range(kv), 1e3)
    scale_first_block("blk.0.attn_q.weight", range(SMALL_CFG.heads * SMALL_CFG.head_dim), 4e5)
    path.write_bytes(raw)
    return path


@pytest.mark.parametrize("lengths", [(37, 21), (64, 5), (15, 190)])
def test_a_failed_pass_leaves_the_requests_as_they_were(model_factory, tmp_path, lengths):
    """Requests that end inside a block of 16 positions, a failed pass that continues those blocks with keys and values
    far larger than theirs, and the passes after it: the bits of a server that saw no failure."""
    path = _one_bad_token(model_factory(SMALL_CFG, "Q8_0"), tmp_path / "bad.gguf")
    with jv.Model(path, kv_pool_mb=64) as m, jv.Server(m, 3, 300, 250) as s, jv.Server(m, 3, 300, 250) as other:
        p = {0: toks(lengths[0], 1), 2: toks(lengths[1], 2)}
        for x in (s, other):
            first = x.forward(p, ROWS)
            assert all(np.isfinite(v).all() for v in first.values())
        for bad in ({0: [2000] * 3, 2: [1001]}, {0: [1500], 1: [2000], 2: [2000]}, {0: [1001] * 20 + [2000], 2: [2000] * 40}):
            with pytest.raises(jv.NumericError):
                s.forward(bad, ROWS)
            assert (s.length(0), s.length(1), s.length(2)) == (lengths[0], 0, lengths[1])
        for step in ({0: [1500], 2: [1501]}, {0: toks(20, 3), 1: toks(9, 4)}, {0: [1502], 1: [1503], 2: [1504]}):
            a, b = s.forward(step, ROWS), other.forward(step, ROWS)
            assert all(np.array_equal(a[r], b[r]) for r in step)
