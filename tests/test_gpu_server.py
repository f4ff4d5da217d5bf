"""jv_server: many requests of one model over the 8-bit cache, against a context's fp16 cache and against
itself. An 8-bit key or value differs from its own by a rounding of rms 1 / (127 sqrt 12) of its block's
largest, about 1 % of a typical element (the largest of 2048 is some 4 sigma); it reaches the output through
the values and, at scores of a few units, the weights: within 3 % of the logits' norm over two layers."""
from __future__ import annotations

import numpy as np
import pytest

import jevstral_b200 as jv
from small_model import SMALL_CFG, WIDE_CFG

pytestmark = pytest.mark.gpu

ROWS = list(range(1000, 1256))


def toks(n, seed):
    return np.random.default_rng(seed).integers(1000, 16384, n).tolist()


def rel_l2(a, b):
    return float(np.linalg.norm(np.asarray(a, np.float64) - b) / np.linalg.norm(b))


@pytest.mark.parametrize("qtype,wide", [("Q8_0", False), ("Q4_0", False), ("Q4_K", False), ("Q8_0", True)])
def test_requests_follow_a_context_s_logits(model_factory, qtype, wide):
    path = model_factory(WIDE_CFG if wide else SMALL_CFG, qtype)
    with jv.Model(path, kv_pool_mb=128) as m, jv.Server(m, 3, 900, 1200) as s:
        assert s.bytes_per_position * 2 <= 1.02 * m.config.layers * m.config.kv_heads * 128 * 2 * 2
        prompts = [toks(n, n) for n in (700, 33, 1)]
        steps = [toks(5, 100 + r) for r in range(3)]
        got = [s.forward(dict(enumerate(prompts)), ROWS)] + [s.forward({r: [steps[r][i]] for r in range(3)}, ROWS) for i in range(5)]
        for r in range(3):
            with jv.MinistralModel(m) as c:
                want = [c.forward_selected(prompts[r], ROWS)] + [c.forward_selected([t], ROWS) for t in steps[r]]
            for a, b in zip(got, want):
                assert rel_l2(a[r], b) < 0.03, (r, rel_l2(a[r], b))
            assert s.length(r) == len(prompts[r]) + 5


def test_yarn_and_the_query_temperature(model_factory):
    from jevstral_b200.synth import SynthConfig, yarn_metadata

    cfg = SynthConfig(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=128, ff=512, vocab=16384,
                      extra=yarn_metadata(original_context=64))
    with jv.Model(model_factory(cfg, "Q8_0"), kv_pool_mb=64) as m, jv.Server(m, 1, 400, 400) as s, jv.MinistralModel(m) as c:
        assert m.config.yarn_active
        p = toks(300, 3)
        assert rel_l2(s.forward({0: p}, ROWS)[0], c.forward_selected(p, ROWS)) < 0.03
        assert rel_l2(s.forward({0: [5000]}, ROWS)[0], c.forward_selected([5000], ROWS)) < 0.03


def test_a_request_s_bits_do_not_depend_on_the_others(model_factory):
    """Prompts, chunks and single tokens mixed in passes against each request alone; then a released slot
    taken over by another request, on the pages of the first."""
    with jv.Model(model_factory(SMALL_CFG, "Q8_0"), kv_pool_mb=64) as m:
        plan = {0: [toks(200, 1), toks(1, 2), toks(60, 3), toks(1, 4)], 1: [toks(1, 5), toks(1, 6), toks(1, 7), toks(9, 8)],
                2: [toks(90, 9), [], toks(3, 10), toks(1, 11)]}
        with jv.Server(m, 3, 600, 400) as s:
            together = [s.forward({r: plan[r][i] for r in plan}, ROWS) for i in range(4)]
            assert 2 not in together[1]
            s.release(0)
            assert s.length(0) == 0 and s.length(2) == 94
            again = s.forward({0: plan[1][0] + plan[1][1], 1: toks(2, 12)}, ROWS)
        for r in plan:
            with jv.Server(m, 2, 600, 300) as s:
                for i in range(4):
                    if plan[r][i]:
                        assert np.array_equal(s.forward({1: plan[r][i]}, ROWS)[1], together[i][r]), (r, i)
                if r == 1:
                    assert np.array_equal(s.forward({1: toks(2, 12)}, ROWS)[1], again[1])
                    assert np.array_equal(s.forward({0: plan[1][0] + plan[1][1]}, ROWS)[0], again[0])


def test_refusals_leave_every_request_as_it_was(model_factory):
    with jv.Model(model_factory(SMALL_CFG, "Q8_0"), kv_pool_mb=64) as m:
        with pytest.raises(jv.ArgumentError):
            jv.Server(m, 0, 100, 100)
        with pytest.raises(jv.ArgumentError):
            jv.Server(m, 1, 1 << 30, 100)
        with jv.Server(m, 2, 200, 150, pages=4) as s, jv.Server(m, 2, 200, 150) as other:
            first = {0: toks(100, 1), 1: toks(20, 2)}
            assert all(np.array_equal(a, b) for a, b in zip(s.forward(first, ROWS).values(), other.forward(first, ROWS).values()))
            for bad, error in (({0: toks(30, 3), 1: toks(60, 4)}, jv.DeviceOutOfMemoryError),  # 3 + 2 pages of 4
                               ({0: toks(101, 5)}, jv.ArgumentOutOfRangeError), ({1: toks(151, 6)}, jv.ArgumentOutOfRangeError),
                               ({}, jv.ArgumentError), ({0: [16384]}, jv.ArgumentOutOfRangeError)):
                with pytest.raises(error):
                    s.forward(bad, ROWS)
            with pytest.raises(jv.ArgumentOutOfRangeError):
                s.forward({0: [1]}, [1 << 30])
            with pytest.raises(jv.ArgumentOutOfRangeError):
                s.release(2)
            assert (s.length(0), s.length(1), s.length(2)) == (100, 20, -1)
            step = {0: [1234], 1: [4321]}
            assert all(np.array_equal(a, b) for a, b in zip(s.forward(step, ROWS).values(), other.forward(step, ROWS).values()))


def test_a_value_outside_fp16_is_reported(model_factory):
    """Norm gains of 1e5 drive the operands out of range: the pass fails with the context's error, and the
    server is usable after it."""
    from dataclasses import replace

    with jv.Model(model_factory(replace(SMALL_CFG, norm_gain=1e5), "Q8_0"), kv_pool_mb=64) as m, jv.Server(m, 1, 100, 100) as s:
        for _ in range(2):
            with pytest.raises(jv.NumericError):
                s.forward({0: toks(9, 1)}, ROWS)
            assert s.length(0) == 0


def test_a_pass_after_one_that_failed(model_factory, tmp_path):
    """One token's embedding is infinite: its pass fails on the device, and the next one, without it, gives what
    it gives on a server that saw no failure."""
    import gguf

    path = tmp_path / "bad.gguf"
    raw = bytearray(open(model_factory(SMALL_CFG, "Q8_0"), "rb").read())
    t = next(t for t in gguf.GGUFReader(model_factory(SMALL_CFG, "Q8_0")).tensors if t.name == "token_embd.weight")
    row = SMALL_CFG.hidden // 32 * 34
    for b in range(t.data_offset + 2000 * row, t.data_offset + 2001 * row, 34):
        raw[b:b + 2] = b"\x00\x7c"  # the block's fp16 scale
    path.write_bytes(raw)
    with jv.Model(path, kv_pool_mb=64) as m, jv.Server(m, 2, 200, 150) as s, jv.Server(m, 2, 200, 150) as other:
        p = {0: toks(32, 1), 1: toks(16, 2)}
        for x in (s, other):
            x.forward(p, ROWS)
        for bad in ({0: [2000] * 3, 1: [1001]}, {0: [2000]}):
            with pytest.raises(jv.NumericError):
                s.forward(bad, ROWS)
            assert (s.length(0), s.length(1)) == (32, 16)
        for step in ({0: toks(70, 3), 1: [1500]}, {0: [1501], 1: [1502]}):
            a, b = s.forward(step, ROWS), other.forward(step, ROWS)
            assert all(np.array_equal(a[r], b[r]) for r in step)
