"""Refusals of the paged-batch operators at the ends of their ranges, without a GPU."""
from __future__ import annotations

import ctypes as C

from test_paged import _batch, _cache, _heads


def test_a_batch_whose_work_lists_would_pass_32_bits_is_refused():
    """4096 requests of 2^30 keys each may have 2^32 chunks; the lists are indexed in 32 bits."""
    from jevstral_b200._lib import JV_ERR_ARG, lib

    blocks = 1 << 24
    b = _batch(requests=4096, max_new=32, max_tokens=4096, max_blocks=blocks, max_keys=4096 * blocks * 64, group=1)
    assert lib.jv_paged_work_bytes(C.byref(b)) == -1 and lib.jv_kv8_attention_bytes(C.byref(b), 1) == -1
    assert lib.jv_paged_plan(C.byref(b), 64, 64, 64, 64, 64, None) == JV_ERR_ARG
    b.max_keys = 4096 * 262144  # the same requests of 262,144 keys
    assert lib.jv_paged_work_bytes(C.byref(b)) > 0


def test_attention_refuses_too_many_items_before_it_queues_any():
    """2^24 pairs of query tiles and 1024 KV heads pass a grid's 2^31 blocks: refused by the host, ahead of the first
    launch (a call that got that far would fail for want of a device here)."""
    from jevstral_b200._lib import JV_ERR_RANGE, lib

    b = _batch(requests=1, max_new=1 << 28, max_tokens=1 << 28, max_blocks=1 << 22, max_keys=1 << 28, group=16)
    c = _cache(kv_heads=1024, page_bytes=1024 * 16384, scale_stride=1024 * 8)
    q = _heads(16384)
    assert lib.jv_kv8_attention(C.byref(c), C.byref(b), 1, C.byref(q), 0.1, 0, 64, 1 << 62, None) == JV_ERR_RANGE


def test_append_refuses_the_query_temperature_on_keys_and_values():
    """The flag is the queries': keys or values that ask for it would not get it."""
    from jevstral_b200._lib import JV_ERR_ARG, JvRopeSpec, lib

    spec = JvRopeSpec()
    assert lib.jv_rope_init(C.byref(spec), 0, 64, 1e4, 0, 1, 0, 32, 1, 1) == 0
    b, c, plain, hot = _batch(), _cache(), _heads(2), _heads(2, temperature=1)
    for k, v in ((hot, plain), (plain, hot)):
        assert lib.jv_kv8_append(C.byref(c), C.byref(b), 1, C.byref(k), C.byref(v), C.byref(spec), None, 1, None) == JV_ERR_ARG
