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
