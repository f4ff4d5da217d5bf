"""Paged batches: the operators of a server that keeps many requests in one 8-bit KV cache
(include/jv.h, the section of that name). Arguments are device pointers (ints), e.g. torch tensors'
data_ptr(); `stream` is a cudaStream_t or 0. The structs are plain values that a program builds once
and passes to every call; they own nothing."""
from __future__ import annotations

import ctypes as C
from typing import Optional

from ._lib import JvHeads, JvKv8Cache, JvPagedBatch, JvRopeSpec, check, lib

PAGE_TOKENS, SCALE_TOKENS, HEAD_DIM = 64, 16, 128
DTYPES = {"f32": 0, "f16": 1, "bf16": 30}
LAYOUTS = {"interleaved": 0, "half": 1}
_OPERANDS = [JvHeads * n for n in range(3)]
SCALINGS = {"none": 0, "linear": 1, "yarn": 2}


def batch(requests: int, max_new: int, max_tokens: int, max_blocks: int, max_keys: int, group: int, pages: int,
          block_table: int, lengths: int, starts: int, request_of: int, positions: int, slots: int, work: int,
          status: int) -> JvPagedBatch:
    """jv_paged_batch: the bounds of a step and the device arrays its plan writes."""
    return JvPagedBatch(requests, max_new, max_tokens, max_blocks, max_keys, group, pages, block_table, lengths, starts,
                        request_of, positions, slots, work, status)


def work_bytes(requests: int, max_new: int, max_tokens: int, max_blocks: int, max_keys: int, group: int) -> int:
    """Bytes of a batch's `work` array."""
    b = JvPagedBatch(requests, max_new, max_tokens, max_blocks, max_keys, group, 1)
    n = int(lib.jv_paged_work_bytes(C.byref(b)))
    if n < 0:
        check(1)
    return n


def plan(b: JvPagedBatch, cached: int, new_tokens: int, free_pages: int, n_free: int, n_free_out: int, stream: int = 0) -> None:
    """Block tables, slots, positions and row starts of a step, from the requests' lengths (jv_paged_plan)."""
    check(lib.jv_paged_plan(C.byref(b), cached, new_tokens, free_pages, n_free, n_free_out, stream))


def rope_spec(layout: str, rotary_dim: int, base: float, scaling: str = "none", factor: float = 1.0,
              original_context: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 1.0,
              temperature_scale: float = 0.0, temperature_context: int = 0) -> JvRopeSpec:
    """Rotary frequencies in 64 bits (jv_rope_init). layout: "interleaved" or "half"; scaling: "none",
    "linear" or "yarn"; temperature_*: the query temperature of far positions, off when either is 0."""
    s = JvRopeSpec()
    check(lib.jv_rope_init(C.byref(s), LAYOUTS[layout], rotary_dim, base, SCALINGS[scaling], factor, original_context,
                           beta_fast, beta_slow, attn_factor))
    s.temperature_scale, s.temperature_ctx = temperature_scale, temperature_context
    return s


def heads(ptr: int, n_heads: int, token_stride: int, head_stride: int, out: int = 0, out_token_stride: Optional[int] = None,
          out_head_stride: Optional[int] = None, temperature: bool = False) -> JvHeads:
    """A [tokens][heads][dim] operand and where its result goes (strides in elements, the output's default
    to the input's)."""
    return JvHeads(ptr, out, token_stride, head_stride, token_stride if out_token_stride is None else out_token_stride,
                   head_stride if out_head_stride is None else out_head_stride, n_heads, int(temperature))


def rope(spec: JvRopeSpec, dtype: str, positions: int, tokens: int, head_dim: int, *operands: JvHeads, stream: int = 0) -> None:
    """Rotates one or two operands (queries and keys) at positions[tokens] (jv_rope)."""
    n = len(operands)
    check(lib.jv_rope(C.byref(spec), DTYPES[dtype], positions, tokens, head_dim, _OPERANDS[n](*operands) if n <= 2 else None, n, stream))


def cache(data: int, scales: int, pages: int, kv_heads: int, page_bytes: Optional[int] = None,
          scale_stride: Optional[int] = None) -> JvKv8Cache:
    """One layer of an 8-bit cache: int8 [pages][kv_heads][2][64][128] and fp32 [pages][kv_heads][2][4]."""
    return JvKv8Cache(data, scales, kv_heads * 2 * PAGE_TOKENS * HEAD_DIM if page_bytes is None else page_bytes,
                      kv_heads * 8 if scale_stride is None else scale_stride, pages, kv_heads)


def kv8_append(c: JvKv8Cache, b: JvPagedBatch, dtype: str, k: JvHeads, v: JvHeads, rope: Optional[JvRopeSpec] = None,
               q: Optional[JvHeads] = None, out_dtype: str = "f16", stream: int = 0) -> None:
    """The batch's new keys and values into the cache in 8 bits, rotated on the way with `rope`, which
    also rotates q into its output (jv_kv8_append)."""
    check(lib.jv_kv8_append(C.byref(c), C.byref(b), DTYPES[dtype], C.byref(k), C.byref(v),
                            C.byref(rope) if rope is not None else None, C.byref(q) if q is not None else None,
                            DTYPES[out_dtype], stream))


def kv8_read(c: JvKv8Cache, slots: int, n: int, dtype: str, k_out: int, v_out: int, row_stride: int, status: int = 0,
             stream: int = 0) -> None:
    """The values at n cache slots (jv_kv8_read)."""
    check(lib.jv_kv8_read(C.byref(c), slots, n, DTYPES[dtype], k_out, v_out, row_stride, status, stream))


def attention_bytes(b: JvPagedBatch, kv_heads: int) -> int:
    """Bytes of kv8_attention's workspace."""
    n = int(lib.jv_kv8_attention_bytes(C.byref(b), kv_heads))
    if n < 0:
        check(1)
    return n


def kv8_attention(c: JvKv8Cache, b: JvPagedBatch, dtype: str, q: JvHeads, scale: float, window: int, workspace: int,
                  workspace_bytes: int, stream: int = 0) -> None:
    """Attention of the batch's new tokens over the cache, causal or in a sliding window (jv_kv8_attention)."""
    check(lib.jv_kv8_attention(C.byref(c), C.byref(b), DTYPES[dtype], C.byref(q), scale, window, workspace, workspace_bytes,
                               stream))
