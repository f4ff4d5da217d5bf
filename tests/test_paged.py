"""The paged-batch operators without a GPU: struct layouts, rotary frequencies and every refusal that the
host makes before it touches a device."""
from __future__ import annotations

import ctypes as C
import math
import subprocess

import pytest

from conftest import REPO


def _batch(**change):
    from jevstral_b200._lib import JvPagedBatch

    v = dict(requests=4, max_new=8, max_tokens=16, max_blocks=4, max_keys=256, group=4, pages=8, block_table=64, lengths=64,
             starts=64, request_of=64, positions=64, slots=64, work=64, status=64)
    v.update(change)
    return JvPagedBatch(*v.values())


def _cache(**change):
    from jevstral_b200._lib import JvKv8Cache

    v = dict(data=64, scales=64, page_bytes=2 * 16384, scale_stride=16, pages=8, kv_heads=2)
    v.update(change)
    return JvKv8Cache(*v.values())


def _heads(n, **change):
    from jevstral_b200._lib import JvHeads

    v = dict(src=64, out=64, in_token=n * 128, in_head=128, out_token=n * 128, out_head=128, heads=n, temperature=0)
    v.update(change)
    return JvHeads(*v.values())


def test_structs_match_a_c_compiler(tmp_path):
    from jevstral_b200 import _lib

    structs = {"jv_kv8_cache": _lib.JvKv8Cache, "jv_paged_batch": _lib.JvPagedBatch, "jv_rope_spec": _lib.JvRopeSpec,
               "jv_heads": _lib.JvHeads}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "jv.h"', "int main(void) {"]
    for st, cls in structs.items():
        lines.append(f'    printf("{st} sizeof %zu\\n", sizeof({st}));')
        lines += [f'    printf("{st} {f} %zu\\n", offsetof({st}, {"in" if f == "src" else f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text("\n".join(lines + ["    return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        st, name, value = line.split()
        cls = structs[st]
        assert int(value) == (C.sizeof(cls) if name == "sizeof" else getattr(cls, name).offset), (st, name)


@pytest.mark.parametrize("change", [dict(requests=0), dict(requests=4097), dict(max_new=0), dict(max_tokens=0),
                                    dict(max_tokens=(1 << 28) + 1), dict(max_blocks=0), dict(max_keys=-1),
                                    dict(max_keys=4 * 4 * 64 + 1), dict(group=0), dict(group=17), dict(pages=0),
                                    dict(work=72), dict(slots=68), dict(block_table=66), dict(status=0), dict(lengths=0),
                                    dict(starts=0), dict(request_of=0), dict(positions=0), dict(block_table=0), dict(work=0)])
def test_bad_batches_are_refused(change):
    from jevstral_b200._lib import JV_ERR_ARG, lib

    b, c, q = _batch(**change), _cache(), _heads(8)
    if "pages" in change:
        c.pages = b.pages
    assert lib.jv_paged_plan(C.byref(b), 64, 64, 64, 64, 64, None) == JV_ERR_ARG
    assert lib.jv_kv8_append(C.byref(c), C.byref(b), 1, C.byref(_heads(2)), C.byref(_heads(2)), None, None, 1, None) == JV_ERR_ARG
    assert lib.jv_kv8_attention(C.byref(c), C.byref(b), 1, C.byref(q), 0.1, 0, 64, 1 << 40, None) == JV_ERR_ARG
    if not set(change) & {"work", "slots", "block_table", "status", "lengths", "starts", "request_of", "positions"}:
        assert lib.jv_paged_work_bytes(C.byref(b)) == -1 and lib.jv_kv8_attention_bytes(C.byref(b), 2) == -1
    assert lib.jv_last_error()


@pytest.mark.parametrize("change", [dict(data=0), dict(scales=0), dict(data=72), dict(scales=68), dict(pages=0),
                                    dict(kv_heads=0), dict(kv_heads=1025), dict(page_bytes=2 * 16384 - 16),
                                    dict(page_bytes=2 * 16384 + 8), dict(scale_stride=12), dict(scale_stride=18), dict(pages=9)])
def test_bad_caches_are_refused(change):
    from jevstral_b200._lib import JV_ERR_ARG, lib

    c, b = _cache(**change), _batch()
    k = _heads(c.kv_heads)
    assert lib.jv_kv8_append(C.byref(c), C.byref(b), 1, C.byref(k), C.byref(k), None, None, 1, None) == JV_ERR_ARG
    assert lib.jv_kv8_attention(C.byref(c), C.byref(b), 1, C.byref(_heads(c.kv_heads * 4)), 0.1, 0, 64, 1 << 40, None) == JV_ERR_ARG
    if change != dict(pages=9):
        assert lib.jv_kv8_read(C.byref(c), 64, 1, 1, 64, 64, 256, None, None) == JV_ERR_ARG


def test_null_arguments_and_bad_operands_are_refused():
    from jevstral_b200._lib import JV_ERR_ARG, JV_ERR_UNSUPPORTED, JvRopeSpec, lib

    b, c, k, q = _batch(), _cache(), _heads(2), _heads(8)
    ref = C.byref
    plan = [64] * 5
    for i in range(5):
        args = plan[:i] + [None] + plan[i + 1:]
        assert lib.jv_paged_plan(ref(b), *args, None) == JV_ERR_ARG
    assert lib.jv_paged_plan(None, *plan, None) == JV_ERR_ARG
    append = lambda **o: lib.jv_kv8_append(o.get("c", ref(c)), o.get("b", ref(b)), o.get("type", 1), o.get("k", ref(k)),  # noqa: E731
                                           o.get("v", ref(k)), o.get("rope"), o.get("q"), o.get("out", 1), None)
    spec = JvRopeSpec()
    assert lib.jv_rope_init(ref(spec), 0, 64, 1e4, 0, 1, 0, 32, 1, 1) == 0
    for o in (dict(c=None), dict(b=None), dict(k=None), dict(v=None), dict(k=ref(_heads(3))), dict(k=ref(_heads(2, src=0))),
              dict(v=ref(_heads(2, src=65))), dict(k=ref(_heads(2, in_token=-1))), dict(q=ref(q)),
              dict(rope=ref(spec), q=ref(_heads(7))), dict(rope=ref(spec), q=ref(_heads(8, src=64, out=64)), out=30),
              dict(rope=ref(spec), q=ref(_heads(8, src=64, out=128, out_head=64)))):
        assert append(**o) == JV_ERR_ARG, o
    assert append(type=8) == JV_ERR_UNSUPPORTED and append(rope=ref(spec), q=ref(_heads(8, out=128)), out=2) == JV_ERR_UNSUPPORTED
    assert lib.jv_rope_init(ref(spec), 0, 36, 1e4, 0, 1, 0, 32, 1, 1) == 0
    assert append(rope=ref(spec)) == JV_ERR_UNSUPPORTED
    attend = lambda **o: lib.jv_kv8_attention(ref(c), ref(b), o.get("type", 1), o.get("q", ref(q)), o.get("scale", 0.1),  # noqa: E731
                                              o.get("window", 0), o.get("ws", 64), o.get("bytes", 1 << 40), None)
    for o in (dict(q=None), dict(q=ref(_heads(6))), dict(q=ref(_heads(8, src=0))), dict(q=ref(_heads(8, out=0))),
              dict(q=ref(_heads(8, src=72))), dict(q=ref(_heads(8, out_token=1028))), dict(q=ref(_heads(8, in_head=132))),
              dict(window=-1), dict(scale=math.nan), dict(scale=math.inf), dict(ws=None), dict(ws=72), dict(bytes=16),
              dict(q=ref(_heads(8, out_head=64))), dict(q=ref(_heads(8, out_head=0)))):
        assert attend(**o) == JV_ERR_ARG, o
    assert attend(type=0) == JV_ERR_UNSUPPORTED
    for args in ((None, 1, 1, 64, 64, 256), (64, -1, 1, 64, 64, 256), (64, 1, 1, None, 64, 256), (64, 1, 1, 64, None, 256),
                 (64, 1, 1, 64, 64, 255), (64, 1, 1, 65, 64, 256), (68, 1, 1, 64, 64, 256)):
        assert lib.jv_kv8_read(ref(c), *args, None, None) == JV_ERR_ARG
    assert lib.jv_kv8_read(ref(c), 64, 1, 3, 64, 64, 256, None, None) == JV_ERR_UNSUPPORTED
    assert lib.jv_kv8_read(ref(c), 64, 0, 1, 64, 64, 256, None, None) == 0


def test_rope_refusals():
    from jevstral_b200._lib import JV_ERR_ARG, JV_ERR_UNSUPPORTED, JvHeads, JvRopeSpec, lib

    s = JvRopeSpec()
    ok = [0, 64, 1e4, 0, 1.0, 0, 32.0, 1.0, 1.0]
    for i, bad in ((0, 2), (0, -1), (1, 63), (1, 0), (1, 258), (2, 0.0), (2, math.inf), (2, math.nan), (3, 3), (8, math.inf)):
        args = ok[:i] + [bad] + ok[i + 1:]
        assert lib.jv_rope_init(C.byref(s), *args) == JV_ERR_ARG, (i, bad)
    assert lib.jv_rope_init(None, *ok) == JV_ERR_ARG
    assert lib.jv_rope_init(C.byref(s), 0, 64, 1e4, 1, 0.0, 0, 32, 1, 1) == JV_ERR_ARG
    assert lib.jv_rope_init(C.byref(s), 0, 64, 1e4, 2, 4.0, 0, 32, 1, 1) == JV_ERR_ARG
    assert lib.jv_rope_init(C.byref(s), *ok) == 0
    call = lambda x, n=1, type=1, dim=128, tokens=3, pos=64, spec=s: lib.jv_rope(  # noqa: E731
        C.byref(spec) if spec is not None else None, type, pos, tokens, dim, x, n, None)
    one = lambda **o: (JvHeads * 1)(_heads(8, **o))  # noqa: E731
    for bad in (call(one(), dim=62), call(one(), dim=127), call(one(), dim=258), call(one(), n=0), call(one(), n=3), call(None),
                call(one(src=0)), call(one(out=0)), call(one(src=65)), call(one(out=65)), call(one(), tokens=-1),
                call(one(), pos=None), call(one(), spec=None), call(one(in_token=-8)), call(one(out=4096, out_head=64)),
                call(one(out=4096, out_token=512)), call(one(out_token=2048)), call((JvHeads * 1)(_heads(0)))):
        assert bad == JV_ERR_ARG
    assert call(one(), type=8) == JV_ERR_UNSUPPORTED
    assert call(one(), tokens=0) == 0


@pytest.mark.parametrize("rot,base,factor,orig", [(128, 1e6, 16.0, 16384), (64, 1e4, 4.0, 4096), (32, 5e5, 1.0, 8192)])
def test_rotary_frequencies_follow_the_model_s_rule(rot, base, factor, orig):
    """Against the rule of Rope.cs:33-106 written out in Python's 64 bits; a turn is 2 pi, so each value may
    differ by a few roundings of 2^-53."""
    from jevstral_b200 import paged

    inv = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    plain = paged.rope_spec("half", rot, base)
    linear = paged.rope_spec("interleaved", rot, base, scaling="linear", factor=factor)
    yarn = paged.rope_spec("half", rot, base, scaling="yarn", factor=factor, original_context=orig, attn_factor=0.5)
    corr = [rot * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0)]
    low, high = max(0.0, math.floor(corr[0])), min(rot / 2 - 1.0, math.ceil(corr[1]))
    for i, f in enumerate(inv):
        keep = 1.0 - min(max((i - low) / max(0.001, high - low), 0.0), 1.0)
        mixed = f / factor * (1 - keep) + f * keep
        for spec, want in ((plain, f), (linear, f / factor), (yarn, mixed)):
            assert math.isclose(spec.turns[i] * 2 * math.pi, want, rel_tol=2 ** -48)
    assert plain.mscale == 1.0 and linear.mscale == 1.0
    assert math.isclose(yarn.mscale, 0.5 * (0.1 * math.log(factor) + 1.0), rel_tol=2 ** -23)


def test_sizes_grow_with_the_bounds():
    from jevstral_b200 import paged
    from jevstral_b200._lib import lib

    small = paged.work_bytes(1, 1, 1, 1, 64, 1)
    assert 0 < small <= paged.work_bytes(64, 8, 512, 128, 64 * 128 * 64, 4)
    with pytest.raises(ValueError):
        paged.work_bytes(0, 1, 1, 1, 64, 1)
    b = _batch()
    assert lib.jv_kv8_attention_bytes(C.byref(b), 2) > 0
    assert lib.jv_kv8_attention_bytes(C.byref(b), 0) == -1


def test_server_entry_points_check_their_handles():
    from jevstral_b200._lib import JV_ERR_ARG, lib

    h = C.c_void_p()
    assert lib.jv_server_create(None, 1, 1, 1, 0, C.byref(h)) == JV_ERR_ARG
    one = (C.c_int32 * 1)(1)
    assert lib.jv_server_forward(None, one, one, one, 0, None) == JV_ERR_ARG
    assert lib.jv_server_release(None, 0) == JV_ERR_ARG
    assert lib.jv_server_length(None, 0) == -1 and lib.jv_server_bytes_per_position(None) == 0
    lib.jv_server_destroy(None)
