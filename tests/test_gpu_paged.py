"""The paged-batch operators on the GPU against plain implementations in 64 bits (or, where a result is an
integer or an exactly rounded value, against the same arithmetic bit for bit).

Tolerances: a rounding is off by at most half a step of its type (HALF). The attention's softmax weights are
rounded once to fp16, so an output may differ by 2^-11 of sum p |v|, plus a weight's subnormal half step
2^-25 per key, plus fp32 arithmetic (taken as 2^-13 of sum p |v|: exponents below 2^7 carry an error of 2^-17
or less into a weight), plus its own rounding."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
RANGE, OOM, NUMERIC = 2, 9, 10


class Server:
    """A cache and a plan as a serving program keeps them, with a plain record of every request."""

    def __init__(self, requests, kv_heads, group, pages, max_new, max_tokens, max_blocks, max_keys=None, page_bytes=None,
                 scale_stride=None, seed=0):
        from jevstral_b200 import paged

        self.p, self.g, self.group, self.pages = paged, kv_heads, group, pages
        self.requests, self.max_tokens, self.max_blocks, self.max_new = requests, max_tokens, max_blocks, max_new
        dev = dict(device="cuda")
        self.page_bytes = page_bytes or kv_heads * 16384
        self.scale_stride = scale_stride or kv_heads * 8
        # stale memory: bytes of any value, scales that are not numbers
        self.data = torch.randint(-128, 128, (pages * self.page_bytes,), dtype=torch.int8, **dev)
        self.scales = torch.full((pages * self.scale_stride,), math.nan, **dev)
        max_keys = requests * max_blocks * 64 if max_keys is None else max_keys
        rng = np.random.default_rng(seed)
        self.free = torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda()
        self.n_free = torch.tensor([pages], dtype=torch.int32, **dev)
        self.table = torch.full((requests, max_blocks), -7, dtype=torch.int32, **dev)
        self.lengths = torch.zeros(requests, dtype=torch.int32, **dev)
        self.starts = torch.full((requests + 1,), -7, dtype=torch.int32, **dev)
        self.request_of, self.positions = (torch.full((max_tokens,), -7, dtype=torch.int32, **dev) for _ in range(2))
        self.slots = torch.full((max_tokens,), -7, dtype=torch.int64, **dev)
        self.status = torch.zeros(2, dtype=torch.int32, **dev)
        self.work = torch.full((paged.work_bytes(requests, max_new, max_tokens, max_blocks, max_keys, group),), 255,
                               dtype=torch.uint8, **dev)
        self.batch = paged.batch(requests, max_new, max_tokens, max_blocks, max_keys, group, pages,
                                 *(t.data_ptr() for t in (self.table, self.lengths, self.starts, self.request_of,
                                                          self.positions, self.slots, self.work, self.status)))
        self.cache = paged.cache(self.data.data_ptr(), self.scales.data_ptr(), pages, kv_heads, self.page_bytes,
                                 self.scale_stride)
        self.ws_bytes = paged.attention_bytes(self.batch, kv_heads)
        self.ws = torch.full((max(self.ws_bytes, 1),), 255, dtype=torch.uint8, **dev)

    def plan(self, new, cached=None, stream=0):
        self.new = torch.as_tensor(new, dtype=torch.int32).cuda()
        cached = self.lengths if cached is None else cached
        self.p.plan(self.batch, cached.data_ptr(), self.new.data_ptr(), self.free.data_ptr(), self.n_free.data_ptr(),
                    self.n_free.data_ptr(), stream)

    def append(self, k, v, dtype, rope=None, q=None, q_out=None, out_dtype="f16", temperature=False, stream=0):
        h = lambda x, o=None: self.p.heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1),  # noqa: E731
                                           *(() if o is None else (o.data_ptr(), o.stride(0), o.stride(1), temperature)))
        self.p.kv8_append(self.cache, self.batch, dtype, h(k), h(v), rope, None if q is None else h(q, q_out), out_dtype, stream)

    def attend(self, q, dtype, scale=None, window=0, out=None, stream=0):
        out = torch.full_like(q, math.nan) if out is None else out
        heads = self.p.heads(q.data_ptr(), q.shape[1], q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1))
        self.p.kv8_attention(self.cache, self.batch, dtype, heads, scale or 128 ** -0.5, window, self.ws.data_ptr(),
                             self.ws_bytes, stream)
        return out

    def fill(self, k, v, r, n):
        """k, v: [n, g, 128] float64 cpu of request r as its first n tokens, exactly as int8 x scale: written by hand."""
        blocks = -(-n // 64)
        pages = self.table[r, :blocks].long().cpu()
        return pages

    def stored(self, r, n):
        """[2][n][g][128] float64: what request r's pages hold for its first n tokens."""
        pages = self.table[r, :-(-n // 64)].long()
        d = self.data.view(self.pages, self.page_bytes)[pages, :self.g * 16384].view(-1, self.g, 2, 64, 128).double()
        s = self.scales.view(self.pages, self.scale_stride)[pages, :self.g * 8].view(-1, self.g, 2, 4).double()
        x = d * s.repeat_interleave(16, -1)[..., None]
        return x.permute(2, 0, 3, 1, 4).reshape(2, -1, self.g, 128)[:, :n].cpu()


def check_plan(s, cached, new, table_before, free_before, n_free_before, rows_before):
    want_len = [c + n for c, n in zip(cached, new)]
    assert s.lengths.tolist() == want_len
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    assert s.starts.tolist() == starts
    table, at = [list(row) for row in table_before], n_free_before
    for r, (c, n) in enumerate(zip(cached, new)):
        for b in range(-(-c // 64), -(-(c + n) // 64)):
            at -= 1
            table[r][b] = free_before[at]
    assert s.table.tolist() == table and s.n_free.item() == at
    req, pos, slot = (list(x) for x in rows_before)
    for r, n in enumerate(new):
        for i in range(n):
            t, p = starts[r] + i, cached[r] + i
            req[t], pos[t], slot[t] = r, p, table[r][p // 64] * 64 + p % 64
    assert s.request_of.tolist() == req and s.positions.tolist() == pos and s.slots.tolist() == slot


@pytest.mark.parametrize("requests,hi_new,hi_len,big", [(1, 1, 0, 0), (1, 1, 63, 0), (1, 2000, 100, 2000), (7, 3, 200, 0),
                                                        (33, 70, 129, 0), (1025, 2, 64, 0), (4096, 1, 130, 0),
                                                        (300, 64, 64, 700)])
def test_plans_of_consecutive_steps(requests, hi_new, hi_len, big):
    rng = random.Random(requests * 31 + hi_new)
    blocks = -(-(hi_len + 3 * max(hi_new, big)) // 64) + 1
    s = Server(requests, 1, 4, requests * blocks, max(hi_new, big), requests * hi_new + big + 5, blocks, seed=requests)
    first = [rng.randrange(hi_len + 1) for _ in range(requests)]
    for step in range(3):
        cached = s.lengths.tolist()
        new = [min(x, hi_new) for x in first] if step == 0 else [rng.randrange(hi_new + 1) for _ in range(requests)]
        if big:
            new[requests // 2] = big
        before = s.table.tolist(), s.free.tolist(), s.n_free.item(), [x.tolist() for x in (s.request_of, s.positions, s.slots)]
        s.plan(new)
        torch.cuda.synchronize()
        assert s.status.tolist() == [0, 0]
        check_plan(s, cached, new, *before)


@pytest.mark.parametrize("what", ["long", "negative", "new", "tokens", "keys", "free", "page", "overflow"])
def test_a_step_beyond_its_bounds_changes_nothing(what):
    s = Server(4, 1, 4, 12, 40, 100, 4, max_keys=4 * 4 * 64 if what != "keys" else 180, seed=3)
    s.plan([30, 64 - 30, 0, 5][:4] if what != "keys" else [30, 34, 0, 5])
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    state = [x.clone() for x in (s.table, s.request_of, s.positions, s.slots, s.free)]
    cached, new = s.lengths.tolist(), [10, 0, 3, 1]
    code = RANGE
    if what == "long":
        cached, new = [250, 0, 0, 0], [10, 0, 0, 0]
    elif what == "negative":
        new[2] = -1
    elif what == "new":
        new[0] = 41
    elif what == "tokens":
        new = [40, 30, 30, 1]
    elif what == "keys":
        new = [40, 40, 40, 0]
    elif what == "overflow":
        cached, new = [2 ** 31 - 1, 0, 0, 0], [40, 0, 0, 0]
    elif what == "free":
        s.n_free.fill_(1)
        new, code = [40, 40, 3, 1], OOM
    elif what == "page":
        s.free[s.n_free.item() - 2] = 12
        new = [40, 40, 3, 1]
        state[4] = s.free.clone()
    n_free = s.n_free.item()
    s.lengths.copy_(torch.tensor(cached, dtype=torch.int32))
    s.plan(new)
    torch.cuda.synchronize()
    assert s.status[0].item() == code and s.status[1].item() > 0
    assert s.lengths.tolist() == cached and s.starts.tolist() == [0] * 5 and s.n_free.item() == n_free
    for a, b in zip(state, (s.table, s.request_of, s.positions, s.slots, s.free)):
        assert torch.equal(a, b)
    # the operators after it do nothing
    data, k = s.data.clone(), torch.ones(100, 1, 128, device="cuda", dtype=torch.float16)
    s.append(k, k, "f16")
    out = s.attend(torch.ones(100, 4, 128, device="cuda", dtype=torch.float16), "f16")
    torch.cuda.synchronize()
    assert torch.equal(data, s.data) and torch.isnan(out).all() and s.status[0].item() == code


# ------------------------------------------------------------------------------------------ rope


def rope64(x, pos, spec, temperature=False):
    """x [T, H, D] float64 numpy; the formula in 64 bits."""
    n = spec.rotary_dim // 2
    turns = np.array(spec.turns[:n])
    angle = 2 * np.pi * np.modf(np.asarray(pos, np.float64)[:, None] * turns)[0]
    c, s = np.cos(angle)[:, None] * spec.mscale, np.sin(angle)[:, None] * spec.mscale
    y = x.copy()
    a, b = (slice(0, n), slice(n, 2 * n)) if spec.layout else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    if temperature:
        y *= (1 + spec.temperature_scale * np.log(1 + np.floor(np.asarray(pos) / spec.temperature_ctx)))[:, None, None]
    return y


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,far,pad,offset", [
    (1, 1, 1, 128, 128, 0, 0, 0), (5, 32, 8, 128, 128, 1 << 20, 0, 0), (17, 3, 1, 128, 64, 131071, 8, 0),
    (33, 4, 2, 64, 32, 5000, 0, 0), (2, 5, 3, 80, 20, 5000, 3, 1), (19, 2, 2, 256, 256, 40000, 0, 0),
    (64, 7, 1, 6, 2, 99, 1, 1), (300, 8, 8, 128, 96, 2 ** 31 - 400, 8, 8), (16, 6, 2, 72, 48, 1000, 4, 2)])
def test_rope(dtype, layout, tokens, heads, kv, dim, rot, far, pad, offset):
    from jevstral_b200 import paged

    spec = paged.rope_spec(layout, rot, 1e4, scaling="yarn" if dim == 64 else "none", factor=8.0, original_context=1024,
                           temperature_scale=0.1, temperature_context=512)
    gen = torch.Generator("cuda").manual_seed(tokens * dim)
    flat = torch.randn(tokens * (heads + kv) * (dim + pad) + offset, generator=gen, device="cuda").to(TYPE[dtype])
    x = flat[offset:].view(tokens, heads + kv, dim + pad)[..., :dim]
    pos = torch.arange(far, far + tokens, dtype=torch.int64).to(torch.int32).cuda()
    pos = pos[torch.randperm(tokens, generator=torch.Generator().manual_seed(1)).cuda()]
    out = torch.full((heads + kv, tokens, dim), 7.0, device="cuda", dtype=TYPE[dtype])  # head-major outputs
    ops = [paged.heads(t.data_ptr(), t.shape[1], t.stride(0), t.stride(1), o.data_ptr(), o.stride(1), o.stride(0), tmp)
           for t, o, tmp in ((x[:, :heads], out[:heads], True), (x[:, heads:], out[heads:], False))]
    before = flat.clone()
    paged.rope(spec, dtype, pos.data_ptr(), tokens, dim, *ops)
    torch.cuda.synchronize()
    assert torch.equal(before, flat)
    x64, p = x.double().cpu().numpy(), pos.cpu().numpy()
    want = np.concatenate([rope64(x64[:, :heads], p, spec, True), rope64(x64[:, heads:], p, spec)], 1)
    # cos and sin to 3 units of 2^-23 (reduction, sincospi, mscale), two products, a sum, the temperature's
    # logarithm and product; then the rounding to the type
    n = rot // 2
    mag = np.abs(x64).copy()
    a, b = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    both = np.abs(x64[..., a]) + np.abs(x64[..., b])
    mag[..., a] = mag[..., b] = both * spec.mscale
    grown = np.abs(want) / np.maximum(np.abs(rope64(x64, p, spec)), 1e-300)
    tol = 8 * 2.0 ** -23 * mag * np.maximum(grown, 1) + HALF[dtype] * np.abs(want) * 1.001 + 2.0 ** -25 * (dtype == "f16")
    got = out.double().cpu().numpy().transpose(1, 0, 2)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())
    # in place gives the same bits
    if offset == 0 and pad == 0:
        paged.rope(spec, dtype, pos.data_ptr(), tokens, dim, paged.heads(x.data_ptr(), heads, x.stride(0), x.stride(1), x.data_ptr(), temperature=True),
                   paged.heads(x[:, heads:].data_ptr(), kv, x.stride(0), x.stride(1), x[:, heads:].data_ptr()))
        torch.cuda.synchronize()
        assert torch.equal(x, out.transpose(0, 1))


# ------------------------------------------------------------------------------------------ append and read


class Blocks:
    """The cache's rule in numpy fp32, operation for operation: (int8 [n, 128], scale) per request, block, head, K/V."""

    def __init__(self):
        self.q, self.s = {}, {}

    def append(self, key, row, x):
        """x [n, 128] fp32 into rows row.. of block `key`."""
        q = self.q.setdefault(key, np.zeros((16, 128), np.int8))
        finite = np.isfinite(x)
        amax = np.float32(np.abs(np.where(finite, x, 0)).max(initial=0))
        amax = np.float32(0) if amax < np.float32(2.0 ** -100) else amax
        scale = np.float32(amax / np.float32(127))
        inv = np.float32(127) / amax if amax > 0 else np.float32(0)
        had = self.s.get(key, np.float32(0)) if row else np.float32(0)
        if had > scale:
            scale, inv = had, np.float32(1) / had
        if row and had != scale:
            q[:row] = np.rint(q[:row].astype(np.float32) * np.float32(had / scale)).astype(np.int8)
        with np.errstate(invalid="ignore", over="ignore"):
            y = np.rint(np.where(np.isnan(x), np.float32(0), x) * inv)
            y = np.where(np.isnan(y), 0, y)  # an infinity in a block of zeros
        q[row:row + len(x)] = np.clip(y, -127, 127).astype(np.int8)
        self.s[key] = scale


def steps_of(rng, requests, hi, n):
    return [[rng.choice([0, 1, 1, rng.randrange(hi + 1)]) for _ in range(requests)] for _ in range(n)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("requests,g,hi,pad,offset", [(1, 1, 1, 0, 0), (3, 2, 40, 8, 0), (9, 8, 5, 0, 0), (4, 3, 200, 1, 1),
                                                      (2, 1, 17, 4, 4)])
def test_append_is_the_rule_bit_for_bit(dtype, requests, g, hi, pad, offset):
    """Several steps of growing requests: every stored int8 and scale equals the rule's, and nothing else in
    the cache changes (garbage behind the last token and other pages stay)."""
    rng = random.Random(requests * 7 + hi)
    blocks = 5 * (hi // 64 + 1) + 1
    s = Server(requests, g, 4, requests * blocks + 2, max(hi, 1), requests * max(hi, 1), blocks, page_bytes=g * 16384 + 32,
               scale_stride=g * 8 + 4, seed=hi)
    gen = torch.Generator("cuda").manual_seed(hi)
    rule, data = Blocks(), s.data.clone()
    for step, new in enumerate(steps_of(rng, requests, hi, 6)):
        old = s.lengths.tolist()
        s.plan(new)
        n = sum(new)
        flat = (torch.randn(max(n, 1) * 2 * (g * 128 + pad) + offset, generator=gen, device="cuda") * 4.0 ** (step % 3)).to(TYPE[dtype])
        kv = flat[offset:].view(max(n, 1), 2, g * 128 + pad)[..., :g * 128].unflatten(-1, (g, 128))
        s.append(kv[:, 0], kv[:, 1], dtype)
        torch.cuda.synchronize()
        x, starts = kv.float().cpu().numpy(), s.starts.tolist()
        for r in range(requests):
            p = old[r]
            while p < old[r] + new[r]:
                end = min(old[r] + new[r], (p // 16 + 1) * 16)
                for h in range(g):
                    for c in range(2):
                        rule.append((r, p // 16, h, c), p % 16, x[starts[r] + p - old[r]:starts[r] + end - old[r], c, h])
                p = end
    assert s.status.tolist() == [0, 0]
    table, lengths = s.table.tolist(), s.lengths.tolist()
    want = data.view(s.pages, s.page_bytes).cpu().numpy().copy()
    scales = np.full((s.pages, s.scale_stride), np.nan, np.float32)
    for (r, b, h, c), q in rule.q.items():
        page, rows = table[r][b // 4], min(16, lengths[r] - 16 * b)
        at = (h * 2 + c) * 8192 + (b % 4) * 2048
        want[page, at:at + rows * 128] = q[:rows].reshape(-1)
        scales[page, (h * 2 + c) * 4 + b % 4] = rule.s[(r, b, h, c)]
    assert np.array_equal(s.data.view(s.pages, s.page_bytes).cpu().numpy(), want)
    assert np.array_equal(s.scales.view(s.pages, s.scale_stride).cpu().numpy(), scales, equal_nan=True)


@pytest.mark.parametrize("layout,rot", [("interleaved", 128), ("half", 128), ("half", 64), ("interleaved", 24), ("half", 40)])
@pytest.mark.parametrize("dtype,out", [("f32", "f16"), ("bf16", "bf16"), ("f16", "f32")])
def test_append_rotates_on_the_way(layout, rot, dtype, out):
    """Keys rotated, then rounded to 8 bits: within half a step of the block's scale of the formula's value (and
    fp32 rounding of the rotation); queries as jv_rope's."""
    from jevstral_b200 import paged

    g, group = 2, 3
    spec = paged.rope_spec(layout, rot, 1e6, temperature_scale=0.1, temperature_context=64)
    s = Server(3, g, group, 20, 100, 200, 6, seed=rot)
    gen = torch.Generator("cuda").manual_seed(rot)
    for new in ([33, 100, 0], [1, 5, 70]):
        old = s.lengths.tolist()
        n = sum(new)
        s.plan(new)
        qkv = torch.randn(n, g * (group + 2), 128, generator=gen, device="cuda").to(TYPE[dtype])
        q, k, v = qkv[:, :g * group], qkv[:, g * group:g * group + g], qkv[:, g * group + g:]
        q_out = torch.full((n, g * group, 128), math.nan, device="cuda", dtype=TYPE[out])
        s.append(k, v, dtype, rope=spec, q=q, q_out=q_out, out_dtype=out, temperature=True)
        torch.cuda.synchronize()
        pos = np.concatenate([np.arange(o, o + c) for o, c in zip(old, new)])
        assert pos.tolist() == s.positions.tolist()[:n]
        k64, q64 = rope64(k.double().cpu().numpy(), pos, spec), rope64(q.double().cpu().numpy(), pos, spec, True)
        tol = HALF[out] * np.abs(q64) + 16 * 2.0 ** -23 * 8 + (2.0 ** -25 if out == "f16" else 0)
        assert (np.abs(q_out.double().cpu().numpy() - q64) <= tol).all()
        starts = s.starts.tolist()
        for r in range(3):
            got = s.stored(r, old[r] + new[r]).numpy()
            pages = s.table[r, :-(-max(s.lengths[r].item(), 1) // 64)].long()
            scale = s.scales.view(s.pages, g, 2, 4)[pages].permute(2, 0, 3, 1).reshape(2, -1, g).repeat_interleave(16, 1).double().cpu().numpy()
            for i in range(new[r]):
                p, t = old[r] + i, starts[r] + i
                for c, want in ((0, k64[t]), (1, v[t].double().cpu().numpy())):
                    step = scale[c, p][:, None]
                    assert (np.abs(got[c, p] - want) <= 0.5 * step * (1 + 2.0 ** -15) + 16 * 2.0 ** -23 * 8).all(), (r, p, c)
    assert s.status.tolist() == [0, 0]


def test_append_of_values_that_are_not_finite():
    s = Server(1, 2, 4, 4, 40, 40, 2)
    s.plan([20])
    k = torch.randn(20, 2, 128, device="cuda")
    v = torch.randn(20, 2, 128, device="cuda")
    k[3, 0, 5], k[4, 0, 6], k[5, 0, 7] = math.inf, -math.inf, math.nan
    v[:, 1] = 1e-38  # below 2^-100: stored as zeros
    s.append(k, v, "f32")
    torch.cuda.synchronize()
    assert s.status[0].item() == NUMERIC
    x = s.stored(0, 20)
    clean = torch.where(torch.isfinite(k), k, 0.0).double().cpu()
    amax = clean[:16].abs().amax((0, 2))
    assert torch.isfinite(x).all() and (x[1, :, 1] == 0).all()
    assert abs(x[0, 3, 0, 5].item() - amax[0].item()) < 1e-5 and abs(x[0, 4, 0, 6].item() + amax[0].item()) < 1e-5
    assert x[0, 5, 0, 7] == 0
    keep = torch.isfinite(k[:16]).cpu()
    assert ((x[0, :16] - clean[:16]).abs()[keep] <= (amax / 254 * 1.001)[None, :, None].expand(16, 2, 128)[keep]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
def test_read_gives_the_stored_values(dtype, pad, offset):
    g = 3
    s = Server(2, g, 4, 6, 100, 150, 2, page_bytes=g * 16384 + 64, scale_stride=g * 8 + 8)
    s.plan([100, 33])
    kv = torch.randn(133, 2, g, 128, device="cuda")
    s.append(kv[:, 0], kv[:, 1], "f32")
    slots = s.slots[:133].clone()
    slots[5], slots[77] = -1, -9
    slots = torch.cat([slots, slots[:1], torch.tensor([6 * 64, 1 << 40], device="cuda")])  # one again; two past the cache
    row = g * 128 + pad
    out = torch.full((2, len(slots) * row + offset), 5.0, device="cuda", dtype=TYPE[dtype])
    s.p.kv8_read(s.cache, slots.data_ptr(), len(slots), dtype, out[0, offset:].data_ptr(), out[1, offset:].data_ptr(), row,
                 s.status.data_ptr())
    torch.cuda.synchronize()
    assert s.status[0].item() == RANGE
    got = out[:, offset:].view(2, -1, row)
    want = torch.full_like(got, 5.0)
    for c in range(2):
        values = torch.cat([s.stored(0, 100)[c], s.stored(1, 33)[c]]).flatten(1).float().to(TYPE[dtype]).cuda()
        want[c, :133, :g * 128] = values
        want[c, 133, :g * 128] = values[0]
        want[c, [5, 77]] = 5.0
    assert torch.equal(got, want) and (out[:, :offset] == 5).all()


# ------------------------------------------------------------------------------------------ attention


def attend64(q, kv, at, scale, window):
    """q [n, H, 128], kv [2][len][g][128] float64, at [n] positions -> out, sum p |v|, largest |v|."""
    n, h = q.shape[:2]
    k, v = (x.repeat_interleave(h // kv.shape[2], 1) for x in (kv[0], kv[1]))
    s = torch.einsum("nhd,lhd->nhl", q, k) * scale
    key = torch.arange(kv.shape[1])
    hide = key[None] > at[:, None]
    if window:
        hide |= key[None] <= at[:, None] - window
    s = s.masked_fill(hide[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l, 0.0)
    return torch.einsum("nhl,lhd->nhd", p, v), torch.einsum("nhl,lhd->nhd", p, v.abs())


def compare(got, q, s, dtype, new, scale, window, lengths=None):
    lengths = s.lengths.tolist() if lengths is None else lengths
    t = 0
    for r, n in enumerate(new):
        if n == 0:
            continue
        kv = s.stored(r, lengths[r])
        at = torch.arange(lengths[r] - n, lengths[r])
        want, mag = attend64(q[t:t + n].double().cpu(), kv, at, scale, window)
        tol = HALF[dtype] * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + lengths[r] * 2.0 ** -25 * kv[1].abs().max() + 1e-30
        if dtype == "f16":
            tol = tol + 2.0 ** -25
        err = (got[t:t + n].double().cpu() - want).abs()
        assert (err <= tol).all(), (r, n, lengths[r], float((err / tol).max()))
        t += n
    if t < len(got):
        assert torch.isnan(got[t:]).all()  # rows behind the last token


ATTENTION = [
    # (lengths before, new, kv heads, group, window)
    ([0], [1], 1, 1, 0), ([15], [1], 2, 4, 0), ([63, 64, 65], [1, 1, 1], 2, 4, 0), ([255, 256, 1023], [1, 1, 1], 8, 4, 0),
    ([700, 0, 130], [1, 0, 1], 2, 8, 0), ([5, 300, 77], [2, 4, 3], 2, 4, 0), ([40, 500], [1, 1], 1, 16, 0),
    ([1000], [5], 1, 3, 0), ([0, 300], [16, 16], 3, 1, 0), ([3000, 10], [1, 1], 2, 4, 100), ([900, 20], [4, 4], 2, 2, 17),
    ([0], [17], 1, 1, 0), ([0, 129], [129, 64], 2, 4, 0), ([511, 3], [90, 200], 1, 8, 0), ([64, 0, 1000], [33, 1, 40], 2, 4, 0),
    ([200, 900], [150, 70], 2, 4, 64), ([0], [300], 2, 5, 0), ([0, 100], [257, 255], 1, 7, 33), ([33000], [1], 1, 4, 0),
    ([2000], [600], 1, 4, 1), ([10], [1], 1, 4, 1), ([1300, 40], [40, 1], 1, 4, 0), ([5000], [70], 2, 4, 0)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("old,new,g,group,window", ATTENTION)
def test_attention(dtype, old, new, g, group, window):
    scale = 128 ** -0.5
    requests, most = len(old), max(max(old), max(new))
    blocks = -(-max(a + b for a, b in zip(old, new)) // 64) + 1
    s = Server(requests, g, group, requests * blocks + 1, max(1, most), max(sum(old), sum(new)) + 3, blocks, seed=sum(old))
    gen = torch.Generator("cuda").manual_seed(sum(old) + sum(new))
    for step in (old, new):
        s.plan(step)
        kv = torch.randn(max(sum(step), 1), 2, g, 128, generator=gen, device="cuda") * (1 + 9 * (torch.arange(128, device="cuda") == 7))
        s.append(kv[:, 0], kv[:, 1], "f32")
    q = (2 * torch.randn(s.max_tokens, g * group, 128, generator=gen, device="cuda")).to(TYPE[dtype])
    got = s.attend(q, dtype, scale, window)
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    compare(got, q, s, dtype, new, scale, window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[1, 3, 2], [40, 1, 130]])
def test_a_request_s_bits_do_not_depend_on_the_batch(dtype, new):
    """The same request alone, and among others in another order, with strided queries and outputs."""
    old, g, group = [700, 90, 1500], 2, 4
    outs = []
    for order in ([0, 1, 2], [2, 0, 1], [0], [1], [2]):
        s = Server(len(order), g, group, 90, 2000, 3000, 40, seed=len(outs))
        for step in (old, new):
            s.plan([step[r] for r in order])
            kv = []
            for r in order:
                gen = torch.Generator("cuda").manual_seed(100 * r + (step is new))
                kv.append(torch.randn(step[r], 2, g, 128, generator=gen, device="cuda"))
            kv = torch.cat(kv)
            s.append(kv[:, 0], kv[:, 1], "f32")
        q = torch.cat([torch.randn(new[r], g * group, 128, generator=torch.Generator("cuda").manual_seed(r), device="cuda")
                       for r in order]).to(TYPE[dtype])
        wide = torch.zeros(len(q), g * group + 3, 136, device="cuda", dtype=q.dtype)
        wide[:, 1:-2, :128] = q
        out = torch.zeros(g * group, len(q), 128, device="cuda", dtype=q.dtype)
        s.attend(wide[:, 1:-2, :128], dtype, out=out.transpose(0, 1))
        torch.cuda.synchronize()
        got, t = {}, 0
        for r in order:
            got[r] = out[:, t:t + new[r]].clone()
            t += new[r]
        outs.append(got)
    for got in outs[1:]:
        for r, x in got.items():
            assert torch.equal(x, outs[0][r]), r


def test_blocks_whose_scales_differ_by_far():
    """V scales from 1e-6 to 1e6 and blocks of zeros: the weights carry the scale, so large and small blocks must
    not push each other out of fp16's range."""
    s = Server(2, 1, 4, 40, 400, 800, 8, seed=5)
    s.plan([333, 200])
    gen = torch.Generator("cuda").manual_seed(8)
    kv = torch.randn(533, 2, 1, 128, generator=gen, device="cuda")
    mag = 10.0 ** (torch.randint(-6, 7, (40,), generator=gen, device="cuda").repeat_interleave(16)[:533].float())
    kv[:, 1] *= mag[:, None, None]
    kv[160:176] = 0
    kv[333:, 1] *= 0  # the second request's values are all zero
    s.append(kv[:, 0], kv[:, 1], "f32")
    s.plan([1, 1])
    last = torch.randn(2, 2, 1, 128, generator=gen, device="cuda")
    last[1, 1] = 0
    s.append(last[:, 0], last[:, 1], "f32")
    for amp in (1.0, 12.0):
        q = (amp * torch.randn(s.max_tokens, 4, 128, generator=gen, device="cuda")).to(torch.float16)
        q[0] = kv[40, 0].half() * amp  # one row that picks a key
        got = s.attend(q, "f16")
        torch.cuda.synchronize()
        compare(got[:2], q, s, "f16", [1, 1], 128 ** -0.5, 0)
        assert (got[1] == 0).all()


@pytest.mark.parametrize("amp", [1e-30, 1e-8, 300.0, 1e30])
def test_bf16_queries_beyond_the_range_of_fp16(amp):
    s = Server(1, 1, 4, 8, 300, 300, 5)
    s.plan([290])
    kv = torch.randn(290, 2, 1, 128, device="cuda")
    s.append(kv[:, 0], kv[:, 1], "f32")
    s.plan([3])
    s.append(kv[:3, 0], kv[:3, 1], "f32")
    q = (amp * torch.randn(300, 4, 128, device="cuda")).to(torch.bfloat16)
    scale = 0.05 / amp if amp > 1 else min(0.05 / amp, 1e30)
    got = s.attend(q, "bf16", scale)
    torch.cuda.synchronize()
    compare(got, q, s, "bf16", [3], scale, 0)


def test_offsets_past_32_bits():
    """Pages 48 MB apart: the cache spans more than 2^32 bytes, its scales more than 2^31."""
    g, pages, page = 2, 100, 48 << 20
    s = Server(2, g, 4, pages, 200, 400, 4, page_bytes=page, scale_stride=6 << 20, seed=9)
    s.free.copy_(torch.arange(pages, dtype=torch.int32))  # the highest pages are taken first
    s.plan([200, 150])
    kv = torch.randn(350, 2, g, 128, device="cuda")
    s.append(kv[:, 0], kv[:, 1], "f32")
    assert s.table[:, 0].min().item() * page > 2 ** 32
    s.plan([1, 20])
    s.append(kv[:21, 0], kv[:21, 1], "f32")
    q = torch.randn(400, 8, 128, device="cuda", dtype=torch.float16)
    got = s.attend(q, "f16")
    k_out = torch.empty(2, 21, g, 128, device="cuda")
    s.p.kv8_read(s.cache, s.slots.data_ptr(), 21, "f32", k_out[0].data_ptr(), k_out[1].data_ptr(), g * 128, s.status.data_ptr())
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    compare(got, q, s, "f16", [1, 20], 128 ** -0.5, 0)
    assert torch.equal(k_out[:, 0].cpu(), s.stored(0, 201)[:, 200].float())  # int8 x scale, rounded once
    assert torch.equal(k_out[:, 1:].cpu(), s.stored(1, 170)[:, 150:].float())


def test_bad_pages_are_reported_and_not_used():
    s = Server(2, 1, 4, 10, 200, 400, 4)
    s.plan([100, 100])
    kv = torch.randn(200, 2, 1, 128, device="cuda")
    s.append(kv[:, 0], kv[:, 1], "f32")
    torch.cuda.synchronize()
    s.plan([1, 1])
    good = s.table.clone()
    for bad in (-1, 10, 2 ** 31 - 1, -2 ** 31):
        s.table[0, :2] = bad
        data = s.data.clone()
        s.append(kv[:2, 0], kv[:2, 1], "f32")
        torch.cuda.synchronize()
        assert s.status[0].item() == RANGE
        changed = (data != s.data).view(10, -1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= {good[1, 1].item()}
        s.status.zero_()
        q = torch.randn(400, 4, 128, device="cuda", dtype=torch.float16)
        got = s.attend(q, "f16")
        torch.cuda.synchronize()
        assert s.status[0].item() == RANGE
        want = attend64(q[1:2].double().cpu(), s.stored(1, 101), torch.tensor([100]), 128 ** -0.5, 0)[0]
        assert (got[1].double().cpu() - want[0]).abs().max() < 1e-2
        s.status.zero_()


# ------------------------------------------------------------------------------------------ together


def test_a_captured_decode_step_replays_with_other_lengths():
    """plan + append (rotating) + attention as one CUDA graph on a side stream: replayed steps continue the
    requests exactly as the same calls made one by one."""
    from jevstral_b200 import paged

    g, group, steps = 2, 4, 70
    spec = paged.rope_spec("half", 64, 1e4)
    first = [60, 3, 250]
    gen = torch.Generator("cuda").manual_seed(2)
    prompt = torch.randn(sum(first), g * (group + 2), 128, generator=gen, device="cuda").half()
    inputs = torch.randn(steps, 3, g * (group + 2), 128, generator=gen, device="cuda").half()
    results = []
    for graph in (False, True):
        s = Server(3, g, group, 40, 250, 320, 8, seed=4)
        x, q_out, out = (torch.zeros(n, h, 128, device="cuda", dtype=torch.float16)
                         for n, h in ((320, g * (group + 2)), (320, g * group), (320, g * group)))
        one = torch.ones(3, dtype=torch.int32, device="cuda")

        def step(stream, new):
            s.p.plan(s.batch, s.lengths.data_ptr(), new.data_ptr(), s.free.data_ptr(), s.n_free.data_ptr(),
                     s.n_free.data_ptr(), stream)
            s.append(x[:, g * group:g * group + g], x[:, g * group + g:], "f16", rope=spec, q=x[:, :g * group], q_out=q_out,
                     stream=stream)
            s.attend(q_out, "f16", out=out, stream=stream)

        x[:sum(first)] = prompt
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(side.cuda_stream, torch.tensor(first, dtype=torch.int32, device="cuda"))
            side.synchronize()
            if graph:
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=side):
                    step(torch.cuda.current_stream().cuda_stream, one)
            kept = []
            for i in range(steps):
                x[:3] = inputs[i]
                if graph:
                    captured.replay()
                else:
                    step(side.cuda_stream, one)
                kept.append(out[:3].clone())
            side.synchronize()
        assert s.status.tolist() == [0, 0] and s.lengths.tolist() == [n + steps for n in first]
        results.append(torch.stack(kept))
        compare(kept[-1], q_out[:3], s, "f16", [1, 1, 1], 128 ** -0.5, 0)
    assert torch.equal(*results)


def test_a_prefix_shared_by_requests():
    """Full pages shared through the block tables: requests that continue one prompt see its keys, and writing
    their own tokens leaves it as it is."""
    g, group = 2, 4
    s = Server(3, g, group, 12, 128, 200, 4, seed=6)
    s.plan([128, 0, 0])
    kv = torch.randn(128, 2, g, 128, device="cuda")
    s.append(kv[:, 0], kv[:, 1], "f32")
    s.table[1:, :2] = s.table[0, :2]
    s.lengths[1:] = 128
    torch.cuda.synchronize()
    prompt = s.stored(0, 128)
    s.plan([1, 20, 3])
    more = torch.randn(24, 2, g, 128, device="cuda")
    s.append(more[:, 0], more[:, 1], "f32")
    q = torch.randn(200, g * group, 128, device="cuda", dtype=torch.bfloat16)
    got = s.attend(q, "bf16")
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    for r in range(3):
        assert torch.equal(s.stored(r, 128), prompt)
    assert len(set(s.table[:, 2].tolist())) == 3
    compare(got, q, s, "bf16", [1, 20, 3], 128 ** -0.5, 0)


def test_two_calls_at_once_on_streams_of_their_own():
    """Two servers on two streams, interleaved: the same bits as one after the other."""
    outs = []
    for together in (False, True):
        streams = [torch.cuda.Stream() if together else torch.cuda.current_stream() for _ in range(2)]
        servers = [Server(8, 2, 4, 300, 900, 4000, 32, seed=i) for i in range(2)]
        data = []
        for i in range(2):
            gen = torch.Generator("cuda").manual_seed(i)
            data.append((torch.randn(8 * 400, 2, 2, 128, generator=gen, device="cuda"),
                         torch.randn(4000, 8, 128, generator=gen, device="cuda").half()))
        torch.cuda.synchronize()
        got = [[], []]
        for new in ([400] * 8, [1] * 8, [3, 50] * 4):
            for i, s in enumerate(servers):
                with torch.cuda.stream(streams[i]):
                    st = streams[i].cuda_stream
                    s.plan(new, stream=st)
                    n = sum(new)
                    s.append(data[i][0][:n, 0], data[i][0][:n, 1], "f32", stream=st)
                    got[i].append(s.attend(data[i][1][:max(n, 1)], "f16", stream=st))
        torch.cuda.synchronize()
        outs.append([torch.cat(x) for x in got])
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_device_memory_is_required():
    from jevstral_b200 import paged
    from jevstral_b200._lib import ArgumentError

    s = Server(1, 1, 4, 2, 4, 4, 2)
    pinned = torch.zeros(2 * 16384, dtype=torch.int8).pin_memory()
    c = paged.cache(pinned.data_ptr(), s.scales.data_ptr(), 2, 1)
    k = torch.zeros(4, 1, 128, device="cuda")
    h = paged.heads(k.data_ptr(), 1, 128, 128)
    with pytest.raises(ArgumentError):
        paged.kv8_append(c, s.batch, "f32", h, h)


# ------------------------------------------------------------------------------------------ at the edges


def filled(requests, g, group, first, new, dtype, seed, **more):
    """A server whose requests hold `first` tokens and are planned and appended for `new` more; queries for them."""
    most = max(max(first), max(new))
    blocks = -(-max(a + b for a, b in zip(first, new)) // 64)
    s = Server(requests, g, group, requests * blocks, most, max(sum(first), sum(new)), blocks, seed=seed, **more)
    gen = torch.Generator("cuda").manual_seed(seed)
    for step in (first, new):
        s.plan(step)
        kv = torch.randn(max(sum(step), 1), 2, g, 128, generator=gen, device="cuda")
        s.append(kv[:, 0], kv[:, 1], "f32")
    q = torch.randn(sum(new), g * group, 128, generator=gen, device="cuda").to(TYPE[dtype])
    return s, q


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[3, 1], [60, 33]])
def test_a_row_that_is_not_finite_stays_its_own(dtype, new):
    s, q = filled(2, 2, 4, [300, 90], new, dtype, 3)
    want = s.attend(q, dtype)
    for bad in (math.nan, math.inf):
        p = q.clone()
        p[1, 3, 17] = bad
        got = s.attend(p, dtype)
        torch.cuda.synchronize()
        assert not torch.isfinite(got[1, 3]).all()
        got[1, 3] = want[1, 3]
        assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0])
@pytest.mark.parametrize("new", [[2], [50]])
def test_scales_of_any_sign(scale, new):
    s, q = filled(1, 2, 4, [260], new, "f16", 4)
    out = torch.empty_like(q)
    h = s.p.heads(q.data_ptr(), 8, q.stride(0), q.stride(1), out.data_ptr())
    s.p.kv8_attention(s.cache, s.batch, "f16", h, scale, 0, s.ws.data_ptr(), s.ws_bytes)
    torch.cuda.synchronize()
    compare(out, q, s, "f16", new, scale, 0)


@pytest.mark.parametrize("new", [[2, 1], [40, 70]])
def test_attention_in_place_and_repeated(new):
    """The output over the queries, and the same call again on an output that holds the last: the same bits."""
    s, q = filled(2, 2, 4, [700, 100], new, "bf16", 5)
    want = s.attend(q, "bf16")
    for _ in range(3):
        assert torch.equal(s.attend(q, "bf16"), want)
    p = q.clone()
    s.attend(p, "bf16", out=p)
    torch.cuda.synchronize()
    assert torch.equal(p, want)


@pytest.mark.parametrize("g,group,first,new", [
    (1, 2, [140001], [1]), (1, 2, [140001], [2]), (1, 2, [530000], [1]), (1, 2, [140001], [40]),
    (2, 4, [20000, 9000, 5000, 3000, 70], [40, 64, 128, 33, 50]), (1, 4, [9000, 9001, 30000], [200, 33, 64]),
    (3, 1, [17000, 6000], [300, 512]), (1, 8, [16000, 16000, 2000, 16000], [40, 3, 40, 1])])
def test_long_contexts_and_their_splits(g, group, first, new):
    """The longer chunks (1024 and 2048 keys), up to 16 splits of several requests, and their joins, against 64
    bits on the GPU."""
    s, q = filled(len(new), g, group, first, new, "f16", 6)
    q *= 3
    got = s.attend(q, "f16")
    at = 0
    for r, (n, m) in enumerate(zip(first, new)):
        pages = s.table[r, :-(-(n + m) // 64)].long()
        x = s.data.view(s.pages, g, 2, 64, 128)[pages].double() * s.scales.view(s.pages, g, 2, 4)[pages].double().repeat_interleave(16, -1)[..., None]
        hide = torch.arange(n + m, device="cuda") > torch.arange(n, n + m, device="cuda")[:, None]
        for h in range(g * group):
            k, v = (x[:, h // group, c].reshape(-1, 128)[:n + m] for c in (0, 1))
            p = torch.softmax((q[at:at + m, h].double() @ k.T * 128 ** -0.5).masked_fill(hide, -math.inf), -1)
            want, mag = p @ v, p @ v.abs()
            tol = HALF["f16"] * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + (n + m) * 2.0 ** -25 * v.abs().max() + 2.0 ** -25
            assert ((got[at:at + m, h].double() - want).abs() <= tol).all(), (r, h)
        at += m
    assert s.status.tolist() == [0, 0]


def test_many_kv_heads_and_one_query_head_each():
    s, q = filled(2, 40, 1, [100, 5], [1, 40], "bf16", 7)
    got = s.attend(q, "bf16")
    torch.cuda.synchronize()
    compare(got, q, s, "bf16", [1, 40], 128 ** -0.5, 0)


def test_rope_at_positions_below_zero():
    """A position below 0 turns backwards and has no query temperature."""
    from jevstral_b200 import paged

    spec = paged.rope_spec("half", 128, 1e4, temperature_scale=0.1, temperature_context=4)
    x = torch.randn(3, 2, 128, device="cuda")
    y = torch.empty_like(x)
    pos = torch.tensor([-1, -100, 3], dtype=torch.int32, device="cuda")
    paged.rope(spec, "f32", pos.data_ptr(), 3, 128, paged.heads(x.data_ptr(), 2, 256, 128, y.data_ptr(), temperature=True))
    torch.cuda.synchronize()
    want = rope64(x.double().cpu().numpy(), pos.cpu().numpy(), spec)
    # two products of factors off by at most 2 steps of 2^-23 each, and their sum: 6 steps of 2^-23 at |a| + |b| < 10
    assert np.abs(y.double().cpu().numpy() - want).max() < 6 * 2.0 ** -23 * 10


def test_the_first_calls_of_a_process_can_be_captured():
    """plan, append and attention of both kinds captured in a fresh process before any of them has run."""
    import subprocess
    import sys

    code = """
import sys
sys.path[:0] = ['llm-shield_b200', 'tests', '.']
import torch
import test_gpu_paged as t
s = t.Server(2, 2, 4, 20, 60, 120, 8)
kv = torch.randn(61, 2, 2, 128, device='cuda')
q = torch.randn(61, 8, 128, device='cuda').half()
out = torch.zeros_like(q)
new = torch.tensor([60, 1], dtype=torch.int32, device='cuda')
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    s.p.plan(s.batch, s.lengths.data_ptr(), new.data_ptr(), s.free.data_ptr(), s.n_free.data_ptr(), s.n_free.data_ptr(), st)
    s.append(kv[:, 0], kv[:, 1], 'f32', stream=st)
    s.attend(q, 'f16', out=out, stream=st)
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
assert s.status.tolist() == [0, 0] and s.lengths.tolist() == [180, 3]
t.compare(out, q, s, 'f16', [60, 1], 128 ** -0.5, 0)
print('captured')
"""
    from conftest import REPO

    r = subprocess.run([sys.executable, "-c", code], cwd=str(REPO), capture_output=True, text=True, timeout=300)
    assert "captured" in r.stdout, (r.stdout[-1000:], r.stderr[-3000:])


def test_wrong_devices_and_pointers_are_refused_before_a_launch():
    s = Server(1, 1, 4, 2, 4, 4, 2)
    before = __import__("jevstral_b200").kernel_launches()
    host = torch.zeros(64)
    from jevstral_b200 import paged
    from jevstral_b200._lib import ArgumentError

    with pytest.raises(ArgumentError):
        paged.rope(paged.rope_spec("half", 64, 1e4), "f32", s.positions.data_ptr(), 1, 64,
                   paged.heads(host.data_ptr(), 1, 64, 64, host.data_ptr()))
    assert __import__("jevstral_b200").kernel_launches() == before
