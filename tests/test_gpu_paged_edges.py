"""The paged-batch operators on the GPU where a result could depend on what it must not: the scales of blocks
without values, the bounds of the batch, the alignment of an operand; and what is recorded when a result does not
fit its type.

Tolerance of the attention (`bounded`). A weight w_j = 2^(e_j - M), e_j = s_j + log2 vs_j, is rounded to fp16: by
2^-11 of itself, or by 2^-25 where it is below 2^-14. The first adds up to 2^-11 sum p |v|. The second adds up to
n 2^-25 127 / L with L = sum_j w_j / vs_j; since M is at most the row's largest e, that one's weight w_k is at least
1, and 1 / L <= w_k / L = p_k vs_k, the largest of all p_j vs_j. fp32 arithmetic is taken as 2^-13 of sum p |v|
(exponents below 2^7 carry an error of 2^-17 or less into a weight); the output is rounded to its type."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_paged import HALF, NUMERIC, RANGE, TYPE, Server, filled  # noqa: E402

ZERO_SCALE = 2.0 ** -60  # what a block of zeros counts as


def bounded(got, q, s, dtype, new, window=0, scale=128 ** -0.5):
    """Every row of `got` against 64 bits; returns the largest error as a share of its bound."""
    lengths, t, worst = s.lengths.tolist(), 0, 0.0
    for r, n in enumerate(new):
        if n == 0:
            continue
        kv = s.stored(r, lengths[r]).cuda()
        pages = s.table[r, :-(-lengths[r] // 64)].long()
        vs = s.scales.view(s.pages, s.scale_stride)[pages, :s.g * 8].view(-1, s.g, 2, 4)[:, :, 1].double()
        vs = vs.permute(0, 2, 1).reshape(-1, s.g).repeat_interleave(16, 0)[:lengths[r]]
        vs = torch.where(vs > 0, vs, ZERO_SCALE)
        key = torch.arange(lengths[r], device="cuda")
        at = torch.arange(lengths[r] - n, lengths[r], device="cuda")[:, None]
        hide = key > at
        if window:
            hide |= key <= at - window
        seen = (~hide).sum(-1)[:, None].double()
        for h in range(s.g * s.group):
            k, v = kv[0, :, h // s.group], kv[1, :, h // s.group]
            p = torch.softmax((q[t:t + n, h].double() @ k.T * scale).masked_fill(hide, -math.inf), -1)
            want, mag = p @ v, p @ v.abs()
            low = seen * 2.0 ** -25 * 127 * (p * vs[:, h // s.group]).amax(-1, keepdim=True)
            tol = HALF[dtype] * want.abs() + (2.0 ** -11 + 2.0 ** -13) * mag + low + (2.0 ** -25 if dtype == "f16" else 1e-38)
            err = (got[t:t + n, h].double() - want).abs()
            assert (err <= tol).all(), (r, h, float((err / tol).max()))
            worst = max(worst, float((err / tol).max()))
        t += n
    return worst


# (lengths before, new): one chunk, several chunks and their join, rows for the tensor cores, parts of a long
# context and their join, both kinds in one call
ROWS = [([40], [1]), ([700], [2]), ([90], [70]), ([3000], [40]), ([500, 1100], [1, 50])]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("amp", [0.1, 1e-3, 1e-4, 1e-6])
@pytest.mark.parametrize("first,new", ROWS)
def test_zero_values_among_small_ones(dtype, amp, first, new):
    """One block of 16 values that are all zero, its keys some 8 log2 units above the others."""
    g, group = 2, 4
    requests, most = len(first), max(max(first), max(new))
    blocks = -(-max(a + b for a, b in zip(first, new)) // 64)
    s = Server(requests, g, group, requests * blocks, most, max(sum(first), sum(new)), blocks, seed=5)
    gen = torch.Generator("cuda").manual_seed(11)
    u = 128 ** -0.5 * torch.sign(torch.randn(128, generator=gen, device="cuda"))
    for step in (first, new):
        s.plan(step)
        kv = torch.randn(sum(step), 2, g, 128, generator=gen, device="cuda")
        kv[:, 1] *= amp
        if step is first:
            at = 0
            for n in first:
                kv[at + 16:at + 32, 1] = 0
                kv[at + 16:at + 32, 0] += 8 * u  # q . k is 64 more, 8.2 in log2 units after the scale
                at += n
        s.append(kv[:, 0], kv[:, 1], "f32")
    q = (torch.randn(sum(new), g * group, 128, generator=gen, device="cuda") + 8 * u).to(TYPE[dtype])
    got = s.attend(q, dtype)
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    bounded(got, q, s, dtype, new)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("first,new,window", [([416], [5], 32), ([304], [200], 32), ([1504], [60], 0), ([704, 96], [1, 33], 20)])
def test_weights_carry_the_scales_of_their_blocks(dtype, first, new, window):
    """Values from 1e-6 to 1e4 by block, some blocks zero; in a window a row may see zeros and tiny values alone."""
    g, group = 2, 4
    requests, most = len(first), max(max(first), max(new))
    blocks = -(-max(a + b for a, b in zip(first, new)) // 64)
    s = Server(requests, g, group, requests * blocks, most, max(sum(first), sum(new)), blocks, seed=6)
    gen = torch.Generator("cuda").manual_seed(13)
    for step in (first, new):
        s.plan(step)
        kv = torch.randn(sum(step), 2, g, 128, generator=gen, device="cuda")
        mag = torch.tensor([1e-6, 0, 1e4, 1e-6, 0, 1e-3, 0, 1], device="cuda").repeat_interleave(16)
        kv[:, 1] *= mag.repeat(-(-sum(step) // 128))[:sum(step), None, None]
        s.append(kv[:, 0], kv[:, 1], "f32")
    q = (2 * torch.randn(sum(new), g * group, 128, generator=gen, device="cuda")).to(TYPE[dtype])
    got = s.attend(q, dtype, window=window)
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    bounded(got, q, s, dtype, new, window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("old,new,bounds", [
    (300, 1, [(301, 6), (1, 6), (2000, 40), (1, 600), (2000, 600), (5, 513)]), (1500, 2, [(1502, 24), (2, 24), (2, 600), (3000, 513)]),
    (2900, 5, [(2905, 46), (5, 46), (2905, 2000)]), (1300, 40, [(1340, 21), (40, 600)]),
    (33000, 1, [(33001, 516), (1, 516), (1, 517), (40000, 3000)])])
def test_a_request_s_bits_do_not_depend_on_the_batch_s_bounds(dtype, old, new, bounds):
    """One request over the same cache, under other max_new and max_blocks."""
    g, group, outs, data = 4, 4, [], None
    gen = torch.Generator("cuda").manual_seed(old)
    kv = torch.randn(old + new, 2, g, 128, generator=gen, device="cuda")
    q = torch.randn(new, g * group, 128, generator=gen, device="cuda").to(TYPE[dtype])
    held, pages = -(-old // 64), -(-(old + new) // 64)
    for max_new, max_blocks in bounds:
        s = Server(2, g, group, pages, max_new, max_new, max_blocks)
        if data is None:  # the first one can take all tokens at once
            s.plan([old + new, 0])
            s.append(kv[:, 0], kv[:, 1], "f32")
            data, scales, table = s.data.clone(), s.scales.clone(), s.table[0, :pages].clone()
        s.data.copy_(data)
        s.scales.copy_(scales)
        s.table[0, :held] = table[:held]
        s.free[:pages - held] = table[held:].flip(0)
        s.n_free.fill_(pages - held)
        s.lengths.copy_(torch.tensor([old, 0], dtype=torch.int32))
        s.plan([new, 0])
        outs.append(s.attend(q, dtype))
        torch.cuda.synchronize()
        assert s.status.tolist() == [0, 0] and s.lengths.tolist() == [old + new, 0]
    for got in outs[1:]:
        assert torch.equal(got.view(torch.int16), outs[0].view(torch.int16))


@pytest.mark.parametrize("first,new", ROWS)
def test_an_output_outside_fp16_is_recorded(first, new):
    """Values of 1e5 as fp16 outputs: infinities, and JV_ERR_NUMERIC; as bf16 outputs neither."""
    s, _ = filled(len(new), 2, 4, first, new, "f16", 7)
    s.scales *= 1e5  # keys too: a row picks one of them
    q = 1e-4 * torch.randn(sum(new), 8, 128, device="cuda")
    got = s.attend(q.bfloat16(), "bf16")
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0] and torch.isfinite(got).all()
    assert got.abs().max() > 65520
    got = s.attend(q.half(), "f16")
    torch.cuda.synchronize()
    assert not torch.isfinite(got).all() and s.status.tolist() == [NUMERIC, 105]


@pytest.mark.parametrize("new", [[1, 1], [40, 1], [70, 90]])
def test_keys_of_a_bad_page_have_no_weight(new):
    """A request whose first page is not in the cache: the result of its other keys."""
    s, q = filled(2, 1, 4, [200, 100], new, "f16", 8)
    torch.cuda.synchronize()
    assert s.status.tolist() == [0, 0]
    s.table[0, 0] = s.pages
    got = s.attend(q, "f16")
    torch.cuda.synchronize()
    assert s.status.tolist() == [RANGE, 106]
    s.table[0, 0] = 0
    kv = s.stored(0, 200 + new[0])[:, 64:, 0]
    for i in range(new[0]):
        x = kv[:, :200 + i + 1 - 64]
        p = torch.softmax(q[i].double().cpu() @ x[0].T * 128 ** -0.5, -1)
        mag = p @ x[1].abs()
        tol = HALF["f16"] * (p @ x[1]).abs() + (2.0 ** -11 + 2.0 ** -13) * mag + 300 * 2.0 ** -25 * x[1].abs().max() + 2.0 ** -25
        assert ((got[i].double().cpu() - p @ x[1]).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout,rot,dim", [("interleaved", 128, 128), ("half", 128, 128), ("half", 64, 128), ("interleaved", 96, 128)])
def test_rope_s_bits_do_not_depend_on_the_alignment(dtype, layout, rot, dim):
    from jevstral_b200 import paged

    spec = paged.rope_spec(layout, rot, 1e4, temperature_scale=0.1, temperature_context=64)
    x = torch.randn(300, 5, dim, generator=torch.Generator("cuda").manual_seed(rot), device="cuda").to(TYPE[dtype])
    pos = torch.arange(1000, 1300, dtype=torch.int32, device="cuda")
    outs = []
    for offset in (0, 1):
        src = torch.zeros(x.numel() + 8, device="cuda", dtype=x.dtype)[offset:offset + x.numel()].view_as(x)
        src.copy_(x)
        out = torch.empty_like(x)
        paged.rope(spec, dtype, pos.data_ptr(), 300, dim, paged.heads(src.data_ptr(), 5, 5 * dim, dim, out.data_ptr(), temperature=True))
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(*outs)


def test_rope_of_the_most_tokens():
    """2^31 - 1 tokens of one pair each, in place: the first, the last and some between (17 GB)."""
    from jevstral_b200 import paged

    n = 2 ** 31 - 1
    spec = paged.rope_spec("interleaved", 2, 1e4)
    x = torch.ones(n, 2, dtype=torch.float16, device="cuda")
    pos = torch.full((n,), 7, dtype=torch.int32, device="cuda")
    at = torch.tensor([0, 1, 12345678, 2 ** 30 + 3, n - 8, n - 2, n - 1], device="cuda")
    pos[at] = torch.arange(1, len(at) + 1, dtype=torch.int32, device="cuda")
    paged.rope(spec, "f16", pos.data_ptr(), n, 2, paged.heads(x.data_ptr(), 1, 2, 2, x.data_ptr()))
    torch.cuda.synchronize()
    angle = pos[at].double()
    want = torch.stack([angle.cos() - angle.sin(), angle.cos() + angle.sin()], 1)
    # cos and sin to 3 units of 2^-23, their sum of at most 1.42; then half a step of fp16
    assert ((x[at].double() - want).abs() <= HALF["f16"] * want.abs() + 8 * 2.0 ** -23).all()
