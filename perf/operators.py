"""The operators of the paged 8-bit KV cache, in plain form and as the framework offers them.

A server that keeps many requests in one cache runs four of them for every step of the model:

  plan       block tables, slots, positions and row starts of a ragged batch, from the requests' lengths
  rope       rotary positions on queries and keys (adjacent or half-split pairs, part of the head, YaRN)
  append     the new tokens' keys and values into 8-bit pages, a scale per 16 tokens and head, with or without
             the rotation on the way; then the touched blocks read back as the values they stand for
  attention  grouped-query attention of the new tokens over the paged 8-bit cache, causal or in a sliding window

The cache: pages of 64 tokens; data int8 [pages][kv_heads][2 (K, V)][64][128]; scales fp32 [pages][kv_heads][2][4],
one per 16 tokens. A block's scale is the largest magnitude written to it / 127 and grows when a later token needs it;
the entries already there are then rounded again at the new scale.
"""
import math
import random
import sys

import torch

own = False

PAGE, BLOCK, DIM = 64, 16, 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _framework():
    if "llm-shield_b200" not in sys.path:
        sys.path.insert(0, "llm-shield_b200")
    from jevstral_b200 import paged

    return paged


# --------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one decode step of a small server: sixteen conversations, one new token each
        dict(name="plan-decode-16", op="plan", requests=16, len_lo=40, len_hi=2000, new_lo=1, new_hi=1, mix=1),
        # a large mixed step: idle requests, single tokens and prompt chunks in one batch
        dict(name="plan-mixed-2048", op="plan", requests=2048, len_lo=0, len_hi=4000, new_lo=0, new_hi=48, mix=2),
        # the queries and keys of a few tokens far into a context, the head layout of the 3B model
        dict(name="rope-7-far", op="rope", tokens=7, heads=32, kv_heads=8, head_dim=128, rotary=128, layout="interleaved",
             scaling="none", base=1e6, factor=1.0, orig=0, far=30000, type="f16"),
        # a whole prompt, half-split pairs on half of the head, YaRN by 16 over 16384 positions
        dict(name="rope-8191-yarn", op="rope", tokens=8191, heads=32, kv_heads=8, head_dim=128, rotary=64, layout="half",
             scaling="yarn", base=1e6, factor=16.0, orig=16384, far=250000, type="bf16"),
        # one new token of each of 64 conversations, straight from the fp32 projection, rotated on the way
        dict(name="append-decode-64", op="append", requests=64, heads=32, kv_heads=8, len_lo=100, len_hi=3000, new_lo=1,
             new_hi=1, mix=3, rope="interleaved", type="f32"),
        # ragged prompt chunks of seven requests, keys already rotated
        dict(name="append-chunks-7", op="append", requests=7, heads=16, kv_heads=8, len_lo=0, len_hi=3000, new_lo=300,
             new_hi=2000, mix=4, rope="", type="bf16"),
        # latency: a single conversation's next token
        dict(name="attention-decode-1", op="attention", requests=1, heads=32, kv_heads=8, len_lo=1025, len_hi=1025, new_lo=1,
             new_hi=1, window=0, mix=5, type="f16"),
        # throughput: 64 conversations of every length
        dict(name="attention-decode-64", op="attention", requests=64, heads=32, kv_heads=8, len_lo=300, len_hi=8000, new_lo=1,
             new_hi=1, window=0, mix=6, type="bf16"),
        # few conversations with long contexts
        dict(name="attention-decode-long", op="attention", requests=3, heads=32, kv_heads=8, len_lo=50000, len_hi=120000,
             new_lo=1, new_hi=1, window=0, mix=7, type="f16"),
        # drafted tokens verified: a few new tokens for each request
        dict(name="attention-verify-24", op="attention", requests=24, heads=32, kv_heads=8, len_lo=1000, len_hi=6000,
             new_lo=2, new_hi=6, window=0, mix=8, type="bf16"),
        # one prompt of 4095 tokens
        dict(name="attention-prompt-4095", op="attention", requests=1, heads=32, kv_heads=8, len_lo=4095, len_hi=4095,
             new_lo=4095, new_hi=4095, window=0, mix=9, type="f16"),
        # prompt chunks that continue longer contexts, in a sliding window
        dict(name="attention-chunks-window", op="attention", requests=5, heads=16, kv_heads=8, len_lo=4000, len_hi=16000,
             new_lo=100, new_hi=1500, window=4096, mix=10, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "append", "append", "attention", "attention", "attention"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 8])
    heads = min(heads, 32) // kv_heads * kv_heads
    mix = rng.randrange(1 << 30)
    if op == "plan":
        new = _log(rng, 1, 48)
        return dict(op=op, requests=_log(rng, 1, 1500), len_lo=rng.randrange(100), len_hi=_log(rng, 100, 4000),
                    new_lo=rng.choice([0, 1]), new_hi=new, mix=mix)
    if op == "rope":
        head_dim = rng.choice([64, 128, 128, 256])
        scaling = rng.choice(["none", "linear", "yarn"])
        return dict(op=op, tokens=_log(rng, 1, 4000), heads=heads, kv_heads=kv_heads, head_dim=head_dim if heads <= 16 else 128,
                    rotary=rng.choice([32, 48, 64]) if head_dim == 64 else rng.choice([32, 64, 96, 128]),
                    layout=rng.choice(["interleaved", "half"]), scaling=scaling, base=rng.choice([1e4, 5e5, 1e6]),
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 16.0]), orig=rng.choice([4096, 16384]),
                    far=_log(rng, 1000, 400000), type=rng.choice(["f32", "f16", "bf16"]))
    if op == "append":
        requests = _log(rng, 1, 200)
        new = _log(rng, 1, max(1, min(2000, 3000 // requests)))
        return dict(op=op, requests=requests, heads=heads, kv_heads=kv_heads, len_lo=rng.randrange(50),
                    len_hi=_log(rng, 50, 3000), new_lo=min(new, rng.choice([1, 1 + new // 2])), new_hi=new, mix=mix,
                    rope=rng.choice(["", "interleaved", "half"]), type=rng.choice(["f32", "f16", "bf16"]))
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    if kind == "decode":
        requests = _log(rng, 1, 64)
        hi = _log(rng, 30, 300000 // (requests + 4))
        return dict(op=op, requests=requests, heads=heads, kv_heads=kv_heads, len_lo=1 + rng.randrange(hi // 2 + 1), len_hi=hi,
                    new_lo=1, new_hi=1, window=rng.choice([0, 0, 1000]), mix=mix, type=rng.choice(["f16", "bf16"]))
    if kind == "verify":
        requests = _log(rng, 1, 32)
        return dict(op=op, requests=requests, heads=heads, kv_heads=kv_heads, len_lo=20, len_hi=_log(rng, 40, 6000), new_lo=1,
                    new_hi=rng.randrange(2, 20), window=0, mix=mix, type=rng.choice(["f16", "bf16"]))
    requests = rng.choice([1, 2, 3])
    new = _log(rng, 30, 2000 // requests)
    return dict(op=op, requests=requests, heads=heads, kv_heads=kv_heads, len_lo=new, len_hi=new + _log(rng, 1, 3000),
                new_lo=1 + new // 2, new_hi=new, window=rng.choice([0, 0, 777]), mix=mix, type=rng.choice(["f16", "bf16"]))


def _ragged(case):
    """(tokens in the cache after the step, new tokens among them) of each request: part of the case, not of the seed."""
    rng = random.Random(case["mix"])
    out = []
    for _ in range(case["requests"]):
        new = rng.randint(case["new_lo"], case["new_hi"])
        total = rng.randint(case["len_lo"], case["len_hi"])
        out.append((max(total, new) if case["op"] == "attention" else total + new, new))
    return out


def work(case):
    op = case["op"]
    if op == "plan":
        rag = _ragged(case)
        tokens, pages = sum(n for _, n in rag), sum(-(-t // PAGE) - -(-(t - n) // PAGE) for t, n in rag)
        # lengths in and out, new counts, starts; request, position and slot of a token; the new pages' ids in and out
        return {"bytes": len(rag) * 16 + tokens * 16 + pages * 8, "flops": 0}
    if op == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": n * case["head_dim"] * 2 * SIZE[case["type"]] + case["tokens"] * 4, "flops": n * case["rotary"] * 3}
    rag = _ragged(case)
    tokens, h, g = sum(n for _, n in rag), case["heads"], case["kv_heads"]
    if op == "append":
        kept = sum((t - n) % BLOCK for t, n in rag if n)
        touched = tokens + kept
        values = tokens * g * 2 * DIM
        io = tokens * h * DIM * (SIZE[case["type"]] + 2) if case["rope"] else 0
        # keys and values in, 8 bits out, the entries kept in a touched block in and out; the blocks read back as 16 bits
        return {"bytes": values * (SIZE[case["type"]] + 1) + kept * g * 2 * DIM * 2 + io + touched * g * 2 * DIM * 3,
                "flops": values * 3 + (tokens * (h + g) * DIM * 3 if case["rope"] else 0)}
    pairs = keys = 0
    for total, new in rag:
        first = total - new
        for p in range(first, total):
            pairs += min(p + 1, case["window"]) if case["window"] else p + 1
        keys += min(total, case["window"] + new - 1) if case["window"] else total
    return {"bytes": keys * g * 2 * (DIM + 4 / BLOCK) + tokens * h * DIM * 2 * SIZE[case["type"]], "flops": 4 * DIM * h * pairs}


# --------------------------------------------------------------------------------------------- inputs


def _frequencies(case):
    """Angles per position (radians), and the factor on cosine and sine, as the model's own YaRN rule has them."""
    rot, base = case["rotary"], case["base"]
    inv = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if case["scaling"] == "linear":
        return [f / case["factor"] for f in inv], 1.0
    if case["scaling"] == "yarn":
        corr = [rot * math.log(case["orig"] / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0)]
        low, high = max(0.0, math.floor(corr[0])), min(rot / 2 - 1.0, math.ceil(corr[1]))
        out = []
        for i, f in enumerate(inv):
            keep = 1.0 - min(max((i - low) / max(0.001, high - low), 0.0), 1.0)
            out.append(f / case["factor"] * (1 - keep) + f * keep)
        return out, 0.1 * math.log(case["factor"]) + 1.0
    return inv, 1.0


def _quantise(x):
    """[..., n * 16, 128] -> int8 of the same shape, fp32 scales [..., n]."""
    b = x.unflatten(-2, (-1, BLOCK))
    scale = b.abs().amax((-1, -2)) / 127
    q = torch.round(b * (127 / b.abs().amax((-1, -2), keepdim=True)))
    return q.to(torch.int8).flatten(-3, -2), scale


def _heads_like(gen, *shape):
    """Projections as a model makes them: unit variance, some channels several times larger than the rest."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    return x * (1 + 4 * (torch.arange(shape[-1], device="cuda") % 29 == 3))


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed * 7919 + 17)
    op, s = case["op"], {"case": case}
    if op == "rope":
        t, h, g, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        freqs, s["mscale"] = _frequencies(case)
        s["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
        start = int(torch.randint(0, case["far"], (1,), generator=gen, device="cuda"))
        s["positions"] = torch.arange(start, start + t, dtype=torch.int32, device="cuda")
        qk = _heads_like(gen, t, h + g, d).to(TYPES[case["type"]])  # one projection's output: queries, then keys
        s["q"], s["k"] = qk[:, :h], qk[:, h:]
        s["q_out"], s["k_out"] = (torch.empty(t, n, d, dtype=qk.dtype, device="cuda") for n in (h, g))
        if own:
            _own_rope(s, case, d)
        return s

    rag = _ragged(case)
    r, tokens = len(rag), sum(n for _, n in rag)
    total = torch.tensor([t for t, _ in rag], dtype=torch.int32, device="cuda")
    new = torch.tensor([n for _, n in rag], dtype=torch.int32, device="cuda")
    s["cached"], s["new"] = total - new, new
    have = [-(-(t - n) // PAGE) for t, n in rag]
    want = [-(-t // PAGE) for t, _ in rag]
    pages = sum(want) + 5
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    blocks = max(max(want), 1)
    col = torch.arange(blocks, device="cuda")
    first = torch.tensor([sum(have[:i]) for i in range(r)], device="cuda")
    inside = col < torch.tensor(have, device="cuda")[:, None]
    s["table"] = torch.where(inside, order[(first[:, None] + col).clamp(max=pages - 1)], -1).to(torch.int32)
    s["free"] = order[sum(have):].clone()
    s["n_free"] = torch.tensor([pages - sum(have)], dtype=torch.int32, device="cuda")
    s["n_free_out"] = torch.zeros_like(s["n_free"])
    room = tokens + 3 if op == "plan" else max(tokens, 1)
    s["max_new"], s["max_tokens"], s["pages"], s["blocks"] = max(1, *(n for _, n in rag)), max(room, 1), pages, blocks
    s["lengths"] = torch.full((r,), -1, dtype=torch.int32, device="cuda")
    s["starts"] = torch.full((r + 1,), -1, dtype=torch.int32, device="cuda")
    s["request_of"], s["positions"] = (torch.full((s["max_tokens"],), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    s["slots"] = torch.full((s["max_tokens"],), -1, dtype=torch.int64, device="cuda")
    s["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    group = case["heads"] // case["kv_heads"] if "heads" in case else 4
    if own:
        p = _framework()
        size = p.work_bytes(r, s["max_new"], s["max_tokens"], blocks, sum(t for t, _ in rag), group)
        s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        s["batch"] = p.batch(r, s["max_new"], s["max_tokens"], blocks, sum(t for t, _ in rag), group, pages,
                             *(s[n].data_ptr() for n in ("table", "lengths", "starts", "request_of", "positions", "slots",
                                                         "work", "status")))
    if op == "plan":
        return s

    # a server has planned the step before it runs the layers
    if own:
        _plan_own(s)
    else:
        _plan_plain(s)
    g = case["kv_heads"]
    content = _heads_like(gen, pages, g, 2, PAGE, DIM)
    s["data"], s["scales"] = _quantise(content)
    del content
    if op == "append":
        h = case["heads"]
        qkv = _heads_like(gen, tokens, h + 2 * g, DIM).to(TYPES[case["type"]])
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]
        s["q_out"] = torch.empty(tokens, h, DIM, dtype=torch.float16, device="cuda")
        if case["rope"]:
            rope = dict(rotary=DIM, layout=case["rope"], scaling="none", base=1e6, factor=1.0, orig=0)
            s["rope_case"] = rope
            freqs, s["mscale"] = _frequencies(rope)
            s["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
        # every slot of a block that the step writes to: the new tokens', and those kept in front of them
        want_read, start = [], 0
        for i, (t, n) in enumerate(rag):
            if n:
                at = torch.arange((t - n) // BLOCK * BLOCK, t, device="cuda")
                want_read.append(s["table"][i, at // PAGE].long() * PAGE + at % PAGE)
        s["read"] = torch.cat(want_read)
        s["k_read"], s["v_read"] = (torch.empty(len(s["read"]), g, DIM, dtype=torch.float16, device="cuda") for _ in range(2))
    else:
        h = case["heads"]
        s["q"] = (1.5 * torch.randn(tokens, h, DIM, generator=gen, device="cuda")).to(TYPES[case["type"]])
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["cache"] = p.cache(s["data"].data_ptr(), s["scales"].data_ptr(), pages, g)
        if op == "append":
            s["spec"] = _spec(s["rope_case"]) if case["rope"] else None
            s["k_heads"], s["v_heads"] = _heads(s["k"]), _heads(s["v"])
            s["q_heads"] = _heads(s["q"], s["q_out"]) if case["rope"] else None
        else:
            s["q_heads"] = _heads(s["q"], s["out"])
            s["ws_bytes"] = p.attention_bytes(s["batch"], g)
            s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------------------------------------- plain forms


def _plan_plain(s):
    cached, new, table = s["cached"].long(), s["new"].long(), s["table"]
    total = cached + new
    starts = torch.zeros(len(new) + 1, dtype=torch.int64, device="cuda")
    torch.cumsum(new, 0, out=starts[1:])
    have, want = (cached + PAGE - 1) // PAGE, (total + PAGE - 1) // PAGE
    before = torch.cumsum(want - have, 0) - (want - have)
    col = torch.arange(s["blocks"], device="cuda")
    fresh = (col >= have[:, None]) & (col < want[:, None])
    take = (s["n_free"].long() - 1 - (before[:, None] + col - have[:, None])).clamp(0, len(s["free"]) - 1)
    table.copy_(torch.where(fresh, s["free"][take], table))
    s["n_free_out"].copy_(s["n_free"] - (want - have).sum())
    t = torch.arange(s["max_tokens"], device="cuda")
    live = t < starts[-1]
    req = (torch.searchsorted(starts, t, right=True) - 1).clamp(0, len(new) - 1)
    pos = cached[req] + t - starts[req]
    slot = table[req, (pos // PAGE).clamp(0, s["blocks"] - 1)].long() * PAGE + pos % PAGE
    for name, value in (("request_of", req), ("positions", pos), ("slots", slot)):
        s[name].copy_(torch.where(live, value.to(s[name].dtype), s[name]))
    s["lengths"].copy_(total)
    s["starts"].copy_(starts)


def _rotate(x, positions, freqs, mscale, layout):
    """[tokens, heads, dim] in fp32, the first 2 * len(freqs) dimensions rotated; the angles in 64 bits."""
    angle = positions.double()[:, None] * freqs
    cos, sin = ((f(angle) * mscale).float()[:, None] for f in (torch.cos, torch.sin))
    x, n = x.float(), len(freqs)
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _append_plain(s):
    data, scales, slots = s["data"], s["scales"], s["slots"]
    cached, starts, req, pos = (s[n].long() for n in ("cached", "starts", "request_of", "positions"))
    block_of = lambda slot: slot // BLOCK  # noqa: E731  a pool-wide block number
    kv = torch.stack([s["k_rotated"] if "freqs" in s else s["k"].float(), s["v"].float()], 2)  # [tokens, g, 2, 128]
    units = -(-s["max_new"] // BLOCK) + 1
    unit = req * units + pos // BLOCK - cached[req] // BLOCK
    largest = torch.zeros(len(cached) * units, *kv.shape[1:3], device="cuda")
    largest.index_reduce_(0, unit, kv.abs().amax(-1), "amax")
    # the first block of a request may hold tokens of earlier steps
    old_scale = scales.flatten(0, 0).permute(0, 3, 1, 2).flatten(0, 1)  # [pages * 4, g, 2]
    first_block = block_of(slots[starts[:-1].clamp(max=len(slots) - 1)])
    kept = cached % BLOCK
    has_kept = ((kept > 0) & (s["new"] > 0))[:, None, None]
    before = torch.where(has_kept, old_scale[first_block], 0.0)
    scale = (largest / 127).unflatten(0, (len(cached), units))
    inverse = torch.where(largest > 0, 127 / largest, 0.0).unflatten(0, (len(cached), units))
    grown = before > scale[:, 0]
    scale[:, 0] = torch.where(grown, before, scale[:, 0])
    inverse[:, 0] = torch.where(grown, 1 / before, inverse[:, 0])
    of_token = scale.flatten(0, 1)[unit]
    q = torch.round(kv * inverse.flatten(0, 1)[unit][..., None]).clamp(-127, 127).to(torch.int8)
    # entries kept in a request's first block, at its new scale; rows that there are none of write their first token again
    row = torch.arange(BLOCK - 1, device="cuda")
    old_slot = first_block[:, None] * BLOCK + row
    ratio = torch.where(has_kept, before / scale[:, 0], 0.0)
    head_token = starts[:-1].clamp(max=len(slots) - 1)
    valid = (row < kept[:, None]) & (s["new"] > 0)[:, None]
    target = torch.where(valid, old_slot, slots[head_token][:, None])
    old_q = data[old_slot // PAGE, :, :, old_slot % PAGE].float()  # [r, 15, g, 2, 128]
    again = torch.round(old_q * ratio[:, None, :, :, None]).to(torch.int8)
    again = torch.where(valid[:, :, None, None, None], again, q[head_token][:, None])
    data[slots // PAGE, :, :, slots % PAGE] = q
    data[target // PAGE, :, :, target % PAGE] = again
    scales[slots // PAGE, :, :, slots % PAGE // BLOCK] = of_token


def _read_plain(s):
    page, row = s["read"] // PAGE, s["read"] % PAGE
    x = s["data"][page, :, :, row].float() * s["scales"][page, :, :, row // BLOCK][..., None]
    return x[:, :, 0].half(), x[:, :, 1].half()


def _attention_plain(s):
    case, table = s["case"], s["table"].long()
    g, h = case["kv_heads"], case["heads"]
    span = s["blocks"] * PAGE
    pages = table.clamp(min=0)
    x = s["data"][pages].float()  # [r, blocks, g, 2, 64, 128]
    x = x.unflatten(-2, (PAGE // BLOCK, BLOCK)) * s["scales"][pages][..., None, None]
    x = x.permute(3, 0, 2, 1, 4, 5, 6).reshape(2, len(table), g, span, DIM)
    k, v = x[0], x[1]
    # the new tokens, padded to the longest request's
    starts, lengths, new = s["starts"].long(), s["lengths"].long(), s["new"].long()
    i = torch.arange(s["max_new"], device="cuda")
    token = (starts[:-1, None] + i).clamp(max=len(s["q"]) - 1)
    q = s["q"][token].float().unflatten(2, (g, h // g)).permute(0, 2, 1, 3, 4)  # [r, g, n, group, 128]
    score = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (len(i), h // g)) / math.sqrt(DIM)
    at = (lengths - new)[:, None] + i
    key = torch.arange(span, device="cuda")
    sees = key <= at[..., None]
    if case["window"]:
        sees = sees & (key > at[..., None] - case["window"])
    score.masked_fill_(~sees[:, None, :, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    weight = torch.exp_(score)
    out = torch.matmul((weight / weight.sum(-1, keepdim=True)).flatten(2, 3), v).unflatten(2, (len(i), h // g))
    req = s["request_of"].long()
    t = torch.arange(len(s["q"]), device="cuda")
    return out.permute(0, 2, 1, 3, 4)[req[:len(t)], t - starts[req[:len(t)]]].flatten(1, 2).to(s["q"].dtype)


# --------------------------------------------------------------------------------------------- the framework's


def _spec(c):
    return _framework().rope_spec(c["layout"], c["rotary"], c["base"], scaling=c["scaling"], factor=c["factor"],
                                  original_context=c["orig"])


def _heads(x, out=None):
    """[tokens, heads, dim], the last dimension contiguous."""
    if out is None:
        return _framework().heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))
    return _framework().heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1))


def _own_rope(s, case, d):
    s["spec"] = _spec(case)
    s["q_heads"], s["k_heads"] = _heads(s["q"], s["q_out"]), _heads(s["k"], s["k_out"])


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _plan_own(s):
    _framework().plan(s["batch"], s["cached"].data_ptr(), s["new"].data_ptr(), s["free"].data_ptr(), s["n_free"].data_ptr(),
                      s["n_free_out"].data_ptr(), stream=_stream())


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "plan":
        if own:
            _plan_own(s)
        else:
            _plan_plain(s)
        return {n: s[n] for n in ("lengths", "starts", "request_of", "positions", "slots", "table", "n_free_out")}
    if op == "rope":
        if own:
            _framework().rope(s["spec"], case["type"], s["positions"].data_ptr(), case["tokens"], case["head_dim"],
                              s["q_heads"], s["k_heads"], stream=_stream())
            return s["q_out"], s["k_out"]
        turn = lambda x: _rotate(x, s["positions"], s["freqs"], s["mscale"], case["layout"]).to(x.dtype)  # noqa: E731
        return turn(s["q"]), turn(s["k"])
    if op == "append":
        if own:
            p = _framework()
            p.kv8_append(s["cache"], s["batch"], case["type"], s["k_heads"], s["v_heads"], rope=s["spec"], q=s["q_heads"],
                         out_dtype="f16", stream=_stream())
            p.kv8_read(s["cache"], s["read"].data_ptr(), len(s["read"]), "f16", s["k_read"].data_ptr(), s["v_read"].data_ptr(),
                       s["k_read"].stride(0), s["status"].data_ptr(), stream=_stream())
            read = s["k_read"], s["v_read"]
        else:
            if case["rope"]:
                s["k_rotated"] = _rotate(s["k"], s["positions"], s["freqs"], s["mscale"], case["rope"])
                s["q_out"] = _rotate(s["q"], s["positions"], s["freqs"], s["mscale"], case["rope"]).half()
            _append_plain(s)
            read = _read_plain(s)
        return (*read, s["q_out"]) if case["rope"] else read
    if own:
        _framework().kv8_attention(s["cache"], s["batch"], case["type"], s["q_heads"], 1 / math.sqrt(DIM), case["window"],
                                   s["ws"].data_ptr(), s["ws_bytes"], stream=_stream())
        return s["out"]
    return _attention_plain(s)


# --------------------------------------------------------------------------------------------- in 64 bits


def _turned(x, positions, freqs, mscale, layout):
    """The same rotation as a product of complex numbers."""
    n = len(freqs)
    x = x.double().cpu()
    z = mscale * torch.polar(torch.ones((), dtype=torch.float64), positions.double().cpu()[:, None] * freqs.cpu())[:, None]
    out = x.clone()
    first, second = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    w = torch.complex(x[..., first], x[..., second]) * z
    out[..., first], out[..., second] = w.real, w.imag
    return out


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    s = prepare(case, seed)
    if op == "rope":
        return tuple(_turned(s[n], s["positions"], s["freqs"], s["mscale"], case["layout"]) for n in ("q", "k"))
    rag = _ragged(case)
    if op == "append":
        k, v = s["k"].double(), s["v"].double()
        if case["rope"]:
            k = _turned(s["k"], s["positions"], s["freqs"], s["mscale"], case["rope"]).cuda()
        read, at = [[], []], 0
        for i, (total, new) in enumerate(rag):
            for b in range((total - new) // BLOCK, -(-total // BLOCK) if new else 0):
                page, rows = int(s["table"][i, b * BLOCK // PAGE]), b * BLOCK % PAGE
                lo, hi = max(b * BLOCK, total - new), min((b + 1) * BLOCK, total)
                for out, kind, fresh in zip(read, (0, 1), (k, v)):
                    x = fresh[at + lo - (total - new):at + hi - (total - new)]  # [n, g, 128]
                    scale = x.abs().amax((0, 2)) / 127
                    if lo > b * BLOCK:
                        had = s["scales"][page, :, kind, rows // BLOCK].double()
                        scale = torch.maximum(scale, had)
                        old = s["data"][page, :, kind, rows:rows + lo - b * BLOCK].double().transpose(0, 1)
                        out.append(torch.round(old * (had / scale)[:, None]) * scale[:, None])
                    out.append(torch.round(x / scale[:, None]) * scale[:, None])
            at += new
        read = [torch.cat(x) for x in read]
        return (*read, _turned(s["q"], s["positions"], s["freqs"], s["mscale"], case["rope"])) if case["rope"] else tuple(read)
    g, per = case["kv_heads"], case["heads"] // case["kv_heads"]
    outs = []
    at = 0
    for i, (total, new) in enumerate(rag):
        pages = s["table"][i, :-(-total // PAGE)].long()
        out = torch.empty(new, case["heads"], DIM, dtype=torch.float64, device="cuda")
        for j in range(g):
            x = s["data"][pages, j].double() * s["scales"][pages, j].double().repeat_interleave(BLOCK, -1)[..., None]
            k, v = (x[:, n].reshape(-1, DIM)[:total] for n in (0, 1))
            for lo in range(0, new, 512):
                hi = min(new, lo + 512)
                p = torch.arange(total - new + lo, total - new + hi, device="cuda")[:, None]
                key = torch.arange(total, device="cuda")
                hide = (key > p) | ((key <= p - case["window"]) if case["window"] else False)
                for c in range(j * per, (j + 1) * per):
                    logits = (s["q"][at + lo:at + hi, c].double() @ k.T) * DIM ** -0.5
                    out[lo:hi, c] = torch.softmax(logits.masked_fill(hide, -math.inf), -1) @ v
        outs.append(out)
        at += new
    return torch.cat(outs)
