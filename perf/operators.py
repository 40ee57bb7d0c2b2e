"""Serving from a cache held in 4 bits, operator by operator: the keys and values of new tokens go into the pages (bias, rotation and
rounding to 4 bits in one), attention reads them there, for single tokens and for portions of prompts, and the next tokens are
drawn from the logits with temperature, top-k, top-p and min-p.

The 4-bit form of a row of ``d`` numbers (one token's key or value of one head): groups of 32 neighbouring numbers, the last one
padded, each with a scale and a centre in half precision, and a code of 4 bits a number: x = centre + (code - 8) * scale, where
scale = (largest - smallest) / 15 and centre = smallest + 8 scale, both rounded to half precision before the codes are chosen.
Numbers beyond +-61440 are stored as that; a group that holds a NaN reads as NaN.

The cache is uint8 [pages, kv heads, page size / 16, 640 G] with G = ceil(d / 32) groups: a tile of 16 tokens holds their key codes
(16 G bytes a token), their value codes, the keys' (scale, centre) pairs (4 G bytes a token) and the values'.  A row's codes lie in
the order in which the tensor cores take them: byte b of word (t, g) of a key row, laid out [4, G, 4], holds numbers 32 g + 8 t +
2 b (low half) and the next; byte b of piece (p, g) of a value row, [8, G, 2], numbers 32 g + 4 p + 2 b and the next.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda:0"
LARGEST = 61440.0
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases --------------------------------------------------------------------------------------------------------
def _store(tokens, heads, kv, d, dtype="bfloat16", rot=None, pairs="halves", bias=True, page=16):
    return {"kind": "store", "tokens": tokens, "heads": heads, "kv": kv, "d": d, "dtype": dtype, "rot": d if rot is None else rot,
            "pairs": pairs, "bias": bias, "page": page}


def _attend(requests, context, heads, kv, d, new=1, dtype="bfloat16", window=0, keep=0, page=16, ragged=True):
    """``context``: keys of the longest request, its new tokens among them (``ragged``: the others are spread down to an eighth of it);
    ``new``: tokens that a request brings, 1 in decoding; above 1 every third request brings one token all the same."""
    return {"kind": "attend", "requests": requests, "context": context, "heads": heads, "kv": kv, "d": d, "new": new, "dtype": dtype,
            "window": window, "keep": keep, "page": page, "ragged": ragged}


def listed():
    return [
        # one token of one conversation on the 7B shape: all latency
        dict(_store(1, 28, 4, 128), name="store-one"),
        # a prompt of the benchmark's length on the 14B shape in one step
        dict(_store(2048, 40, 8, 128), name="store-prompt-2k"),
        # 32-bit activations, half of each head rotated in neighbouring pairs, an odd number of tokens
        dict(_store(509, 14, 2, 64, dtype="float32", rot=32, pairs="interleaved", bias=False), name="store-fp32-part"),
        # one short question to a small model
        dict(_attend(1, 61, 12, 2, 128, ragged=False), name="decode-short-b1"),
        # the headline workload of the benchmark: batch 8 after 2,048-token prompts
        dict(_attend(8, 2049, 28, 4, 128, ragged=False), name="decode-b8-2k"),
        # a loaded server: 64 conversations of different length
        dict(_attend(64, 8191, 28, 4, 128), name="decode-b64-8k"),
        # long documents on the 14B shape, up to its 32,768 positions: the largest
        dict(_attend(16, 32768, 40, 8, 128), name="decode-b16-32k"),
        # the path with 32-bit activations, in which results are checked
        dict(_attend(4, 1021, 12, 2, 128, dtype="float32"), name="decode-fp32"),
        # a mixed step: portions of prompts beside decoded tokens, under a window that keeps the first tokens
        dict(_attend(12, 4093, 28, 4, 128, new=171, window=1024, keep=16), name="mixed-window"),
        # the benchmark's prompt in one step
        dict(_attend(1, 2048, 28, 4, 128, new=2048, ragged=False), name="prompt-2k"),
        # the next token of one conversation, 7B vocabulary
        {"kind": "sample", "rows": 1, "vocab": 152064, "name": "sample-b1"},
        # the next tokens of 64 conversations, each with settings of its own
        {"kind": "sample", "rows": 64, "vocab": 152064, "name": "sample-b64"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, uniform over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "decode", "portions", "portions", "sample"])
    heads, kv, d = rng.choice([(28, 4, 128), (12, 2, 128), (40, 8, 128), (14, 2, 64), (16, 16, 80), (32, 2, 64)])
    page = rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if kind == "store":
        return _store(_spread(rng, 1, 4096), heads, kv, d, dtype, rng.choice([d, d, d // 2, 0]), rng.choice(["halves", "interleaved"]),
                      rng.random() < 0.5, page)
    if kind == "sample":
        return {"kind": "sample", "rows": _spread(rng, 1, 64), "vocab": rng.choice([32000, 32003, 151936, 152064])}
    window, keep = rng.choice([(0, 0), (0, 0), (rng.randint(100, 2000), 0), (rng.randint(100, 2000), rng.randint(1, 64))])
    if kind == "decode":
        requests = _spread(rng, 1, 64)
        return _attend(requests, _spread(rng, 16, min(32768, 196608 // requests)), heads, kv, d, 1, dtype, window, keep, page, rng.random() < 0.7)
    requests = _spread(rng, 1, 8)
    new = _spread(rng, 2, 512 // requests)
    return _attend(requests, new + _spread(rng, 1, 2048), heads, kv, d, new, dtype, window, keep, page, rng.random() < 0.7)


# ---- what a case means ------------------------------------------------------------------------------------------------
def _groups(d):
    return -(-d // 32)


def _lengths(case):
    """(new tokens, tokens cached before them) of every request."""
    n, longest, new = case["requests"], case["context"], case["new"]
    got = []
    for r in range(n):
        total = longest if not case["ragged"] or n == 1 else longest - (longest - longest // 8) * ((r * 7) % n) // n
        take = 1 if new > 1 and r % 3 == 2 else min(new, total)
        got.append((take, max(0, total - take)))
    return got


def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 32), "flops": 4 * case["rows"] * case["vocab"]}
    size = 2 if case["dtype"] == "bfloat16" else 4
    heads, kv, d = case["heads"], case["kv"], case["d"]
    row = 40 * _groups(d)                                   # key and value of a token and head, with scales and centres
    if case["kind"] == "store":
        tokens = case["tokens"]
        return {"bytes": tokens * ((heads + 2 * kv) * d * 4 + heads * d * size + 2 * kv * row + kv * 2 * d * 2), "flops": tokens * (heads + 2 * kv) * d * 6}
    moved, pairs = 0, 0
    for new, start in _lengths(case):
        first = max(0, start - case["window"] + 1) if case["window"] else 0
        moved += (start + new - first + min(case["keep"], first)) * kv * row + 2 * new * heads * d * size
        for p in range(start, start + new):
            lo = max(0, p - case["window"] + 1) if case["window"] else 0
            pairs += p + 1 - lo + min(case["keep"], lo)
    return {"bytes": moved, "flops": 4 * pairs * heads * d}


# ---- what a program has in hand -----------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"store": _prepare_store, "attend": _prepare_attend, "sample": _prepare_sample}[case["kind"]](case, gen)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _prepare_store(case, gen):
    tokens, heads, kv, d, page = case["tokens"], case["heads"], case["kv"], case["d"], case["page"]
    pages = -(-tokens // page) + 3
    # a few channels of the keys stand far out, as they do in trained models
    out = torch.where(torch.rand(kv, d, generator=gen, device=DEV) < 0.05, 6.0, 1.0)
    lift = torch.cat([torch.ones(heads * d, device=DEV), out.flatten(), torch.ones(kv * d, device=DEV)])
    projected = _normal(gen, tokens, (heads + 2 * kv) * d) * lift
    order = torch.randperm(pages, generator=gen, device=DEV)
    at = torch.arange(tokens, device=DEV)
    start = 0 if tokens > 1 else 4096
    inv_freq = 1e6 ** (-torch.arange(max(case["rot"] // 2, 1), dtype=torch.float64) * 2 / max(case["rot"], 1))
    return SimpleNamespace(
        case=case, projected=projected, bias=_normal(gen, (heads + 2 * kv) * d) if case["bias"] else None,
        positions=(start + at).to(torch.int32), inv_freq=inv_freq.to(torch.float32).to(DEV) if case["rot"] else None,
        slots=(order[at // page] * page + at % page).to(torch.int32),
        cache=torch.zeros((pages, kv, page // 16, 640 * _groups(d)), dtype=torch.uint8, device=DEV))


def _prepare_attend(case, gen):
    heads, kv, d, page, n = case["heads"], case["kv"], case["d"], case["page"], _groups(case["d"])
    lengths = _lengths(case)
    need = [-(-(new + start) // page) for new, start in lengths]
    pages, width = sum(need) + 3, max(need)
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    counts = torch.tensor(need, device=DEV)
    first = torch.cumsum(counts, 0) - counts
    column = torch.arange(width, device=DEV)
    held = column < counts[:, None]
    table = torch.where(held, order[torch.where(held, first[:, None] + column, 0)], -1).to(torch.int32)
    # codes as numbers near a normal distribution have them; memory that no token was written to is all ones (NaN)
    codes = (_normal(gen, pages, kv, page // 16, 512 * n, 2) * 2.9 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    pairs = torch.stack([torch.rand(pages, kv, page // 16, 32 * n, generator=gen, device=DEV) * 0.25 + 0.15,
                         _normal(gen, pages, kv, page // 16, 32 * n) * 0.1], -1).to(torch.float16)
    cache = torch.cat([codes[..., 0] | (codes[..., 1] << 4), pairs.view(torch.uint8).flatten(-2)], -1).contiguous()
    rows = cache.view(pages, kv, page // 16, -1)
    ends = torch.zeros(pages, dtype=torch.long, device=DEV)
    total = torch.tensor([new + start for new, start in lengths], device=DEV)
    filled = (total[:, None] - column * page).clamp(0, page)
    ends[table[held].long()] = filled[held]
    empty = torch.arange(page, device=DEV) >= ends[:, None]                              # [pages, page]
    empty = empty.view(pages, 1, page // 16, 16).expand(-1, kv, -1, -1)
    for at, size in ((0, 16 * n), (256 * n, 16 * n), (512 * n, 4 * n), (576 * n, 4 * n)):
        rows[..., at:at + 16 * size].unflatten(-1, (16, size)).masked_fill_(empty[..., None], 255)
    new = torch.tensor([new for new, _ in lengths])
    cu_q = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(new, 0)])
    starts = torch.tensor([start for _, start in lengths])
    queries = (_normal(gen, int(cu_q[-1]), heads * d) * 2.0).to(TYPES[case["dtype"]])
    step = SimpleNamespace(
        cu_q=cu_q.to(torch.int32).to(DEV), q_start=starts.to(torch.int32).to(DEV), max_q_len=int(new.max()),
        max_ctx_len=max(a + b for a, b in lengths), host_lengths=[a for a, _ in lengths], host_starts=[b for _, b in lengths],
        token_request=torch.repeat_interleave(torch.arange(len(lengths)), new).to(torch.int32).to(DEV))
    return SimpleNamespace(case=case, queries=queries, cache=cache, table=table, step=step, scale=d ** -0.5)


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    uniform = torch.rand(rows, generator=gen, device=DEV)
    # sharp and flat rows: logits of a standard deviation from 0.5 to 4, a few dozen tokens above the rest
    logits = _normal(gen, rows, vocab) * (0.5 + 3.5 * torch.rand(rows, 1, generator=gen, device=DEV))
    logits += torch.where(torch.rand(rows, vocab, generator=gen, device=DEV) < 32 / vocab, 6.0, 0.0)
    at = torch.arange(rows, device=DEV)
    return SimpleNamespace(
        case=case, logits=logits, uniform=uniform,
        # what requests ask for: mostly a temperature and top-p, some with top-k or min-p too, some greedy
        temperature=torch.where(at % 8 == 7, 0.0, 0.6 + 0.1 * (at % 6)).to(torch.float32),
        top_k=torch.where(at % 3 == 1, 50, 0).to(torch.int32),
        top_p=torch.where(at % 5 == 4, 1.0, 0.8 + 0.05 * (at % 4)).to(torch.float32),
        min_p=torch.where(at % 4 == 2, 0.05, 0.0).to(torch.float32))


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"store": _own_store, "attend": _own_attend, "sample": _own_sample}[state.case["kind"]](state)
    return {"store": _plain_store, "attend": _plain_attend, "sample": _plain_sample}[state.case["kind"]](state)


def _own_store(s):
    from flexengine_b200 import ops
    c = s.case
    queries = ops.qkv_rope_kv4(s.projected, s.bias, s.positions, s.inv_freq, c["rot"], s.slots, s.cache, c["heads"], c["kv"], c["d"],
                               c["page"], pairs=c["pairs"], out_dtype=TYPES[c["dtype"]])
    keys, values = ops.kv4_rows(s.cache, s.slots, c["kv"], c["d"], c["page"], torch.bfloat16)
    return {"queries": queries, "keys": keys, "values": values}


def _own_attend(s):
    from flexengine_b200 import ops
    c = s.case
    return ops.paged_attention_kv4(s.queries, s.cache, s.table, s.step, c["heads"], c["kv"], c["d"], c["page"], s.scale, c["window"],
                                   keep_first=c["keep"])


def _own_sample(s):
    from flexengine_b200 import ops
    tokens, probability, kept = ops.sample_filtered(s.logits, s.temperature, s.top_k, s.top_p, s.min_p, s.uniform)
    return {"tokens": tokens, "probability": probability, "kept": kept}


# ---- the plain forms ----------------------------------------------------------------------------------------------------
def _pieces(cache, n):
    """Views of the cache's parts: key codes, value codes [..., 16, 16 n], and the pairs [..., 16, n, 2] of keys and values."""
    codes = [cache[..., at:at + 256 * n].unflatten(-1, (16, 16 * n)) for at in (0, 256 * n)]
    pairs = [cache[..., at:at + 64 * n].unflatten(-1, (16, 4 * n)) for at in (512 * n, 576 * n)]
    return codes + pairs


def _read(codes, pairs, inner, d):
    """The numbers [..., d] that code rows [..., 16 n] and pair rows [..., 4 n] stand for; ``inner``: 4 words or 8 pieces a row."""
    n = codes.shape[-1] // 16
    each = torch.stack([codes & 15, codes >> 4], -1).unflatten(-2, (inner, n, 16 // inner))
    each = each.transpose(-4, -3).flatten(-3).to(torch.float32) - 8.0                     # [..., n, 32]
    pair = pairs.contiguous().view(torch.float16).unflatten(-1, (n, 2)).to(torch.float32)
    return (pair[..., 1:] + each * pair[..., :1]).flatten(-2)[..., :d]


def _write(x, inner):
    """(code rows, pair rows) of x [..., d] in 32 bits."""
    d = x.shape[-1]
    n = _groups(d)
    x = x.clamp(-LARGEST, LARGEST)
    low = torch.nn.functional.pad(x, (0, 32 * n - d), value=math.inf).unflatten(-1, (n, 32)).amin(-1)
    high = torch.nn.functional.pad(x, (0, 32 * n - d), value=-math.inf).unflatten(-1, (n, 32)).amax(-1)
    scale = ((high - low) / 15.0).to(torch.float16)
    centre = (low + 8.0 * scale.to(torch.float32)).to(torch.float16)
    s, c = scale.to(torch.float32)[..., None], centre.to(torch.float32)[..., None]
    x = torch.nn.functional.pad(x, (0, 32 * n - d)).unflatten(-1, (n, 32))
    codes = torch.where(s > 0, (torch.round((x - c) / s) + 8.0).clamp(0.0, 15.0), 8.0).to(torch.uint8)
    codes = codes.unflatten(-1, (inner, 16 // inner, 2)).transpose(-4, -3).flatten(-4, -2)
    return codes[..., 0] | (codes[..., 1] << 4), torch.stack([scale, centre], -1).flatten(-2).view(torch.uint8)


def _turn(x, angle_cos, angle_sin, rot, pairs):
    """Heads x [tokens, heads, d] with their first ``rot`` entries rotated."""
    if not rot:
        return x
    turned = x[..., :rot]
    a, b = (turned[..., :rot // 2], turned[..., rot // 2:]) if pairs == "halves" else (turned[..., ::2], turned[..., 1::2])
    first, second = a * angle_cos - b * angle_sin, b * angle_cos + a * angle_sin
    done = torch.cat([first, second], -1) if pairs == "halves" else torch.stack([first, second], -1).flatten(-2)
    return torch.cat([done, x[..., rot:]], -1)


def _plain_store(s):
    c = s.case
    heads, kv, d, page = c["heads"], c["kv"], c["d"], c["page"]
    x = s.projected.to(torch.float32)
    if s.bias is not None:
        x = x + s.bias
    x = x.unflatten(-1, (heads + 2 * kv, d))
    cos = sin = None
    if c["rot"]:
        angle = s.positions.to(torch.float64)[:, None, None] * s.inv_freq.to(torch.float64)
        cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    queries = _turn(x[:, :heads], cos, sin, c["rot"], c["pairs"]).flatten(-2).to(TYPES[c["dtype"]])
    keys = _turn(x[:, heads:heads + kv], cos, sin, c["rot"], c["pairs"])
    parts = _pieces(s.cache, _groups(d))
    at = (s.slots.long() // page, slice(None), s.slots.long() % page // 16, s.slots.long() % 16)
    key_codes, key_pairs = _write(keys, 4)
    value_codes, value_pairs = _write(x[:, heads + kv:], 8)
    parts[0][at], parts[1][at], parts[2][at], parts[3][at] = key_codes, value_codes, key_pairs, value_pairs
    held = [p[at] for p in parts]
    return {"queries": queries, "keys": _read(held[0], held[2], 4, d).to(torch.bfloat16),
            "values": _read(held[1], held[3], 8, d).to(torch.bfloat16)}


def _plain_attend(s):
    c = s.case
    heads, kv, d = c["heads"], c["kv"], c["d"]
    parts = _pieces(s.cache[s.table.clamp(min=0).long()], _groups(d))                     # [R, pages, kv, tiles, 16, ...]
    keys, values = (_read(codes, pairs, inner, d).permute(0, 2, 1, 3, 4, 5).flatten(2, 4)
                    for codes, pairs, inner in ((parts[0], parts[2], 4), (parts[1], parts[3], 8)))      # [R, kv, L, d]
    lengths = s.step.cu_q[1:] - s.step.cu_q[:-1]
    row = torch.arange(s.step.max_q_len, device=DEV)
    real = row < lengths[:, None]                                                         # [R, Q]
    position = s.step.q_start[:, None] + row
    at = torch.where(real, s.step.cu_q[:-1, None] + row, 0).long()
    q = s.queries[at].to(torch.float32).unflatten(-1, (kv, heads // kv, d)).permute(0, 2, 3, 1, 4)      # [R, kv, G, Q, d]
    t = torch.arange(keys.shape[2], device=DEV)
    seen = t <= position[..., None]
    if c["window"]:
        seen &= (t > position[..., None] - c["window"]) | (t < c["keep"])
    written = (t < (s.step.q_start + lengths)[:, None])[:, None, :, None]
    keys, values = torch.where(written, keys, 0.0), torch.where(written, values, 0.0)
    scores = torch.matmul(q.flatten(2, 3), keys.transpose(-1, -2)).unflatten(2, (heads // kv, -1)) * s.scale
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    mixed = torch.matmul(weights.flatten(2, 3), values).unflatten(2, (heads // kv, -1))
    return mixed.permute(0, 3, 1, 2, 4).flatten(2)[real].to(s.queries.dtype)


def _plain_sample(s):
    # in 64 bits: a token's share of the whole is small where many are kept
    x = s.logits.to(torch.float64)
    greedy = s.temperature == 0
    largest, best = x.max(-1, keepdim=True)
    best = torch.argmax((x == largest).to(torch.int8), -1)
    mass = torch.exp((x - largest) / torch.where(greedy, 1.0, s.temperature).to(torch.float64)[:, None])
    _, order = torch.sort(x, dim=-1, descending=True, stable=True)
    ranked = mass.gather(-1, order)
    k = torch.where((s.top_k > 0) & ~greedy, s.top_k, x.shape[1])[:, None]
    ranked = torch.where(torch.arange(x.shape[1], device=DEV) < k, ranked, 0.0)
    upto = torch.cumsum(ranked, -1)
    # a token stays where those before it do not hold top_p of the mass yet, and where it has min_p of the largest one's
    share = s.top_p.to(torch.float64)[:, None]
    stays = (ranked > 0) & ((share >= 1) | (upto - ranked < share * upto[:, -1:])) & (ranked >= s.min_p.to(torch.float64)[:, None])
    kept = torch.zeros_like(stays).scatter_(-1, order, stays)
    mass = torch.where(kept, mass, 0.0)
    total = torch.cumsum(mass, -1)
    target = s.uniform.to(torch.float64)[:, None] * total[:, -1:]
    token = torch.where(greedy, best, torch.argmax((total > target).to(torch.int8), -1))
    chance = mass.gather(-1, token[:, None])[:, 0] / total[:, -1]
    return {"tokens": token.to(torch.int32), "probability": torch.where(greedy, 1.0, chance).to(torch.float32),
            "kept": torch.where(greedy, 1, kept.sum(-1)).to(torch.int32)}


# ---- the same in 64 bits, from the definitions --------------------------------------------------------------------------
def exact(case, seed):
    return {"store": _exact_store, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](prepare(case, seed))


def _exact_store(s):
    c = s.case
    heads, kv, d, rot = c["heads"], c["kv"], c["d"], c["rot"]
    x = s.projected.double() + (s.bias.double() if s.bias is not None else 0.0)
    x = x.view(-1, heads + 2 * kv, d)
    if rot:
        z = torch.exp(1j * s.positions.double()[:, None] * s.inv_freq.double())
        i = torch.arange(rot // 2, device=DEV)
        a, b = (i, i + rot // 2) if c["pairs"] == "halves" else (2 * i, 2 * i + 1)
        turned = torch.complex(x[:, :heads + kv, a], x[:, :heads + kv, b]) * z[:, None]
        x[:, :heads + kv, a], x[:, :heads + kv, b] = turned.real, turned.imag
    stored = x[:, heads:].clone()
    for first in range(0, d, 32):
        g = stored[..., first:first + 32].clamp(-LARGEST, LARGEST)
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        scale = ((high - low) / 15).half().double()
        centre = (low + 8 * scale).half().double()
        code = torch.where(scale > 0, torch.round((g - centre) / scale), 0.0).clamp(-8, 7)
        stored[..., first:first + 32] = centre + code * scale
    return {"queries": x[:, :heads].reshape(-1, heads * d), "keys": stored[:, :kv], "values": stored[:, kv:]}


def _exact_attend(s):
    c = s.case
    heads, kv, d, page, n = c["heads"], c["kv"], c["d"], c["page"], _groups(c["d"])
    i = torch.arange(32 * n, device=DEV)
    group, within = i // 32, i % 32
    # nibble (two a byte) of every number of a key and of a value row
    key_at = ((within // 8) * n + group) * 8 + within % 8
    value_at = ((within // 4) * n + group) * 4 + within % 4
    out = torch.zeros((s.queries.shape[0], heads, d), dtype=torch.float64, device=DEV)
    for r, (new, start) in enumerate(zip(s.step.host_lengths, s.step.host_starts)):
        length = start + new
        tiles = s.cache[s.table[r, :-(-length // page)].long()].transpose(1, 2).flatten(0, 1)             # [tiles, kv, bytes]
        first = int(s.step.cu_q[r])
        position = torch.arange(start, length, device=DEV)[:, None]
        t = torch.arange(length, device=DEV)
        seen = (t <= position) & (((t > position - c["window"]) | (t < c["keep"])) if c["window"] else True)
        for h in range(kv):
            tile = tiles[:, h]
            numbers = []
            for codes, pairs, at in ((0, 512 * n, key_at), (256 * n, 576 * n, value_at)):
                byte = tile[:, codes:codes + 256 * n].reshape(-1, 16 * n)[:length]
                nibble = (byte[:, at // 2] >> (4 * (at % 2)).to(torch.uint8)) & 15
                pair = tile[:, pairs:pairs + 64 * n].reshape(-1, 4 * n)[:length].contiguous().view(torch.float16).view(-1, n, 2).double()
                numbers.append((pair[:, group, 1] + (nibble.double() - 8) * pair[:, group, 0])[:, :d])
            mine = slice(h * (heads // kv), (h + 1) * (heads // kv))
            q = s.queries[first:first + new].double().view(new, heads, d)[:, mine]
            scores = torch.einsum("qgd,ld->gql", q, numbers[0]) * s.scale
            weights = torch.softmax(torch.where(seen, scores, -math.inf), -1)
            out[first:first + new, mine] = torch.einsum("gql,ld->qgd", weights, numbers[1])
    return out.flatten(1)


def _exact_sample(s):
    chances, tokens, kept = [], [], []
    for row in range(s.logits.shape[0]):
        x = s.logits[row].double().cpu()
        heat, k, p, least = (float(v[row]) for v in (s.temperature, s.top_k, s.top_p, s.min_p))
        if heat == 0:
            chances.append(1.0), tokens.append(int(x.numpy().argmax())), kept.append(1)
            continue
        weight = ((x - x.max()) / heat).exp().numpy()
        order = (-x.numpy()).argsort(kind="stable")[:int(k) if k > 0 else None]
        running = weight[order].cumsum()
        count = len(order) if p >= 1 else int((running < p * running[-1]).sum()) + 1
        chosen = order[:count]
        chosen = chosen[weight[chosen] >= least]
        chosen.sort()
        running = weight[chosen].cumsum()
        place = min(int((running <= float(s.uniform[row]) * running[-1]).sum()), len(chosen) - 1)
        tokens.append(int(chosen[place])), kept.append(len(chosen)), chances.append(float(weight[chosen[place]] / running[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probability": torch.tensor(chances, dtype=torch.float64),
            "kept": torch.tensor(kept, dtype=torch.int32)}
