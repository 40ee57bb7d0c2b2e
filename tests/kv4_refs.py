"""Keys and values in 4 bits and sampling with top-p and min-p, written plainly: every operation of the CPU reference set
(``kernel_refs``) and these on top, so that an engine can run on them.  Numbers are taken in 64 bits."""
import math

import torch

from kernel_refs import *  # noqa: F401,F403 - the set of operations an engine asks for
import kernel_refs

LARGEST = 61440.0


def __getattr__(name):
    return getattr(kernel_refs, name)


def groups(d):
    return -(-d // 32)


def places(d, key):
    """For every number of a row: the nibble of the row's codes that holds it (two a byte, the low one first)."""
    i, n = torch.arange(d), groups(d)
    g, w = i // 32, i % 32
    return ((w // 8) * n + g) * 8 + w % 8 if key else ((w // 4) * n + g) * 4 + w % 4


def quantised(x):
    """(codes, scales, centres) of x [..., d] in float64: codes [..., d] whole, the pairs [..., groups] as half precision holds them."""
    x = x.double()
    d = x.shape[-1]
    codes, scales, centres = torch.empty_like(x), [], []
    for first in range(0, d, 32):
        part = x[..., first:first + 32]
        nan = part.isnan().any(-1, keepdim=True)
        part = part.clamp(-LARGEST, LARGEST)
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        scale = torch.where(nan, math.nan, ((high - low) / 15).half().double())
        centre = (low + 8 * scale).half().double()
        codes[..., first:first + 32] = torch.where(scale > 0, (torch.round((part - centre) / scale) + 8).clamp(0, 15), 8.0)
        scales.append(scale)
        centres.append(centre)
    return codes, torch.cat(scales, -1), torch.cat(centres, -1)


def tile_parts(cache, d):
    """Views [..., 16, bytes] of a cache's key codes, value codes, key pairs and value pairs."""
    n = groups(d)
    return [cache[..., at:at + 16 * size].unflatten(-1, (16, size)) for at, size in ((0, 16 * n), (256 * n, 16 * n), (512 * n, 4 * n), (576 * n, 4 * n))]


def write_rows(cache, slots, keys, values):
    """Puts rows [T, nkv, d] into the cache [pages, nkv, page / 16, bytes] at their slots (below 0: left out)."""
    d, page = keys.shape[-1], cache.shape[2] * 16
    parts = tile_parts(cache, d)
    for t, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        at = (slot // page, slice(None), slot % page // 16, slot % 16)
        for side, x in enumerate((keys[t], values[t])):
            codes, scale, centre = quantised(x.cpu())
            nibbles = torch.zeros(x.shape[0], 32 * groups(d), dtype=torch.uint8)
            nibbles[:, places(d, side == 0)] = codes.to(torch.uint8)
            parts[side][at] = (nibbles[:, ::2] | (nibbles[:, 1::2] << 4)).to(cache.device)
            pairs = torch.stack([scale.half(), centre.half()], -1).contiguous().view(torch.uint8).flatten(1)
            parts[2 + side][at] = pairs.to(cache.device)


def read_rows(cache, slots, d):
    """(keys, values) [N, nkv, d] in float64 that the cache holds at slots [N]; zeros below 0."""
    page = cache.shape[2] * 16
    s = slots.long().clamp(min=0)
    parts = [p[s // page, :, s % page // 16, s % 16].cpu() for p in tile_parts(cache, d)]
    out = []
    for side in range(2):
        at = places(d, side == 0)
        code = (parts[side][..., at // 2] >> (4 * (at % 2)).to(torch.uint8)) & 15
        pair = parts[2 + side].contiguous().view(torch.float16).unflatten(-1, (groups(d), 2)).double()
        g = torch.arange(d) // 32
        x = pair[..., g, 1] + (code.double() - 8) * pair[..., g, 0]
        out.append(torch.where(slots.cpu()[:, None, None] >= 0, x, 0.0))
    return out


def turned(x, positions, inv_freq, rot, pairs, gain=1.0):
    """Heads x [T, heads, d] in float64 with their first ``rot`` entries rotated."""
    if not rot:
        return x
    angle = positions.cpu().double()[:, None] * inv_freq.cpu().double()
    cos, sin = torch.cos(angle)[:, None] * gain, torch.sin(angle)[:, None] * gain
    i = torch.arange(rot // 2)
    a, b = (i, i + rot // 2) if pairs == "halves" else (2 * i, 2 * i + 1)
    out = x.clone()
    out[..., a], out[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    return out


def split_heads(projected, bias, positions, inv_freq, rot, nq, nkv, d, pairs="halves", gain=1.0):
    """(queries, keys, values) [T, heads, d] in float64: bias and rotation added."""
    x = projected[:, :(nq + 2 * nkv) * d].cpu().double()
    if bias is not None:
        x = x + bias.cpu().double()
    x = x.view(-1, nq + 2 * nkv, d)
    x = torch.cat([turned(x[:, :nq + nkv], positions, inv_freq, rot, pairs, gain), x[:, nq + nkv:]], 1)
    return x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]


def qkv_rope_kv4(projected, bias, positions, inv_freq, rot, slot_mapping, cache, nq, nkv, d, page_size, pairs="halves", rot_gain=1.0,
                 out_dtype=None):
    q, k, v = split_heads(projected, bias, positions, inv_freq, rot, nq, nkv, d, pairs, rot_gain)
    if slot_mapping is not None:
        write_rows(cache, slot_mapping, k.float(), v.float())
    return q.flatten(1).to(projected.device, out_dtype or projected.dtype)


def attention64(q, cache, block_table, cu_q, q_start, nq, nkv, d, page_size, scale, window=0, keep_first=0, sink=False):
    """[T, nq d] in float64, request by request."""
    out = torch.zeros(q.shape[0], nq, d, dtype=torch.float64)
    cu, starts = cu_q.tolist(), q_start.tolist()
    for r, start in enumerate(starts):
        new = cu[r + 1] - cu[r]
        if new <= 0:
            continue
        length = start + new
        position = torch.arange(start, length)[:, None]
        t = torch.arange(length)
        seen = t <= position
        if window:
            seen = seen & ((t > position - window) | (t < keep_first))
        pages = block_table[r].cpu().long()[t // page_size]
        slots = torch.where((pages >= 0) & seen.any(0), pages * page_size + t % page_size, -1)
        keys, values = read_rows(cache, slots, d)
        seen = seen & (pages >= 0)
        mine = q[cu[r]:cu[r + 1], :nq * d].cpu().double().view(new, nkv, nq // nkv, d)
        scores = torch.einsum("qhgd,lhd->hgql", mine, keys) * scale
        scores = torch.where(seen, scores, -math.inf)
        top = scores.amax(-1, keepdim=True)
        if sink:
            top = top.clamp(min=0.0)
        weights = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
        total = weights.sum(-1, keepdim=True) + (torch.exp(-top) if sink else 0.0)
        weights = torch.where(total > 0, weights / total, 0.0)
        # what is not seen takes no part, whatever it holds
        mixed = torch.zeros(nkv, nq // nkv, new, d, dtype=torch.float64)
        for h in range(nkv):
            for i in range(new):
                at = seen[i].nonzero().flatten()
                mixed[h, :, i] = weights[h, :, i][:, at] @ values[at, h]
        out[cu[r]:cu[r + 1]] = mixed.permute(2, 0, 1, 3).flatten(1, 2)
    return out.flatten(1)


def paged_attention_kv4(q, cache, block_table, ctx, nq, nkv, d, page_size, scale, window=0, keep_first=0, sink=False):
    return attention64(q, cache, block_table, ctx.cu_q, ctx.q_start, nq, nkv, d, page_size, scale, window, keep_first, sink).to(q.device, q.dtype)


def sample_filtered(logits, temperature, top_k, top_p, min_p, uniform, blocks=0):
    """Row by row in float64: (tokens, probabilities, numbers of tokens that stay)."""
    tokens, chances, numbers = [], [], []
    for r in range(logits.shape[0]):
        x = logits[r].cpu().double()
        x = torch.where(x.isnan(), -math.inf, x)
        top = float(x.max())
        heat = float(temperature[r])
        if top == -math.inf:
            tokens.append(0), chances.append(0.0), numbers.append(0)
            continue
        if not heat > 0:
            tokens.append(int((x == top).nonzero()[0])), chances.append(1.0), numbers.append(1)
            continue
        mass = torch.where(x == top, 1.0, torch.exp((x - top) / heat))
        order = torch.sort(x, descending=True, stable=True).indices
        k = int(top_k[r])
        if 0 < k < len(x):
            order = order[:k]
        order = order[mass[order] > 0]
        upto = torch.cumsum(mass[order], 0)
        p = float(top_p[r])
        if p < 1:
            stays = upto - mass[order] < p * upto[-1]
            stays[0] = True
            order = order[stays]
        order = order[mass[order] >= min(float(min_p[r]), 1.0)]
        order = order.sort().values
        upto = torch.cumsum(mass[order], 0)
        u = min(max(float(uniform[r]), 0.0), 1.0)
        at = min(int((upto <= u * float(upto[-1])).sum()), len(order) - 1)
        tokens.append(int(order[at])), chances.append(float(mass[order[at]] / upto[-1])), numbers.append(len(order))
    dev = logits.device
    return (torch.tensor(tokens, dtype=torch.int32, device=dev), torch.tensor(chances, dtype=torch.float32, device=dev),
            torch.tensor(numbers, dtype=torch.int32, device=dev))
