"""The kernels of a cache held in 4 bits against 64-bit plain forms: storing with bias and rotation, reading rows back, attention for single
tokens and portions, and the engine on them."""
import math
import types

import pytest
import torch

import kv4_refs
from flexengine_b200.cache.manager import kv4_shape

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}       # of a rounding to the type, relative


def ops():
    from flexengine_b200 import ops as cuda_ops
    return cuda_ops


@pytest.fixture()
def gen():
    g = torch.Generator(device=DEV)
    g.manual_seed(77)
    return g


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


# ---- storing --------------------------------------------------------------------------------------------------------------
def check_stored(cache, slots, keys, values, what=""):
    """What the cache holds against the exact rows.  A scale is the group's range / 15 and a centre its smallest number + 8 scales, each rounded
    to half precision (2^-11 of it, or 2^-25 among its smallest) from 32-bit arithmetic (4 roundings of 2^-24 of the group's largest number);
    a code is the nearest one to the number, both ends' apart, which may lie beyond by what the pair's rounding moved them."""
    d = keys.shape[-1]
    got = kv4_refs.read_rows(cache.cpu(), slots.cpu(), d)
    page = cache.shape[2] * 16
    for side, want in enumerate((keys, values)):
        pairs = kv4_refs.tile_parts(cache.cpu(), d)[2 + side]
        s = slots.cpu().long()
        held = pairs[s // page, :, s % page // 16, s % 16].contiguous().view(torch.float16).unflatten(-1, (kv4_refs.groups(d), 2)).double()
        for i, first in enumerate(range(0, d, 32)):
            w = want[..., first:first + 32].clamp(-61440, 61440)
            big = w.abs().amax(-1)
            low, high = w.amin(-1), w.amax(-1)
            scale, centre = held[..., i, 0], held[..., i, 1]
            rough = 4 * 2.0 ** -24 * big
            assert ((scale - (high - low) / 15).abs() <= 2.0 ** -11 * scale + 2.0 ** -25 + rough).all(), f"{what}: scale of group {i}, side {side}"
            assert ((centre - (low + 8 * scale)).abs() <= 2.0 ** -11 * centre.abs() + 2.0 ** -25 + rough).all(), f"{what}: centre of group {i}, side {side}"
            off = (got[side][..., first:first + 32] - w).abs()
            ends = 15 * (2.0 ** -11 * scale + 2.0 ** -25) + 2.0 ** -11 * centre.abs() + 2.0 ** -25
            assert (off <= (scale / 2 + ends + 4 * rough)[..., None]).all(), f"{what}: numbers of group {i}, side {side}"
            inner = off[(w > (low + scale)[..., None]) & (w < (high - scale)[..., None])]
            bound = (scale / 2 * (1 + 1e-3) + 4 * rough)[..., None].expand_as(w)[(w > (low + scale)[..., None]) & (w < (high - scale)[..., None])]
            assert (inner <= bound).all(), f"{what}: a number away from the ends is not at its nearest code"


@pytest.mark.parametrize("source,out", [(torch.float32, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("T,nq,nkv,d,rot,pairs,page,bias,wider", [
    (1, 28, 4, 128, 128, "halves", 16, True, 0), (1, 2, 1, 16, 0, "halves", 16, False, 0), (5, 3, 3, 48, 6, "halves", 32, True, 0),
    (37, 14, 2, 64, 32, "interleaved", 16, False, 8), (33, 6, 2, 80, 80, "interleaved", 48, True, 0), (17, 8, 1, 256, 200, "halves", 64, True, 4),
    (300, 16, 8, 112, 112, "halves", 16, False, 3), (2000, 4, 2, 128, 128, "halves", 16, True, 0), (901, 3, 1, 64, 32, "interleaved", 32, False, 4),
    (700, 2, 2, 256, 192, "halves", 16, True, 0), (777, 3, 1, 80, 20, "halves", 16, True, 2), (149, 4, 2, 208, 14, "interleaved", 16, True, 1)])
def test_store(source, out, T, nq, nkv, d, rot, pairs, page, bias, wider, gen):
    width = (nq + 2 * nkv) * d
    projected = normal(gen, T, width + wider).to(source)[:, :width] if wider else normal(gen, T, width).to(source)
    b = normal(gen, width) if bias else None
    positions = torch.randint(0, 131072, (T,), generator=gen, device=DEV, dtype=torch.int32)
    inv_freq = (1e6 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))).float().to(DEV) if rot else None
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:T].to(torch.int32)
    if T > 4:
        slots[3] = -1
    cache = torch.full(kv4_shape(pages, nkv, page, d), 90, dtype=torch.uint8, device=DEV)
    q = ops().qkv_rope_kv4(projected, b, positions, inv_freq, rot, slots, cache, nq, nkv, d, page, pairs=pairs, rot_gain=1.25 if rot else 1.0, out_dtype=out)
    ops().check_status(DEV)
    want = kv4_refs.split_heads(projected, b, positions, inv_freq, rot, nq, nkv, d, pairs, 1.25 if rot else 1.0)
    # six 32-bit roundings of numbers up to the pair's, then the one to the queries' type
    loose = HALF_STEP[out] * want[0].abs() + 6 * 2.0 ** -24 * 1.25 * 2 * float(want[0].abs().max())
    assert ((q.cpu().double().view(T, nq, d) - want[0]).abs() <= loose).all()
    kept = slots >= 0
    check_stored(cache, slots[kept], want[1][kept.cpu()], want[2][kept.cpu()])
    # what no slot names is left as it was
    page_of = torch.full((pages * page,), True, device=DEV)
    page_of[slots[kept].long()] = False
    for part in kv4_refs.tile_parts(cache, d):
        rows = part.permute(0, 2, 3, 1, 4).reshape(pages * page, -1)
        assert (rows[page_of] == 90).all()


def test_store_without_slots_gives_the_queries(gen):
    projected = normal(gen, 3, 4 * 32)
    cache = torch.full(kv4_shape(1, 1, 16, 32), 7, dtype=torch.uint8, device=DEV)
    q = ops().qkv_rope_kv4(projected, None, torch.zeros(3, dtype=torch.int32, device=DEV), None, 0, None, cache, 2, 1, 32, 16)
    assert torch.equal(q, projected[:, :64]) and (cache == 7).all()
    assert ops().qkv_rope_kv4(projected[:0], None, torch.zeros(0, dtype=torch.int32, device=DEV), None, 0, None, cache, 2, 1, 32, 16).shape == (0, 64)


def test_store_special_numbers(gen):
    """Equal numbers, numbers beyond the largest, infinities, a NaN, next to nothing; and a slot beyond the cache."""
    x = normal(gen, 8, 4, 64)
    x[0], x[1, :, 3], x[2, :, 40], x[3] = 2.5, 1e30, -math.inf, x[3] * 1e-9
    x[4, 1, 7] = x[4, 2, 50] = math.nan
    x[5] = 0.0
    projected = torch.cat([x[:, :2], x[:, 2:]], 1).reshape(8, -1)
    cache = torch.zeros(kv4_shape(2, 1, 16, 64), dtype=torch.uint8, device=DEV)
    slots = torch.tensor([0, 1, 2, 3, 4, 5, 6, 32], dtype=torch.int32, device=DEV)
    ops().qkv_rope_kv4(projected, None, torch.zeros(8, dtype=torch.int32, device=DEV), None, 0, slots, cache, 2, 1, 64, 16)
    with pytest.raises(RuntimeError, match="slot out of range"):
        ops().check_status(DEV)
    keys, values = ops().kv4_rows(cache, slots[:7], 1, 64, 16, torch.float32)
    nan = torch.zeros(7, 1, 64, dtype=torch.bool)
    assert torch.equal(keys.cpu().isnan(), nan | False if not x[:7, 2].isnan().any() else keys.cpu().isnan())
    for got, head in ((keys, 2), (values, 3)):
        want = x[:7, head].cpu().double().clamp(-61440, 61440)
        for t in range(7):
            for first in (0, 32):
                a, w = got[t, 0, first:first + 32].cpu().double(), want[t, first:first + 32]
                if w.isnan().any():
                    assert a.isnan().all()
                else:
                    step = float(w.max() - w.min()) / 15
                    assert float((a - w).abs().max()) <= step / 2 + 16 * (step * 2.0 ** -11 + 2.0 ** -25) + float(w.abs().max()) * 2.0 ** -10 + 2.0 ** -24
    assert keys[4].isnan().sum() == 32 and values[4].isnan().sum() == 0


@pytest.mark.parametrize("d,page", [(16, 16), (96, 48), (128, 16), (256, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_are_what_the_bytes_say(d, page, dtype, gen):
    cache = torch.randint(0, 256, kv4_shape(5, 3, page, d), generator=gen, device=DEV, dtype=torch.uint8)
    n = kv4_refs.groups(d)
    pairs = cache[..., 512 * n:].view(torch.float16)
    pairs.copy_((normal(gen, *pairs.shape)).half())
    slots = torch.randint(-1, 5 * page, (41,), generator=gen, device=DEV, dtype=torch.int32)
    got = ops().kv4_rows(cache, slots, 3, d, page, dtype)
    for g, w in zip(got, kv4_refs.read_rows(cache, slots, d)):
        assert torch.equal(g.cpu(), w.float().to(dtype))       # code times scale is exact, the sum rounds once
    empty = ops().kv4_rows(cache, slots[:0], 3, d, page, dtype)
    assert empty[0].shape == (0, 3, d)


# ---- attention -------------------------------------------------------------------------------------------------------------
def problem(gen, lengths, nq, nkv, d, dtype, page=16, scale_of=1.0, garbage=True, wider=0, order="scattered"):
    """A cache, its table and a step of queries.  ``lengths``: (new tokens, cached ones before them) a request.  Places that no token was
    written to hold NaN."""
    need = [max(1, -(-(a + b) // page)) for a, b in lengths]
    pages = sum(need) + 2
    n = kv4_refs.groups(d)
    cache = torch.randint(0, 256, kv4_shape(pages, nkv, page, d), generator=gen, device=DEV, dtype=torch.uint8)
    pairs = cache[..., 512 * n:].view(torch.float16).unflatten(-1, (-1, 2))
    pairs[..., 0] = ((torch.rand(pairs.shape[:-1], generator=gen, device=DEV) * 0.3 + 0.05) * scale_of).half()
    pairs[..., 1] = (normal(gen, *pairs.shape[:-1]) * 0.3 * scale_of).half()
    ids = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32) if order == "scattered" else torch.arange(pages, device=DEV, dtype=torch.int32)
    table = torch.full((len(lengths), max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = ids[at:at + k]
        at += k
        total = sum(lengths[r])
        if garbage:
            for slot in range(total, k * page):
                for part in kv4_refs.tile_parts(cache, d):
                    part[ids[at - k + slot // page], :, slot % page // 16, slot % 16] = 255
    new = torch.tensor([a for a, _ in lengths])
    cu = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).to(torch.int32)
    ctx = types.SimpleNamespace(cu_q=cu.to(DEV), q_start=torch.tensor([b for _, b in lengths], dtype=torch.int32, device=DEV), max_q_len=int(new.max()),
                                max_ctx_len=max(a + b for a, b in lengths), host_lengths=new.tolist(), host_starts=[b for _, b in lengths])
    q = (normal(gen, int(cu[-1]), nq * d + wider) * 2).to(dtype)
    return q[:, :nq * d] if wider else q, cache, table, ctx


def largest_value(cache, d):
    n = kv4_refs.groups(d)
    pairs = cache[..., 576 * n:].view(torch.float16).unflatten(-1, (-1, 2)).double()
    pairs = torch.where(pairs.isnan(), 0.0, pairs)
    return float((pairs[..., 1].abs() + 8 * pairs[..., 0].abs()).max())


def check_attention(got, want, cache, d, what=""):
    """bfloat16: the result's rounding (2^-8); the weights' to half precision (2^-11 of the sums of codes times scales, up to the largest value); and
    scores whose sums over raised codes are off by up to 2^-23 a product of numbers near 2^15 in units of a code (2^-9 of a weight at these
    scales): together within 2^-8 of the largest value.  32-bit: 22 bits of queries and weights, sums and exponentials in 32 bits."""
    got = got.cpu().double()
    top = largest_value(cache, d)
    off = (got - want).abs()
    if got.shape[0] == 0:
        return
    assert not got.isnan().any(), what
    if what.endswith("float32"):
        assert float(off.max()) <= 2e-5 * top, f"{what}: {float(off.max()) / top:.2e} of the largest value"
    else:
        assert (off <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * top).all(), f"{what}: {float(off.max()) / top:.2e} of the largest value"
        assert float((got - want).norm()) <= 2.0 ** -8 * float(want.norm()) + 1e-30, what


def run_attention(q, cache, table, ctx, nq, nkv, d, page, **more):
    out = ops().paged_attention_kv4(q, cache, table, ctx, nq, nkv, d, page, d ** -0.5, **more)
    ops().check_status(DEV)
    want = kv4_refs.attention64(q, cache, table, ctx.cu_q, ctx.q_start, nq, nkv, d, page, d ** -0.5, **more)
    return out, want


HEADS = [(28, 4, 128), (12, 2, 128), (14, 2, 64), (3, 3, 16), (6, 2, 48), (16, 16, 80), (20, 1, 96), (33, 3, 112), (8, 2, 160), (4, 1, 192), (9, 3, 224), (8, 2, 256), (2, 2, 32)]
DECODE = {"one key": [(1, 0)], "a tile": [(1, 15)], "a tile and one": [(1, 16)], "two": [(1, 30), (1, 300)],
          "ragged": [(1, 700), (1, 3), (1, 1030), (1, 0), (1, 64), (1, 255)], "long and short": [(1, 5000), (1, 17)]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", list(DECODE))
@pytest.mark.parametrize("nq,nkv,d", HEADS)
def test_decode(nq, nkv, d, lengths, dtype, gen):
    if lengths == "long and short" and d not in (64, 128, 256):
        lengths = "two"
    args = problem(gen, DECODE[lengths], nq, nkv, d, dtype)
    out, want = run_attention(*args, nq, nkv, d, 16)
    check_attention(out, want, args[1], d, f"{lengths} {nq}/{nkv}/{d} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,keep", [(1, 0), (7, 0), (16, 0), (100, 0), (100, 1), (100, 16), (33, 40), (5000, 3), (64, 700)])
@pytest.mark.parametrize("page", [16, 48, 64])
def test_decode_windows(window, keep, page, dtype, gen):
    args = problem(gen, [(1, 640), (1, 99), (1, 100), (1, 0), (1, 1500)], 7, 1, 64, dtype, page=page)
    out, want = run_attention(*args, 7, 1, 64, page, window=window, keep_first=keep)
    check_attention(out, want, args[1], 64, f"window {window} keep {keep} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(28, 4, 128), (14, 2, 64), (6, 2, 48), (8, 2, 256), (16, 16, 80)])
@pytest.mark.parametrize("lengths,window,keep", [
    ([(5, 0)], 0, 0), ([(1, 40), (9, 100), (1, 0), (33, 31)], 0, 0), ([(70, 3), (2, 500), (0, 60), (17, 0)], 0, 0), ([(40, 200), (1, 90), (3, 3)], 50, 0),
    ([(40, 200), (1, 90), (3, 300)], 50, 20), ([(130, 500)], 16, 1), ([(300, 0)], 0, 0)])
def test_portions(nq, nkv, d, lengths, window, keep, dtype, gen):
    args = problem(gen, lengths, nq, nkv, d, dtype, page=32)
    out, want = run_attention(*args, nq, nkv, d, 32, window=window, keep_first=keep)
    check_attention(out, want, args[1], d, f"{lengths} window {window} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[(1, 3), (1, 900)], [(20, 40), (1, 5)], [(1, 4000)], [(200, 100)]])
def test_sink(lengths, dtype, gen):
    args = problem(gen, lengths, 14, 2, 128, dtype)
    out, want = run_attention(*args, 14, 2, 128, 16, sink=True)
    check_attention(out, want, args[1], 128, f"sink {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale_of", [2e-4, 30.0, 2000.0])
def test_scales_far_from_one(scale_of, dtype, gen):
    """Values of any size that half precision holds, beside scores near one (the queries go the other way)."""
    q, cache, table, ctx = problem(gen, [(1, 600), (1, 20)], 12, 2, 128, dtype, scale_of=scale_of)
    q = (q.float() / scale_of).to(dtype)
    out, want = run_attention(q, cache, table, ctx, 12, 2, 128, 16)
    check_attention(out, want, cache, 128, f"scales times {scale_of} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_far_key_decides(dtype, gen):
    """A key whose score stands far above the others, in the first, a middle and the last tile; queries of 10^4 and of 10^-4 times the rest."""
    for place in (0, 700, 1233):
        q, cache, table, ctx = problem(gen, [(1, 1233)], 8, 2, 64, dtype)
        keys, _ = kv4_refs.read_rows(cache, table[0, place // 16].cpu() * 16 + torch.tensor([place % 16]), 64)
        q = (keys[0].repeat_interleave(4, 0).flatten()[None] * 8).to(dtype).to(DEV)
        out, want = run_attention(q, cache, table, ctx, 8, 2, 64, 16)
        check_attention(out, want, cache, 64, f"far key {place} {dtype}")
        for size in (1e4, 1e-4):
            sized = (q.float() * size).to(dtype)
            out = ops().paged_attention_kv4(sized, cache, table, ctx, 8, 2, 64, 16, 64 ** -0.5 / size)
            want = kv4_refs.attention64(sized, cache, table, ctx.cu_q, ctx.q_start, 8, 2, 64, 16, 64 ** -0.5 / size)
            check_attention(out, want, cache, 64, f"far key {place} size {size} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_is_seen_only_where_it_is_visible(dtype, gen):
    """A stored value group that reads as NaN makes NaN of its 32 numbers for the queries that see it, of nothing else."""
    q, cache, table, ctx = problem(gen, [(20, 200), (1, 90)], 4, 2, 64, dtype)
    n = kv4_refs.groups(64)
    for r, place, group in ((0, 210, 1), (1, 40, 0)):
        pairs = cache[..., 576 * n:].view(torch.float16).view(cache.shape[:3] + (16, n, 2))
        pairs[int(table[r, place // 16]), 1, 0, place % 16, group, 0] = math.nan
    out = ops().paged_attention_kv4(q, cache, table, ctx, 4, 2, 64, 16, 0.125).view(21, 4, 64)
    bad = torch.zeros(21, 4, 64, dtype=torch.bool, device=DEV)
    bad[10:20, 2:, 32:] = True
    bad[20, 2:, :32] = True
    assert torch.equal(out.isnan(), bad)


def test_strides_empty_steps_and_types(gen):
    q, cache, table, ctx = problem(gen, [(1, 50), (1, 9)], 6, 2, 48, torch.bfloat16, wider=40)
    out, want = run_attention(q, cache, table, ctx, 6, 2, 48, 16)
    check_attention(out, want, cache, 48, "strided bfloat16")
    none = types.SimpleNamespace(cu_q=torch.zeros(3, dtype=torch.int32, device=DEV), q_start=ctx.q_start, max_q_len=0, max_ctx_len=50)
    assert ops().paged_attention_kv4(q[:0], cache, table, none, 6, 2, 48, 16, 0.1).shape == (0, 288)
    with pytest.raises(TypeError):
        ops().paged_attention_kv4(q.half(), cache, table, ctx, 6, 2, 48, 16, 0.1)
    with pytest.raises(ValueError, match="tensors on"):
        ops().paged_attention_kv4(q, cache, table.cpu(), ctx, 6, 2, 48, 16, 0.1)


@pytest.mark.parametrize("lengths", [[(1, 40), (1, 1600)], [(1, 9000)], [(1, 40)], [(30, 100)]])
def test_pages_that_are_not_there(lengths, gen):
    """A table that names no page, or one beyond the cache: those keys are left out and the status word says so."""
    q, cache, table, ctx = problem(gen, lengths, 8, 2, 64, torch.bfloat16)
    table[-1, 1] = cache.shape[0]
    table[-1, 0] = -7
    out = ops().paged_attention_kv4(q, cache, table, ctx, 8, 2, 64, 16, 0.125)
    with pytest.raises(RuntimeError, match="page id out of range"):
        ops().check_status(DEV)
    table[-1, 1] = -1
    want = kv4_refs.attention64(q, cache, table, ctx.cu_q, ctx.q_start, 8, 2, 64, 16, 0.125)
    check_attention(out, want, cache, 64, "pages missing bfloat16")


def test_offsets_beyond_32_bits(gen):
    """A cache of more than 2^32 bytes, its last pages in use, written and read."""
    nkv, d, page = 8, 128, 64
    pages = (1 << 32) // (nkv * page * 160) + 40
    cache = torch.empty(kv4_shape(pages, nkv, page, d), dtype=torch.uint8, device=DEV)
    T = 150
    projected = normal(gen, T, 3 * nkv * d)
    ids = [pages - 1, 3, pages - 5]
    slots = torch.tensor([ids[t // page] * page + t % page for t in range(T)], dtype=torch.int32, device=DEV)
    q = ops().qkv_rope_kv4(projected, None, torch.arange(T, device=DEV, dtype=torch.int32), None, 0, slots, cache, nkv, nkv, d, page, out_dtype=torch.float32)
    small = torch.empty(kv4_shape(3, nkv, page, d), dtype=torch.uint8, device=DEV)
    ops().qkv_rope_kv4(projected, None, torch.arange(T, device=DEV, dtype=torch.int32), None, 0, torch.arange(T, device=DEV, dtype=torch.int32), small, nkv, nkv, d, page)
    ctx = types.SimpleNamespace(cu_q=torch.tensor([0, 1], dtype=torch.int32, device=DEV), q_start=torch.tensor([T - 1], dtype=torch.int32, device=DEV), max_q_len=1, max_ctx_len=T)
    there = ops().paged_attention_kv4(q[-1:], cache, torch.tensor([ids], dtype=torch.int32, device=DEV), ctx, nkv, nkv, d, page, 0.1)
    here = ops().paged_attention_kv4(q[-1:], small, torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV), ctx, nkv, nkv, d, page, 0.1)
    assert torch.equal(there, here)
    assert all(torch.equal(a, b) for a, b in zip(ops().kv4_rows(cache, slots, nkv, d, page), ops().kv4_rows(small, torch.arange(T, device=DEV, dtype=torch.int32), nkv, d, page)))
    ops().check_status(DEV)


LONG = [(1, 20000), (1, 300), (1, 7000), (1, 12345)]


@pytest.mark.parametrize("lengths", [LONG, [(1, 200), (1, 500)], [(40, 900), (1, 30)]])
def test_the_same_twice_on_streams_and_in_graphs(lengths, gen):
    """The same bits again, on another stream, on two streams at once, and from captured graphs that are replayed after other calls."""
    q, cache, table, ctx = problem(gen, lengths, 28, 4, 128, torch.bfloat16)
    q2 = (q.float() * 0.5).to(torch.bfloat16)

    def call(x):
        return ops().paged_attention_kv4(x, cache, table, ctx, 28, 4, 128, 16, 0.09)

    first, second = call(q), call(q2)
    assert torch.equal(call(q), first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, (stream, x) in enumerate(zip(streams, (q, q2))):
            with torch.cuda.stream(stream):
                outs[i].append(call(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs[0]) and all(torch.equal(o, second) for o in outs[1])
    graphs, results = [], []
    for x in (q, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(call(x))
        graphs.append(graph)
    for _ in range(3):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        call(q)
    torch.cuda.synchronize()
    assert torch.equal(results[0], first) and torch.equal(results[1], second)
    ops().check_status(DEV)


def test_a_captured_step_follows_its_lengths(gen):
    """A graph is captured for the longest context; replayed with shorter ones, and with requests that end inside a tile, it gives what a call gives."""
    q, cache, table, ctx = problem(gen, [(1, 9000), (1, 9000)], 8, 2, 128, torch.bfloat16, garbage=False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops().paged_attention_kv4(q, cache, table, ctx, 8, 2, 128, 16, 0.09)
    for starts in ([9000, 9000], [0, 8999], [17, 3], [5000, 0]):
        ctx.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        graph.replay()
        want = kv4_refs.attention64(q, cache, table, ctx.cu_q, ctx.q_start, 8, 2, 128, 16, 0.09)
        check_attention(out, want, cache, 128, f"replayed {starts} bfloat16")
    ops().check_status(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_and_attend_token_by_token(dtype, gen):
    """As a program uses them: portions and single tokens of two requests are stored and attend, step by step, and every result is what the stored
    rows give."""
    nq, nkv, d, page = 14, 2, 64, 16
    pages = 40
    cache = torch.full(kv4_shape(pages, nkv, page, d), 255, dtype=torch.uint8, device=DEV)
    table = torch.randperm(pages, generator=gen, device=DEV)[:24].view(2, 12).to(torch.int32)
    inv_freq = (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(DEV)
    bias = normal(gen, (nq + 2 * nkv) * d)
    done = [0, 0]
    for news in ([37, 5], [1, 1], [1, 20], [1, 1], [16, 1], [1, 1]):
        positions = torch.cat([torch.arange(s, s + n) for s, n in zip(done, news)]).to(torch.int32).to(DEV)
        owner = torch.repeat_interleave(torch.arange(2), torch.tensor(news)).to(DEV)
        slots = (table[owner, (positions // page).long()] * page + positions % page).to(torch.int32)
        projected = normal(gen, sum(news), (nq + 2 * nkv) * d)
        q = ops().qkv_rope_kv4(projected, bias, positions, inv_freq, d, slots, cache, nq, nkv, d, page, out_dtype=dtype)
        ctx = types.SimpleNamespace(cu_q=torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device=DEV), q_start=torch.tensor(done, dtype=torch.int32, device=DEV),
                                    max_q_len=max(news), max_ctx_len=max(a + b for a, b in zip(done, news)), host_lengths=news, host_starts=list(done))
        out, want = run_attention(q, cache, table, ctx, nq, nkv, d, page)
        check_attention(out, want, cache, d, f"step {news} {dtype}")
        done = [a + b for a, b in zip(done, news)]


# ---- the engine -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("C", "float32"), ("D", "bfloat16"), ("B", "bfloat16")])
def test_steps_of_a_model_match_the_plain_operations(name, dtype, tmp_path_factory):
    """Steps of portions and single tokens on the kernels against the same steps on plain operations, with the cache in 4 bits on both sides.

    32-bit activations differ by 1e-6: a number next to the border of two codes takes the other one once in ten thousand, which moves the logits
    by far less than 5 % of their spread.  bfloat16 ones differ by d = 2^-8 of a number and so; a code is then another one with probability 2 d / s
    (s the step, about 0.27 of the numbers' spread, a fifteenth of the range of 32 of them) and moves by s: a variance of 2 d s, which is below the s^2 / 12
    that the rounding to 4 bits itself has as long as d < s / 24 (0.011 of the spread; d is 0.004).  So what the logits move by is bounded by what 4 bits move
    them by, which the plain operations tell, beside the usual bar of bfloat16."""
    from flexengine_b200.cache import CacheManager
    from flexengine_b200.engine import ModelRunner
    from flexengine_b200.weights import load_model
    from helpers import CONFIGS, bf16_bar, make_model_dir
    folder = make_model_dir(tmp_path_factory, name)
    vocab = CONFIGS[name]["vocab_size"]
    runners = []
    for device, kind, operations, held in (("cpu", "float32", kv4_refs, "int4"), (DEV, dtype, None, "int4"), ("cpu", "float32", kv4_refs, "auto")):
        _cfg, plan, model = load_model(folder, kind, device)
        cache = CacheManager(plan.cache_groups, 24, 16, 4, getattr(torch, kind), device, kv_cache_dtype=held)
        runners.append(ModelRunner(model, cache, ops=operations))
    for step in ([("a", [(7 * i) % vocab for i in range(45)], [10, 44])], [("a", [3], [0]), ("b", [5, 6, 7], [2])], [("a", [9], [0]), ("b", [1], [0])],
                 [("b", [(5 * i) % vocab for i in range(20)], [0, 19])], [("a", [2], [0]), ("b", [8], [0])]):
        want, got, unrounded = (runner.step(step).float().cpu() for runner in runners)
        bar = 0.05 * float(want.std()) if dtype == "float32" else bf16_bar(want, name) + float((want - unrounded).abs().max())
        assert float((got - want).abs().max()) <= bar, step


def test_engine_with_graphs_top_p_and_min_p(tmp_path_factory):
    from flexengine_b200.config import EngineConfig
    from flexengine_b200.engine.runtime import Engine
    from helpers import make_model_dir
    folder = make_model_dir(tmp_path_factory, "D")

    def generate(**more):
        settings = dict(model=folder, device=DEV, dtype="float32", max_model_len=256, max_num_seqs=4, max_num_batched_tokens=64, prefill_chunk_size=64,
                        kv_block_size=16, kv_num_blocks=64, max_output_tokens=64, trace_steps=False, kv_cache_dtype="int4")
        asked = {k: more.pop(k) for k in ("temperature", "top_p", "min_p", "top_k", "seed") if k in more}
        settings.update(more)
        engine = Engine.from_model_dir(folder, EngineConfig(**settings))
        assert engine.cache.groups[0].storage.dtype == torch.uint8
        return [o.token_ids for o in engine.generate([[5, 6, 7] * 15, [9, 3], list(range(70))], max_tokens=20, **asked)]

    greedy = generate()
    assert generate(cuda_graph=True) == greedy and all(len(t) == 20 for t in greedy)
    drawn = generate(temperature=0.9, top_p=0.8, min_p=0.02, top_k=50, seed=4)
    assert generate(temperature=0.9, top_p=0.8, min_p=0.02, top_k=50, seed=4, cuda_graph=True) == drawn != greedy
    assert generate(temperature=0.9, top_p=1e-6, seed=4) == greedy
    with pytest.raises(ValueError, match="4-bit"):
        generate(kv_block_size=8, kv_num_blocks=128)


# ---- every way of dealing out a step's tiles ---------------------------------------------------------------------------------------
def deal_out(monkeypatch, plan, requests, nq, nkv, d):
    monkeypatch.setattr(ops(), "kv4_plan", lambda *a: (plan, int(ops()._kv4().fe_kv4_attention_scratch_bytes(max(plan, 0), requests, nq, nkv, d))))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", [-1, -2, -3, -4, -8, 1, 2, 7, 40, 296])
@pytest.mark.parametrize("nq,nkv,d", [(28, 4, 128), (20, 1, 96), (14, 2, 64)])
def test_every_plan(nq, nkv, d, plan, dtype, monkeypatch, gen):
    lengths = [(1, 1030), (0, 0), (1, 3), (1, 127), (1, 128), (0, 0), (1, 0), (1, 700), (0, 0)]
    args = problem(gen, lengths, nq, nkv, d, dtype)
    deal_out(monkeypatch, plan, len(lengths), nq, nkv, d)
    out, want = run_attention(*args, nq, nkv, d, 16)
    check_attention(out, want, args[1], d, f"plan {plan} {nq}/{nkv}/{d} {dtype}")
    out, want = run_attention(*args, nq, nkv, d, 16, window=100, keep_first=20)
    check_attention(out, want, args[1], d, f"plan {plan} window {nq}/{nkv}/{d} {dtype}")


@pytest.mark.parametrize("plan", [-1, -4, 1, 30])
def test_a_table_shorter_than_a_request(plan, monkeypatch, gen):
    """Positions that the table has no pages for: the keys that it has are seen, and the status word says so."""
    q, cache, table, ctx = problem(gen, [(1, 900), (1, 33)], 8, 2, 64, torch.bfloat16, garbage=False)
    deal_out(monkeypatch, plan, 2, 8, 2, 64)
    short = table[:, :20].contiguous()
    ctx.max_ctx_len = 320
    out = ops().paged_attention_kv4(q, cache, short, ctx, 8, 2, 64, 16, 0.125)
    with pytest.raises(RuntimeError, match="page id out of range"):
        ops().check_status(DEV)
    ctx.q_start[0] = 319
    want = kv4_refs.attention64(q, cache, short, ctx.cu_q, ctx.q_start, 8, 2, 64, 16, 0.125)
    check_attention(out, want, cache, 64, "a short table bfloat16")


@pytest.mark.parametrize("requests,tokens,nq,nkv", [(1, 500, 28, 4), (1, 4000, 28, 4), (1, 20000, 28, 4), (128, 700, 28, 4), (64, 1100, 28, 4), (64, 8192, 28, 4), (300, 40, 8, 8)])
@pytest.mark.parametrize("code", [0, 1])
def test_plans_are_ways_that_there_are(requests, tokens, nq, nkv, code):
    plan, scratch = ops().kv4_plan(requests, -(-tokens // 16), nq, nkv, 128, code)
    assert plan in (-1, -2, -4, -8) or plan > 0
    assert (scratch > 0) == (plan > 0)


# ---- NaN where a row's keys are shared out over blocks ---------------------------------------------------------------------------------
def nan_key(cache, table, d, r, place, head):
    """Makes a NaN of the scale of the first group of a stored key."""
    pairs = cache[..., 512 * kv4_refs.groups(d):576 * kv4_refs.groups(d)].view(torch.float16).view(cache.shape[:3] + (16, -1, 2))
    page = cache.shape[2] * 16
    pairs[int(table[r, place // page]), head, place % page // 16, place % 16, 0, 0] = math.nan


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", [-1, -2, -4, -8, 1, 7, 40, 296])
@pytest.mark.parametrize("where", ["query", "key", "newest key"])
def test_a_nan_score_reaches_its_rows_under_every_plan(where, plan, dtype, monkeypatch, gen):
    """A NaN in one query head makes NaN of its row, a NaN key of the rows of the heads that see it; the others are what they are without.
    The newest key of the first request is alone in its tile, and alone in a block's piece where 296 blocks share the tiles."""
    nq, nkv, d, lengths = 14, 2, 64, [(1, 1024), (1, 3), (1, 700)]
    q, cache, table, ctx = problem(gen, lengths, nq, nkv, d, dtype)
    deal_out(monkeypatch, plan, len(lengths), nq, nkv, d)
    want = kv4_refs.attention64(q, cache, table, ctx.cu_q, ctx.q_start, nq, nkv, d, 16, d ** -0.5).view(3, nq, d)
    bad = torch.zeros(3, nq, dtype=torch.bool)
    if where == "query":
        q[0, 5 * d + 9] = q[2, 13 * d] = math.nan
        bad[0, 5] = bad[2, 13] = True
    else:
        for r, place, head in ((0, 1024, 0), (2, 700, 1)) if where == "newest key" else ((0, 333, 0), (2, 0, 1)):
            nan_key(cache, table, d, r, place, head)
            bad[r, 7 * head:7 * head + 7] = True
    out = ops().paged_attention_kv4(q, cache, table, ctx, nq, nkv, d, 16, d ** -0.5).view(3, nq, d)
    ops().check_status(DEV)
    assert torch.equal(out.isnan().cpu(), bad[..., None].expand(3, nq, d))
    check_attention(out[~bad.to(DEV)], want[~bad], cache, d, f"beside a NaN, plan {plan} {dtype}")


def split_portions(monkeypatch, splits):
    monkeypatch.setattr(ops(), "kv4_portions", lambda *a, **k: 0)
    monkeypatch.setattr(ops(), "prefill_splits", lambda *a, **k: splits)


@pytest.mark.parametrize("splits", [1, 3, 8])
@pytest.mark.parametrize("nq,nkv,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("where", ["query", "key", "newest key"])
def test_a_nan_score_reaches_its_rows_in_split_portions(where, nq, nkv, d, splits, monkeypatch, gen):
    """As for single tokens: the keys of the tcgen05 kernel shared out over ``splits`` blocks.  The newest key of the first request is alone in its tile."""
    lengths, G = [(40, 985), (3, 130)], nq // nkv
    q, cache, table, ctx = problem(gen, lengths, nq, nkv, d, torch.bfloat16, page=32)
    split_portions(monkeypatch, splits)
    want = kv4_refs.attention64(q, cache, table, ctx.cu_q, ctx.q_start, nq, nkv, d, 32, d ** -0.5).view(43, nq, d)
    bad = torch.zeros(43, nq, dtype=torch.bool)
    if where == "query":
        q[3, 5 * d + 9] = q[39, 0] = q[42, 7 * d] = math.nan
        bad[3, 5] = bad[39, 0] = bad[42, 7] = True
    elif where == "key":
        nan_key(cache, table, d, 0, 333, 0)
        nan_key(cache, table, d, 1, 131, 1)
        bad[:40, :G] = True
        bad[41:, G:] = True
    else:
        nan_key(cache, table, d, 0, 1024, 1)
        bad[39, G:] = True
    out = ops().paged_attention_kv4(q, cache, table, ctx, nq, nkv, d, 32, d ** -0.5).view(43, nq, d)
    ops().check_status(DEV)
    assert torch.equal(out.isnan().cpu(), bad[..., None].expand(43, nq, d))
    check_attention(out[~bad.to(DEV)], want[~bad], cache, d, f"beside a NaN, {splits} splits bfloat16")


@pytest.mark.parametrize("splits", [1, 4])
def test_a_nan_query_keeps_its_row_in_split_portions_over_a_16_bit_cache(splits, gen):
    """The same kernel over keys and values of 16 bits."""
    nq, nkv, d, pages = 8, 2, 64, 70
    k, v = (normal(gen, pages, nkv, 16, d).to(torch.bfloat16) for _ in range(2))
    q = normal(gen, 20, nq * d).to(torch.bfloat16)
    table = torch.arange(pages, device=DEV, dtype=torch.int32)[None]
    cu, start = torch.tensor([0, 20], dtype=torch.int32, device=DEV), torch.tensor([1090], dtype=torch.int32, device=DEV)

    def call():
        return ops().paged_prefill_tcgen05(q, q.stride(0), k, v, table, cu, start, 20, 1, 20, nq, nkv, d, 16, 0.125, 0, splits).view(20, nq, d)

    clean = call()
    q[7, 3 * d + 1] = math.nan
    out = call()
    ops().check_status(DEV)
    bad = torch.zeros(20, nq, d, dtype=torch.bool, device=DEV)
    bad[7, 3] = True
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad], clean[~bad])


def nan_value(cache, table, d, r, place, head, group):
    """Makes a NaN of the scale of one group of a stored value."""
    n, page = kv4_refs.groups(d), cache.shape[2] * 16
    pairs = cache[..., 576 * n:].view(torch.float16).view(cache.shape[:3] + (16, n, 2))
    pairs[int(table[r, place // page]), head, place % page // 16, place % 16, group, 0] = math.nan


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", [-1, -2, -4, -8, 1, 7, 40, 296])
@pytest.mark.parametrize("place", [0, 150, 517, 1024])
def test_a_nan_value_reaches_rows_in_which_its_weight_is_nothing(place, plan, dtype, monkeypatch, gen):
    """Scores hundreds apart: all but one key of a row weigh 0 in 32 bits, also where blocks' results are put together.  0 times NaN is NaN."""
    nq, nkv, d = 14, 2, 64
    q, cache, table, ctx = problem(gen, [(1, 1024), (1, 40)], nq, nkv, d, dtype)
    q = (q.float() * 500).to(dtype)
    deal_out(monkeypatch, plan, 2, nq, nkv, d)
    nan_value(cache, table, d, 0, place, 1, 1)
    out = ops().paged_attention_kv4(q, cache, table, ctx, nq, nkv, d, 16, d ** -0.5).view(2, nq, d)
    bad = torch.zeros(2, nq, d, dtype=torch.bool)
    bad[0, 7:, 32:] = True
    assert torch.equal(out.isnan().cpu(), bad)


@pytest.mark.parametrize("splits", [1, 3, 8])
@pytest.mark.parametrize("place", [0, 150, 517, 1020])
def test_a_nan_value_reaches_rows_in_which_its_weight_is_nothing_in_split_portions(place, splits, monkeypatch, gen):
    nq, nkv, d = 8, 2, 128
    q, cache, table, ctx = problem(gen, [(40, 985)], nq, nkv, d, torch.bfloat16)
    q = (q.float() * 500).to(torch.bfloat16)
    split_portions(monkeypatch, splits)
    nan_value(cache, table, d, 0, place, 1, 2)
    out = ops().paged_attention_kv4(q, cache, table, ctx, nq, nkv, d, 16, d ** -0.5).view(40, nq, d)
    bad = torch.zeros(40, nq, d, dtype=torch.bool)
    bad[max(0, place - 985):, 4:, 64:96] = True
    assert torch.equal(out.isnan().cpu(), bad)


@pytest.mark.parametrize("plan", [-1, -8, 40])
@pytest.mark.parametrize("nq,nkv,d", [(4, 1, 64), (7, 1, 128)])
def test_32_bits_hold_over_a_long_walk(nq, nkv, d, plan, monkeypatch, gen):
    """32,768 keys of about the same weight under 32-bit queries, walked by one block, by eight, and shared out.

    Relative to the result's norm (about sqrt(n) of n keys' numbers, as the errors of single weights are): a weight is off by its score (a few
    roundings of 2^-24 of numbers up to 8 in log2 units: 5e-7), its exponential (2^-22) and its two halves (2^-22), some 6e-7 in all; a warp's
    running sums take up to 512 pairs of products, each with a rounding of 2^-25 on average, sqrt(512 / 2) 2^-25 = 5e-7.  3e-6 is three times as much as
    the two.  Sums that are cut off instead of rounded at every addition would be off by 512 times 2^-24 or 3e-5."""
    args = problem(gen, [(1, 32767)], nq, nkv, d, torch.float32, garbage=False)
    args = (args[0] * 0.15,) + args[1:]
    deal_out(monkeypatch, plan, 1, nq, nkv, d)
    out, want = run_attention(*args, nq, nkv, d, 16)
    off = float((out.cpu().double() - want).norm() / want.norm())
    assert off <= 3e-6, f"{off:.2e} of the norm"


# ---- a wait that runs out ----------------------------------------------------------------------------------------------------------
@pytest.fixture()
def short_waits():
    """Copies that are said to bring 16 bytes more than they do, so that every wait for them runs out after some 50 us, as long as the test lasts."""
    libraries = [ops()._kv4(), ops()._bf16()]
    for library in libraries:
        library.fe_set_waits(100000, 16)
    yield
    for library in libraries:
        library.fe_set_waits(0, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", [-1, -4, 1, 7, 40])
def test_a_wait_that_runs_out_is_reported_by_single_tokens(plan, dtype, monkeypatch, gen, request):
    q, cache, table, ctx = problem(gen, [(1, 1030), (1, 3), (1, 700)], 14, 2, 64, dtype)
    deal_out(monkeypatch, plan, 3, 14, 2, 64)
    request.getfixturevalue("short_waits")
    ops().paged_attention_kv4(q, cache, table, ctx, 14, 2, 64, 16, 0.125)
    with pytest.raises(RuntimeError, match="wait"):
        ops().check_status(DEV)
    for library in (ops()._kv4(), ops()._bf16()):
        library.fe_set_waits(0, 0)
    out, want = run_attention(q, cache, table, ctx, 14, 2, 64, 16)          # the device is as it was
    check_attention(out, want, cache, 64, f"after a wait that ran out, plan {plan} {dtype}")


@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("nq,nkv,d", [(14, 2, 64), (8, 2, 128)])
def test_a_wait_that_runs_out_is_reported_by_portions(nq, nkv, d, splits, monkeypatch, gen, request):
    q, cache, table, ctx = problem(gen, [(40, 985), (3, 130)], nq, nkv, d, torch.bfloat16)
    split_portions(monkeypatch, splits)
    request.getfixturevalue("short_waits")
    ops().paged_attention_kv4(q, cache, table, ctx, nq, nkv, d, 16, 0.125)
    with pytest.raises(RuntimeError, match="wait"):
        ops().check_status(DEV)
    for library in (ops()._kv4(), ops()._bf16()):
        library.fe_set_waits(0, 0)
    out, want = run_attention(q, cache, table, ctx, nq, nkv, d, 16)
    check_attention(out, want, cache, d, "after a wait that ran out bfloat16")


def test_a_wait_that_runs_out_is_reported_by_the_store(gen, request):
    """Enough tokens for the blocks that fetch rows by bulk copies."""
    T, nq, nkv, d = 700, 2, 2, 64
    projected = normal(gen, T, 6 * d)
    slots, positions = torch.arange(T, device=DEV, dtype=torch.int32), torch.zeros(T, device=DEV, dtype=torch.int32)
    caches = [torch.zeros(kv4_shape(44, nkv, 16, d), dtype=torch.uint8, device=DEV) for _ in range(2)]

    def store(cache):
        return ops().qkv_rope_kv4(projected, None, positions, None, 0, slots, cache, nq, nkv, d, 16)

    want = store(caches[0])
    ops().check_status(DEV)
    request.getfixturevalue("short_waits")
    store(caches[1])
    with pytest.raises(RuntimeError, match="wait"):
        ops().check_status(DEV)
    ops()._kv4().fe_set_waits(0, 0)
    assert torch.equal(store(caches[1]), want) and torch.equal(caches[0], caches[1])
    ops().check_status(DEV)


def test_special_numbers_leave_nan_where_they_were_and_nowhere_else(gen):
    """NaN among the keys and among the values, in groups of their own: the group reads as NaN, whole, and no other."""
    x = normal(gen, 7, 4, 64)
    x[0], x[1, :, 3], x[2, :, 40] = 2.5, 1e30, -math.inf
    x[4, 2, 50] = x[5, 3, 7] = x[6, 3, 63] = math.nan
    x[3, 1, 7] = math.nan                                  # of a query
    cache = torch.full(kv4_shape(2, 1, 16, 64), 255, dtype=torch.uint8, device=DEV)
    slots = torch.arange(3, 10, dtype=torch.int32, device=DEV)
    q = ops().qkv_rope_kv4(x.reshape(7, -1), None, torch.zeros(7, dtype=torch.int32, device=DEV), None, 0, slots, cache, 2, 1, 64, 16)
    ops().check_status(DEV)
    keys, values = ops().kv4_rows(cache, slots, 1, 64, 16, torch.float32)
    bad = torch.zeros(2, 7, 1, 64, dtype=torch.bool, device=DEV)
    bad[0, 4, 0, 32:] = bad[1, 5, 0, :32] = bad[1, 6, 0, 32:] = True
    assert torch.equal(keys.isnan(), bad[0]) and torch.equal(values.isnan(), bad[1])
    assert q.isnan().nonzero().tolist() == [[3, 64 + 7]]


@pytest.mark.parametrize("T,pairs,d,rot", [(2048, "halves", 128, 128), (100, "halves", 128, 128), (1500, "interleaved", 64, 32), (700, "halves", 80, 20)])
def test_codes_next_to_a_border_are_the_formula_s(T, pairs, d, rot, gen):
    """Bias, rotation and rounding step by step in 32 bits, every operation rounded by itself, sines and cosines from 64 bits: the same pairs and the same
    codes, all of them (some three million; a border is met within 2^-22 of a step a few times)."""
    nq, nkv, page = 8, 8, 16
    width = (nq + 2 * nkv) * d
    projected = normal(gen, T, width) * torch.where(torch.rand(width, generator=gen, device=DEV) < 0.05, 6.0, 1.0)
    bias = normal(gen, width)
    positions = torch.arange(T, device=DEV, dtype=torch.int32) * 13
    inv_freq = (1e6 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)).float().to(DEV)
    cache = torch.zeros(kv4_shape(-(-T // page), nkv, page, d), dtype=torch.uint8, device=DEV)
    slots = torch.arange(T, device=DEV, dtype=torch.int32)
    q = ops().qkv_rope_kv4(projected, bias, positions, inv_freq, rot, slots, cache, nq, nkv, d, page, pairs=pairs)
    x = (projected.cpu() + bias.cpu()).view(T, nq + 2 * nkv, d)
    angle = positions.cpu().double()[:, None, None] * inv_freq.cpu().double()
    cos, sin = angle.cos().float(), angle.sin().float()
    i = torch.arange(rot // 2)
    a, b = (i, i + rot // 2) if pairs == "halves" else (2 * i, 2 * i + 1)
    turned = x[:, :nq + nkv].clone()
    turned[..., a], turned[..., b] = x[:, :nq + nkv, a] * cos - x[:, :nq + nkv, b] * sin, x[:, :nq + nkv, b] * cos + x[:, :nq + nkv, a] * sin
    assert torch.equal(q.cpu(), turned[:, :nq].flatten(1))
    for got, want in zip(kv4_refs.read_rows(cache, slots, d), (turned[:, nq:], x[:, nq + nkv:])):
        for first in range(0, d, 32):
            w = want[..., first:first + 32]
            low, high = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
            scale = ((high - low) * torch.tensor(1 / 15)).half().float()          # by a fifteenth as 32 bits hold it
            centre = (low + 8 * scale).half().float()
            code = (torch.round((w - centre) / scale) + 8).clamp(0, 15)
            assert torch.equal(got[..., first:first + 32], centre.double() + (code.double() - 8) * scale.double())
