"""Sampling with top-p and min-p on the device against the plain form in 64 bits: tokens and the numbers that stay have to be equal."""
import math

import pytest
import torch

import kv4_refs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from flexengine_b200 import ops as cuda_ops
    return cuda_ops


def rows(seed, R, V, **more):
    g = torch.Generator(device=DEV).manual_seed(seed)
    at = torch.arange(R, device=DEV)
    logits = torch.randn(R, V, generator=g, device=DEV) * (0.3 + 4 * torch.rand(R, 1, generator=g, device=DEV))
    logits += torch.where(torch.rand(R, V, generator=g, device=DEV) < 16 / V, 6.0, 0.0)
    given = dict(logits=logits, temperature=torch.where(at % 9 == 8, 0.0, 0.3 + 0.2 * (at % 7)).float(),
                 top_k=torch.where(at % 3 == 1, 40, torch.where(at % 7 == 2, V // 3, 0)).to(torch.int32),
                 top_p=torch.where(at % 5 == 4, 1.0, 0.5 + 0.12 * (at % 4)).float(), min_p=torch.where(at % 4 == 2, 0.03, 0.0).float(),
                 uniform=torch.rand(R, generator=g, device=DEV))
    given.update(more)
    return given


def check(given, blocks=(0, 1, 2, 4, 8), what=""):
    want = kv4_refs.sample_filtered(**given)
    for b in blocks:
        got = ops().sample_filtered(**given, blocks=b)
        assert torch.equal(got[0], want[0]), f"{what} blocks {b}: tokens {(got[0] != want[0]).nonzero().flatten().tolist()}"
        assert torch.equal(got[2], want[2]), f"{what} blocks {b}: numbers that stay"
        # exponentials of 32 bits (2 units in the last place each), one quotient rounded
        torch.testing.assert_close(got[1], want[1], rtol=1e-6, atol=0.0)


@pytest.mark.parametrize("V", [1, 2, 3, 31, 257, 1000, 4099, 32003, 50257, 152064])
def test_vocabularies(V):
    check(rows(V, 12 if V > 40000 else 40, V), what=f"V {V}")


@pytest.mark.parametrize("R", [1, 5, 17, 40, 150])
def test_row_counts_choose_how_many_blocks_share_a_row(R):
    check(rows(R, R, 2048), blocks=(0,), what=f"R {R}")


def full(value, like, dtype=None):
    return torch.full_like(like, value) if dtype is None else torch.full(like.shape, value, dtype=dtype, device=DEV)


CASES = {
    "equal logits": lambda g: dict(logits=torch.zeros_like(g["logits"])),
    "16-bit logits": lambda g: dict(logits=g["logits"].bfloat16().float()),
    "few values": lambda g: dict(logits=(g["logits"] * 2).round() / 2),
    "k one": lambda g: dict(top_k=full(1, g["top_k"])),
    "k all but one": lambda g: dict(top_k=full(g["logits"].shape[1] - 1, g["top_k"])),
    "k of all": lambda g: dict(top_k=full(g["logits"].shape[1], g["top_k"])),
    "k beyond": lambda g: dict(top_k=full(2 ** 31 - 1, g["top_k"])),
    "k below zero": lambda g: dict(top_k=full(-3, g["top_k"])),
    "k large": lambda g: dict(top_k=full(3001, g["top_k"])),
    "cold": lambda g: dict(temperature=full(0.02, g["temperature"]), top_k=full(100, g["top_k"])),
    "hot": lambda g: dict(temperature=full(5.0, g["temperature"])),
    "p next to nothing": lambda g: dict(top_p=full(1e-9, g["top_p"])),
    "p nothing": lambda g: dict(top_p=full(0.0, g["top_p"])),
    "p next to one": lambda g: dict(top_p=full(1 - 2.0 ** -20, g["top_p"])),
    "p beyond one": lambda g: dict(top_p=full(1.5, g["top_p"])),
    "min_p alone": lambda g: dict(top_p=full(1.0, g["top_p"]), top_k=full(0, g["top_k"]), min_p=full(0.2, g["min_p"])),
    "min_p one": lambda g: dict(min_p=full(1.0, g["min_p"])),
    "min_p tiny": lambda g: dict(top_p=full(1.0, g["top_p"]), min_p=full(1e-20, g["min_p"])),
    "no limit": lambda g: dict(top_p=full(1.0, g["top_p"]), top_k=full(0, g["top_k"]), min_p=full(0.0, g["min_p"])),
    "greedy": lambda g: dict(temperature=full(0.0, g["temperature"])),
    "ends of the numbers": lambda g: dict(uniform=torch.where(torch.arange(len(g["uniform"]), device=DEV) % 2 == 0, 0.0, 1 - 2.0 ** -24)),
    "numbers outside": lambda g: dict(uniform=torch.where(torch.arange(len(g["uniform"]), device=DEV) % 2 == 0, -1.0, 2.0)),
}


@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("V", [777, 20011])
def test_settings(name, V):
    given = rows(7, 24, V)
    given.update(CASES[name](given))
    check(given, blocks=(0, 1, 4), what=name)


def test_masked_and_special_logits():
    given = rows(3, 20, 5003)
    x = given["logits"]
    x[:, ::2] = -math.inf
    x[:, 1::4] = torch.finfo(torch.float32).min
    x[0] = -math.inf                                   # nothing is left: token 0 with no probability
    x[1] = math.nan
    x[2, 4001] = math.inf
    x[3, 17] = x[3, 4999] = math.inf
    x[4, ::3] = math.nan
    x[5, 0] = 3e38
    x[6] = -math.inf
    x[6, 1234] = -5.0
    check(given)
    tokens, probability, kept = ops().sample_filtered(**given)
    assert tokens[:2].tolist() == [0, 0] and probability[:2].tolist() == [0.0, 0.0] and kept[:2].tolist() == [0, 0]


def test_strides_alignment_and_streams():
    given = rows(5, 9, 3001)
    wide = torch.zeros(9, 3011, device=DEV)
    wide[:, 5:3006] = given["logits"]
    want = ops().sample_filtered(**given)
    moved = dict(given, logits=wide[:, 5:3006])
    assert all(torch.equal(a, b) for a, b in zip(ops().sample_filtered(**moved), want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ops().sample_filtered(**given)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops().sample_filtered(**given)
    given["uniform"].copy_(given["uniform"].flip(0))
    graph.replay()
    again = ops().sample_filtered(**given)
    assert all(torch.equal(a, b) for a, b in zip(held, again))
    empty = {k: v[:0] for k, v in given.items()}
    assert [t.shape for t in ops().sample_filtered(**empty)] == [(0,)] * 3


def test_refusals():
    given = rows(5, 3, 64)
    with pytest.raises(RuntimeError, match="blocks a row"):
        ops().sample_filtered(**given, blocks=3)
    with pytest.raises(ValueError, match="tensors on"):
        ops().sample_filtered(**dict(given, uniform=given["uniform"].cpu()))


def test_draws_follow_the_distribution():
    """50,000 draws from one row: the frequencies of the tokens that stay lie within five standard deviations of their probabilities."""
    V, n = 40, 50000
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(V, generator=g, device=DEV) * 1.5
    given = dict(logits=x.expand(n, V).contiguous(), temperature=torch.full((n,), 0.8, device=DEV), top_k=torch.full((n,), 20, dtype=torch.int32, device=DEV),
                 top_p=torch.full((n,), 0.9, device=DEV), min_p=torch.full((n,), 0.02, device=DEV), uniform=torch.rand(n, generator=g, device=DEV))
    tokens, probability, kept = ops().sample_filtered(**given)
    counts = torch.bincount(tokens.long(), minlength=V).double()
    chance = torch.zeros(V, dtype=torch.float64, device=DEV)
    chance[tokens.long()] = probability.double()
    assert abs(float(chance.sum()) - 1) < 1e-5 and int((counts > 0).sum()) == int(kept[0])
    assert ((counts - n * chance).abs() <= 5 * torch.sqrt(n * chance * (1 - chance)) + 1).all()


def test_sampler_on_the_device_is_the_plain_one():
    from flexengine_b200.sampling import Sampler
    g = torch.Generator(device=DEV).manual_seed(2)
    logits = torch.randn(9, 3000, generator=g, device=DEV) * 3
    heats, ks, seeds, draws = [0.0, 0.7, 1.3, 0.9, 1.0, 0.9, 0.0, 2.0, 0.5], [0, 5, 0, 3, 40, 0, 0, 7, 0], list(range(9)), list(range(5, 14))
    top_ps, min_ps = [0.5, 1.0, 0.8, 1.0, 0.9, 1.0, 1.0, 0.3, 0.95], [0.0, 0.0, 0.0, 0.1, 0.01, 0.2, 0.5, 0.0, 0.0]
    got = Sampler().sample(logits, heats, ks, seeds, draws, top_ps, min_ps)
    assert got == Sampler(kv4_refs).sample(logits, heats, ks, seeds, draws, top_ps, min_ps)


@pytest.mark.parametrize("top_p,top_k", [(1.0, 0), (0.5, 0), (1.0, 100), (0.5, 100)])
def test_an_infinite_temperature_leaves_the_finite_logits_alike(top_p, top_k):
    R, V = 6, 1000
    given = rows(3, R, V)
    given["logits"][:, ::2] = -math.inf
    given["logits"][:, 5] = math.nan
    given.update(temperature=full(math.inf, given["temperature"]), top_p=full(top_p, given["top_p"]), top_k=full(top_k, given["top_k"]), min_p=full(0.0, given["min_p"]))
    n = 100 if top_k else V // 2 - 1
    n = math.ceil(n * top_p)
    for blocks in (1, 2, 8):
        tokens, probability, kept = ops().sample_filtered(**given, blocks=blocks)
        assert given["logits"].gather(1, tokens.long()[:, None]).isfinite().all()
        assert kept.tolist() == [n] * R
        torch.testing.assert_close(probability, torch.full_like(probability, 1 / n), rtol=1e-6, atol=0.0)


def levels(distance, numbers, seed):
    """A row of few different logits, ``distance`` apart, ``numbers`` of each in a random order; and the shares of the mass that the first levels hold."""
    g = torch.Generator().manual_seed(seed)
    x = torch.cat([torch.full((n,), -distance * j) for j, n in enumerate(numbers)])
    x = x[torch.randperm(len(x), generator=g)]
    held = torch.tensor([n * math.exp(float(torch.tensor(-distance * j).double())) for j, n in enumerate(numbers)], dtype=torch.float64)
    return x.to(DEV), (held.cumsum(0) / held.sum()).tolist()


@pytest.mark.parametrize("distance", [1.003, 1.0052, 0.6931])
def test_a_limit_next_to_the_border_of_far_apart_logits(distance):
    """Thousands of equal logits in each of a few steps far apart, and top-p next to the mass of the first of them: the coarse sums (13 bits a token)
    take the limit to lie on one side of the border or the other, and the exact ones decide.  Nothing lies in the steps between: they
    are not gone through one by one, so that such a row takes no more than a few walks longer than one whose limit lies well inside a level."""
    x, shares = levels(distance, [3000, 5000, 4000, 6000, 3500], 1)
    for blocks in (1, 8):
        slow, usual = 0.0, 0.0
        for level in range(4):
            for off in (-3e-5, -3e-6, -4e-7, 4e-7, 3e-6, 3e-5, 0.03):
                p = shares[level] * (1 + off)
                given = dict(logits=x[None].contiguous(), temperature=torch.ones(1, device=DEV), top_k=torch.zeros(1, dtype=torch.int32, device=DEV),
                             top_p=torch.tensor([p], device=DEV), min_p=torch.zeros(1, device=DEV), uniform=torch.tensor([0.3], device=DEV))
                check(given, blocks=(blocks,), what=f"level {level} off {off}")
                times = []
                for _ in range(7):
                    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    torch.cuda.synchronize()
                    a.record()
                    ops().sample_filtered(**given, blocks=blocks)
                    b.record()
                    torch.cuda.synchronize()
                    times.append(a.elapsed_time(b))
                t = sorted(times)[3]
                if off == 0.03:
                    usual = max(usual, t)
                else:
                    slow = max(slow, t)
        assert slow <= 3 * usual, f"{blocks} blocks: {1000 * slow:.0f} us against {1000 * usual:.0f}"
