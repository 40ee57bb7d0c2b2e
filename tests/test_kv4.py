"""A cache held in 4 bits and sampling with top-p and min-p without a GPU: sizes, settings, refusals, and the engine on plain operations."""
import types

import numpy as np
import pytest
import torch

import kernel_refs
import kv4_refs
from flexengine_b200.cache import CacheManager
from flexengine_b200.cache.manager import kv4_row_bytes, kv4_shape
from flexengine_b200.cli.generate import build_parser, engine_config_from_args
from flexengine_b200.config import EngineConfig
from flexengine_b200.engine.runtime import Engine, check_kv4, pages_that_fit
from flexengine_b200.parts.spec import CacheGroupSpec
from flexengine_b200.sampling import Sampler
from flexengine_b200.sampling.sampler import uniforms
from helpers import make_model_dir


# ---- the form --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,groups", [(16, 1), (32, 1), (48, 2), (64, 2), (80, 3), (128, 4), (256, 8)])
def test_sizes(d, groups):
    assert kv4_row_bytes(d) == 40 * groups
    assert kv4_shape(3, 2, 32, d) == (3, 2, 2, 640 * groups)
    every = kv4_refs.places(d, True)
    assert len(set(every.tolist())) == d and int(every.max()) < 32 * groups
    every = kv4_refs.places(d, False)
    assert len(set(every.tolist())) == d and int(every.max()) < 32 * groups


@pytest.mark.parametrize("d", [0, 8, 24, 272])
def test_head_sizes_that_are_refused(d):
    with pytest.raises(ValueError, match="head size"):
        kv4_row_bytes(d)


@pytest.mark.parametrize("page", [1, 8, 15, 24])
def test_page_sizes_that_are_refused(page):
    with pytest.raises(ValueError, match="multiple of 16"):
        kv4_shape(3, 2, page, 64)
    with pytest.raises(ValueError, match="multiple of 16"):
        EngineConfig(kv_block_size=page, kv_num_blocks=10000, kv_cache_dtype="int4")
    EngineConfig(kv_block_size=page, kv_num_blocks=10000)                  # other caches take any


def test_rows_come_back_within_half_a_step():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(7, 3, 80, generator=gen) * torch.tensor([1e-4, 1.0, 3e3])[:, None]
    x[0, 0, 5], x[1, 1, 40] = 1e9, -np.inf                                 # stored as +-61440
    x[2, 2, 70] = np.nan
    cache = torch.full(kv4_shape(2, 3, 16, 80), 255, dtype=torch.uint8)
    slots = torch.tensor([3, 31, 16, 0, -1, 7, 15], dtype=torch.int32)
    kv4_refs.write_rows(cache, slots, x, -x)
    for side, sign in zip(kv4_refs.read_rows(cache, slots, 80), (1, -1)):
        for t in range(7):
            want = (sign * x[t].double()).clamp(-61440, 61440)
            if slots[t] < 0:
                assert (side[t] == 0).all()
                continue
            for first in (0, 32, 64):
                got, w = side[t, :, first:first + 32], want[:, first:first + 32]
                for h in range(3):
                    if w[h].isnan().any():
                        assert got[h].isnan().all()
                        continue
                    # half a step, and what rounding the scale (times 8 at the ends) and the centre to half precision adds
                    step = float(w[h].max() - w[h].min()) / 15
                    slack = step / 2 + 8 * (step * 2 ** -11 + 2 ** -25) + float(w[h].abs().max()) * 2 ** -10 + 2 ** -24
                    assert float((got[h] - w[h]).abs().max()) <= slack, (t, h, first)


# ---- cache manager and engine settings -------------------------------------------------------------------------------------
def spec(**more):
    return CacheGroupSpec("keys", more.pop("kind", "full"), slots=3, kv_heads=2, head_dim=64, **more)


def test_manager_keeps_tiles():
    cache = CacheManager([spec(), CacheGroupSpec("s", "state", slots=1, state_shape=(4,))], 6, 32, 2, torch.bfloat16, "cpu", kv_cache_dtype="int4")
    group = cache.groups[0]
    assert group.four_bit and group.storage.dtype == torch.uint8 and tuple(group.storage.shape) == (3, 6, 2, 2, 1280)
    assert group.bytes_per_token() == 3 * 2 * 80
    assert group.storage.numel() == group.bytes_per_token() * 6 * 32
    with pytest.raises(TypeError, match="4 bits"):
        group.kv_slot(0)
    cache.reserve("a", 40)
    cache.commit("a", 40)
    assert cache.slot_mapping("a", 0, 33, 2) == [33, 34]
    cache.free("a")
    cache.assert_invariants()
    plain = CacheManager([spec()], 6, 32, 2, torch.bfloat16, "cpu")
    assert not plain.groups[0].four_bit and plain.groups[0].storage.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        CacheManager([spec()], 6, 32, 2, torch.bfloat16, "cpu", kv_cache_dtype="int2")


def test_settings():
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineConfig(kv_cache_dtype="int3")
    args = build_parser().parse_args(["--model", "m", "--kv-cache-dtype", "int4", "--top-p", "0.9", "--min-p", "0.05"])
    assert engine_config_from_args(args).kv_cache_dtype == "int4" and args.top_p == 0.9 and args.min_p == 0.05


def test_pages_that_fit_counts_four_bits(monkeypatch):
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (1 << 20, 1 << 20))
    plan = types.SimpleNamespace(cache_groups=[spec()])
    settings = dict(device="cuda:0", max_model_len=64, kv_block_size=16, kv_num_blocks=0, kv_memory_fraction=1.0)
    assert pages_that_fit(plan, EngineConfig(**settings, kv_cache_dtype="int4"), torch.bfloat16) == (1 << 20) // (3 * 2 * 80 * 16)
    assert pages_that_fit(plan, EngineConfig(**settings), torch.bfloat16) == (1 << 20) // (3 * 2 * 64 * 2 * 2 * 16)


def plan_of(kind, group):
    return types.SimpleNamespace(cache_groups=[group], layers=[types.SimpleNamespace(mixer=types.SimpleNamespace(kind=kind))],
                                 run=[types.SimpleNamespace(layer=0, cache_group=0, more=())])


def test_mixers_that_do_not_read_four_bits_are_refused():
    check_kv4(plan_of("attention", spec()))
    check_kv4(plan_of("attention", spec(kind="window", window=8)))
    for kind, group in (("gated_attention", spec()), ("latent_attention", spec(planes=1)), ("attention", spec(planes=1)),
                        ("attention", spec(kind="chunk", window=8))):
        with pytest.raises(ValueError, match="does not read a 4-bit cache"):
            check_kv4(plan_of(kind, group))
    check_kv4(plan_of("gated_attention", CacheGroupSpec("s", "state", slots=1, state_shape=(4,))))


# ---- the engine on plain operations ------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def model_a(tmp_path_factory):
    return make_model_dir(tmp_path_factory, "A")


def engine_of(model_dir, ops=kv4_refs, **more):
    settings = dict(model=model_dir, device="cpu", dtype="float32", max_model_len=128, max_num_seqs=4, max_num_batched_tokens=48,
                    prefill_chunk_size=48, kv_block_size=16, kv_num_blocks=40, max_output_tokens=32, trace_steps=False, kv_cache_dtype="int4")
    settings.update(more)
    return Engine.from_model_dir(model_dir, EngineConfig(**settings), ops=ops)


def test_engine_generates_from_a_four_bit_cache(model_a):
    prompts = [list(range(60, 90)), [7, 200] * 9, [3]]
    whole = [o.token_ids for o in engine_of(model_a).generate(prompts, max_tokens=6)]
    cut = [o.token_ids for o in engine_of(model_a, max_num_batched_tokens=7, prefill_chunk_size=7).generate(prompts, max_tokens=6)]
    assert whole == cut and all(len(ids) == 6 for ids in whole)
    # near what 16 bits a number give: the logits of the first sampled token agree to a few hundredths of their spread
    first = [engine_of(model_a, kv_cache_dtype=kind).runner.step([("r", prompts[0], [29])]) for kind in ("int4", "auto")]
    assert float((first[0] - first[1]).std()) < 0.2 * float(first[1].std())
    assert float((first[0] - first[1]).abs().max()) > 0.0


def test_requests_ask_for_top_p_and_min_p(model_a):
    engine = engine_of(model_a)
    for wrong in (dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=1.5), dict(top_p=float("nan"))):
        with pytest.raises(ValueError, match="top_p|min_p"):
            engine.submit([1], max_tokens=4, temperature=1.0, **wrong)
    prompts = [[5, 6, 7], [9] * 20, [1]]
    alone = [engine_of(model_a).generate([p], max_tokens=5, temperature=1.0, top_p=0.7, min_p=0.02, seed=11 + i)[0].token_ids
             for i, p in enumerate(prompts)]
    together = engine_of(model_a, max_num_batched_tokens=6).generate(prompts, max_tokens=5, temperature=1.0, top_p=0.7, min_p=0.02, seed=11)
    assert [o.token_ids for o in together] == alone
    # a nucleus of next to nothing is the likeliest token
    greedy = engine_of(model_a).generate([prompts[0]], max_tokens=5)[0].token_ids
    assert engine_of(model_a).generate([prompts[0]], max_tokens=5, temperature=1.0, top_p=1e-6, seed=3)[0].token_ids == greedy


# ---- the sampler -----------------------------------------------------------------------------------------------------------
def test_uniforms_are_the_kernel_s():
    seeds, draws = [0, 1, 42, 2 ** 63 - 1, -5], [0, 7, 1000, 3, 2]
    assert uniforms(seeds, draws).tolist() == [np.float32(kernel_refs.uniform_from(s, d)) for s, d in zip(seeds, draws)]


def test_neighbours_with_other_settings_change_nothing():
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(6, 300, generator=gen) * 3
    heats, ks, seeds, draws = [0.0, 0.7, 1.3, 0.0, 1.0, 0.9], [0, 5, 0, 3, 40, 0], [1, 2, 3, 4, 5, 6], [0, 1, 2, 3, 4, 5]
    top_ps, min_ps = [0.5, 1.0, 0.8, 1.0, 0.9, 1.0], [0.0, 0.0, 0.0, 0.1, 0.01, 0.2]
    sampler = Sampler(kv4_refs)
    together = sampler.sample(logits, heats, ks, seeds, draws, top_ps, min_ps)
    for i in range(6):
        one = [[v[i]] for v in (heats, ks, seeds, draws, top_ps, min_ps)]
        assert sampler.sample(logits[i:i + 1], *one) == [together[i]]
    plain = sampler.sample(logits, heats, ks, seeds, draws)
    for i in (0, 1, 3):                                                    # greedy, or neither limit: as without the two
        assert together[i] == plain[i]
    assert sampler.sample(logits, heats, ks, seeds, draws, [1.0] * 6, None) == plain


def test_sampler_refuses():
    sampler, logits = Sampler(kv4_refs), torch.zeros(2, 8)
    for more in (dict(top_ps=[0.0, 1.0]), dict(top_ps=[2.0, 1.0]), dict(min_ps=[-1.0, 0.0]), dict(min_ps=[0.0, float("nan")])):
        with pytest.raises(ValueError, match="top_p|min_p"):
            sampler.sample(logits, [1.0, 1.0], [0, 0], [1, 2], [0, 0], **more)
    with pytest.raises(ValueError, match="a row"):
        sampler.sample(logits, [1.0, 1.0], [0, 0], [1, 2], [0, 0], top_ps=[0.5])


# ---- what the operators refuse, before anything is launched -------------------------------------------------------------------
@pytest.fixture()
def unlaunched(monkeypatch):
    """The operators with CPU tensors let through, and a launch that fails the test."""
    from flexengine_b200 import ops

    def launched(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(ops, "_on", lambda what, *tensors: ops._NO_GUARD)
    monkeypatch.setattr(ops, "_run", launched)
    monkeypatch.setattr(ops, "_kv4", lambda: None)
    return ops


def store_arguments():
    return dict(projected=torch.zeros(3, 8 * 64), bias=torch.zeros(8 * 64), positions=torch.zeros(3, dtype=torch.int32), inv_freq=torch.ones(32), rot=64,
                slot_mapping=torch.arange(3, dtype=torch.int32), cache=torch.zeros(kv4_shape(2, 2, 16, 64), dtype=torch.uint8), nq=4, nkv=2, d=64, page_size=16)


@pytest.mark.parametrize("change", [
    dict(projected=torch.zeros(3, 511)), dict(projected=torch.zeros(512, 3).t()), dict(projected=torch.zeros(512)), dict(bias=torch.zeros(511)),
    dict(bias=torch.zeros(512, dtype=torch.bfloat16)), dict(positions=torch.zeros(3, dtype=torch.int64)), dict(positions=torch.zeros(2, dtype=torch.int32)),
    dict(inv_freq=torch.ones(31)), dict(inv_freq=None), dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), dict(pairs="thirds"), dict(page_size=32),
    dict(page_size=8), dict(d=72), dict(nkv=3), dict(cache=torch.zeros(kv4_shape(2, 2, 16, 64), dtype=torch.int8)),
    dict(cache=torch.zeros(kv4_shape(4, 2, 16, 64), dtype=torch.uint8)[::2]), dict(projected=torch.zeros(3, 512, dtype=torch.float16)),
    dict(rot=66), dict(rot=63)])
def test_store_refuses(unlaunched, change):
    with pytest.raises((ValueError, TypeError)):
        unlaunched.qkv_rope_kv4(**dict(store_arguments(), **change))


@pytest.mark.parametrize("change", [
    dict(slots=torch.zeros(3, dtype=torch.int64)), dict(page_size=32), dict(d=80), dict(dtype=torch.float16), dict(slots=torch.zeros(6, dtype=torch.int32)[::2]),
    dict(slots=torch.zeros(3, 1, dtype=torch.int32))])
def test_rows_refuse(unlaunched, change):
    good = dict(cache=torch.zeros(kv4_shape(2, 2, 16, 64), dtype=torch.uint8), slots=torch.zeros(3, dtype=torch.int32), nkv=2, d=64, page_size=16)
    with pytest.raises((ValueError, TypeError)):
        unlaunched.kv4_rows(**dict(good, **change))


def attention_arguments(**step):
    ctx = dict(cu_q=torch.tensor([0, 1, 2], dtype=torch.int32), q_start=torch.tensor([5, 6], dtype=torch.int32), max_q_len=1, max_ctx_len=7)
    ctx.update(step)
    return dict(q=torch.zeros(2, 256, dtype=torch.bfloat16), cache=torch.zeros(kv4_shape(2, 2, 16, 64), dtype=torch.uint8),
                block_table=torch.zeros(2, 1, dtype=torch.int32), ctx=types.SimpleNamespace(**ctx), nq=4, nkv=2, d=64, page_size=16, scale=0.1)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 255)), dict(q=torch.zeros(2, 256, dtype=torch.float16)), dict(q=torch.zeros(2, 260)[:, :256]), dict(q=torch.zeros(256, 2).t()),
    dict(block_table=torch.zeros(2, 1, dtype=torch.int64)), dict(block_table=torch.zeros(3, 1, dtype=torch.int32)), dict(window=-1), dict(keep_first=2),
    dict(window=4, keep_first=-1), dict(page_size=48), dict(nq=5), dict(nq=4, nkv=3), dict(ctx=attention_arguments(max_ctx_len=17)["ctx"]),
    dict(ctx=attention_arguments(cu_q=torch.tensor([0, 1, 2]))["ctx"]), dict(ctx=attention_arguments(q_start=torch.zeros(3, dtype=torch.int32))["ctx"])])
def test_attention_refuses(unlaunched, change):
    with pytest.raises((ValueError, TypeError)):
        unlaunched.paged_attention_kv4(**dict(attention_arguments(), **change))


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 8, dtype=torch.bfloat16)), dict(logits=torch.zeros(8, 2).t()), dict(temperature=torch.ones(3)), dict(top_k=torch.zeros(2, dtype=torch.int64)),
    dict(top_p=torch.ones(2, dtype=torch.float64)), dict(min_p=torch.zeros(1)), dict(uniform=torch.zeros(4)[::2])])
def test_sample_filtered_refuses(unlaunched, change):
    good = dict(logits=torch.zeros(2, 8), temperature=torch.ones(2), top_k=torch.zeros(2, dtype=torch.int32), top_p=torch.ones(2), min_p=torch.zeros(2), uniform=torch.zeros(2))
    with pytest.raises((ValueError, TypeError)):
        unlaunched.sample_filtered(**dict(good, **change))


def test_operators_want_cuda_tensors():
    from flexengine_b200 import ops
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qkv_rope_kv4(**store_arguments())
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention_kv4(**attention_arguments())


# ---- which kernel takes portions ----------------------------------------------------------------------------------------------
def test_portions_choose_their_kernel():
    from flexengine_b200.ops import kv4_portions

    def of(n, context, new, **more):
        return kv4_portions([new] * n, [context - new] * n, 28, 4, 128, sms=148, **more)

    assert of(1, 2048, 2048) == 0 and of(4, 4096, 512) == 0 and of(8, 1000, 32) == 0            # long portions: tcgen05
    assert of(1, 300, 4) == 1 and of(32, 500, 2) == 1 and of(32, 2000, 4) == 1                    # few rows, enough blocks or short walks
    assert of(1, 4000, 2) == 8                                                                    # few rows late in a context: clusters
    assert of(1, 2048, 2048, tensor=False) == 1 and of(1, 4000, 2, tensor=False) == 8             # head sizes and types that tcgen05 does not take
    assert of(1, 100000, 1000, window=64) in (0, 1)
    assert kv4_portions([0, 3], [50, 0], 4, 2, 64, sms=148) == 1
    assert kv4_portions([1], [0], 64, 1, 64, sms=148) == 1


# ---- the walk to a limit of the sampling kernel -----------------------------------------------------------------------------------
def test_the_walk_to_a_limit_never_turns_back(tmp_path):
    """What one step sends on, the next does not send back: sums of 62 bits, whose limits lie next to the border between the two."""
    import ctypes
    import os
    import random
    import subprocess
    from flexengine_b200.ops import library
    source = tmp_path / "way.cpp"
    source.write_text('#include "cut.cuh"\nextern "C" int way(unsigned long long before, unsigned long long here, double limit)'
                      ' { return fe::cut_way(before, here, limit); }\n')
    built = str(tmp_path / "way.so")
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-I", library.CSRC, "-o", built, str(source)], check=True, timeout=120)
    way = ctypes.CDLL(built).way
    way.argtypes = [ctypes.c_ulonglong, ctypes.c_ulonglong, ctypes.c_double]
    rng = random.Random(3)
    pairs = [(1772367175443750147, 501071425968473999)] + [(rng.randrange(1 << 62), rng.randrange(1 << rng.randrange(50, 62))) for _ in range(5000)]
    for before, here in pairs:
        after = before + here
        near = np.float64(after)
        for limit in (np.nextafter(near, 0), near, np.nextafter(near, np.inf), float(before), float(before) + float(here)):
            first, then = way(before, here, limit), way(after, 1, limit)
            assert not (first > 0 and then < 0), (before, here, limit)
            assert first <= 0 or float(after) < limit
            assert first >= 0 or float(before) >= limit
    assert [way(5, 3, 5.0), way(5, 3, 5.5), way(5, 3, 8.0), way(5, 3, 8.5), way(0, 0, 1.0)] == [-1, 0, 0, 1, 1]


def test_the_host_s_work_grows_with_the_batch_not_its_square():
    """Half the rows with a limit: eight times the rows take about eight times as long (64 times where each row looks through all of them)."""
    import time

    class Nothing:
        @staticmethod
        def sample(logits, *_):
            return torch.zeros(logits.shape[0], dtype=torch.int32)

        @staticmethod
        def sample_filtered(logits, *_):
            return (torch.zeros(logits.shape[0], dtype=torch.int32),)

    def seconds(n):
        logits, best = torch.zeros(n, 1), 1e9
        for _ in range(5):
            start = time.perf_counter()
            Sampler(Nothing).sample_on_device(logits, [1.0] * n, [0] * n, list(range(n)), [0] * n, [0.5, 1.0] * (n // 2), [0.0] * n)
            best = min(best, time.perf_counter() - start)
        return best

    seconds(64)
    assert seconds(4096) <= 24 * seconds(512)


# ---- how much shared memory a kernel may have --------------------------------------------------------------------------------------
HARNESS = r"""
// errors.cu on a driver that is played: the call for LATE bytes holds on until another call has come and gone.
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

static std::atomic<int> set_to{0}, calls{0}, refuse{0};
static std::atomic<bool> hold{false}, inside{false};
static constexpr int LATE = 100;
static cudaError_t played_set(const void*, cudaFuncAttribute, int bytes) {
    if (refuse) return cudaErrorInvalidValue;
    ++calls;
    set_to = bytes;
    if (bytes == LATE && hold) {
        inside = true;
        for (int i = 0; i < 400 && calls < 2; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));      // a lock keeps the other out: no longer than that
        std::this_thread::sleep_for(std::chrono::milliseconds(50));
    }
    return cudaSuccess;
}
static cudaError_t played_device(int* device) { *device = 0; return cudaSuccess; }
#define cudaFuncSetAttribute played_set
#define cudaGetDevice played_device
#include "errors.cu"

int main() {
    static char kernels[2];
    const void *first = (const void*)((size_t)kernels & ~(size_t)15), *second = (const void*)((size_t)first + 4096);
    fe_allow_smem(first, 10);
    calls = 0;
    hold = true;
    std::thread wide([&] { fe_allow_smem(first, LATE); });
    while (!inside) std::this_thread::yield();
    std::thread narrow([&] { fe_allow_smem(first, 50); });
    wide.join();
    narrow.join();
    hold = false;
    if (!fe_allow_smem(first, LATE)) return 1;
    std::printf("%d\n", set_to.load());
    // one after the other: raised, never lowered, and not asked for again
    calls = 0;
    fe_allow_smem(second, 30), fe_allow_smem(second, 60), fe_allow_smem(second, 40), fe_allow_smem(second, 60);
    std::printf("%d %d\n", set_to.load(), calls.load());
    refuse = 1;
    const bool refused = !fe_allow_smem(second, 70), still = fe_allow_smem(second, 60);
    std::printf("%d %d\n", (int)refused, (int)still);
    return 0;
}
"""


def test_two_threads_do_not_lower_what_shared_memory_a_kernel_may_have(tmp_path):
    """A thread that asks for 50 bytes while another is on its way to 100: afterwards a kernel that needs 100 has them."""
    import subprocess
    from flexengine_b200.ops import library
    source = tmp_path / "harness.cu"
    source.write_text(HARNESS)
    built = str(tmp_path / "harness")
    subprocess.run([library.find_nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", library.CSRC, "-o", built, str(source)], check=True, timeout=300)
    out = subprocess.run([built], capture_output=True, text=True, check=True, timeout=60).stdout.split("\n")
    assert out[:3] == ["100", "60 2", "1 1"]


@pytest.mark.parametrize("scale", [-0.125, float("nan"), float("inf"), -float("inf")])
def test_attention_refuses_scales_that_would_turn_masks_into_numbers(unlaunched, scale):
    with pytest.raises(ValueError, match="not negative"):
        unlaunched.paged_attention_kv4(**dict(attention_arguments(), scale=scale))
