"""Page copies (mi_kv_copy_blocks via worker.hip_kv_blocks.copy_blocks), bit
for bit against a copy of the pool: independent pairs, forks of one page,
chains, swaps and cycles, leading rows only, every layout and element size.
"""

import random

import pytest
import torch

from microinfer_amd.runner import capture_graph
from microinfer_amd.worker.hip_kv_blocks import copy_blocks
from microinfer_amd.worker.kv_cache import KVCache
from tests.support import bits

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYOUTS = ["paired", "head_major", "token_major"]


def _cache(layers, blocks, block, heads, dim, dtype=torch.bfloat16, layout="paired", seed=0):
    cache = KVCache(layers, blocks, block, heads, dim, dtype=dtype, device=DEV, layout=layout)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cache.keys.copy_(torch.randn(cache.keys.shape, generator=gen, device=DEV))
    cache.values.copy_(torch.randn(cache.values.shape, generator=gen, device=DEV))
    return cache


def _check(keys, values, src, dst, tokens=None):
    block = keys.shape[-3]
    rows = tokens if tokens is not None else [block] * len(src)
    want = []
    for pool in (keys, values):
        before = pool.clone()
        after = before.clone()
        for s, d, n in zip(src, dst, rows):
            after[..., d, :n, :, :] = before[..., s, :n, :, :]
        want.append(after)
    copy_blocks(keys, values, src, dst, tokens=tokens)
    for pool, after in zip((keys, values), want):
        assert torch.equal(pool.contiguous().view(torch.uint8),
                           after.contiguous().view(torch.uint8))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("layers,block,heads,dim,dtype", [
    (3, 16, 8, 128, torch.bfloat16), (2, 16, 2, 64, torch.float32), (1, 32, 3, 80, torch.float16),
    (5, 1, 1, 8, torch.bfloat16), (2, 12, 5, 7, torch.float16), (2, 16, 1, 2, torch.bfloat16),
    (1, 256, 8, 128, torch.float32), (4, 8, 3, 5, torch.float32),
])
def test_independent_pairs(layout, layers, block, heads, dim, dtype):
    cache = _cache(layers, 40, block, heads, dim, dtype, layout)
    rng = random.Random(block + heads)
    ids = rng.sample(range(40), 40)
    _check(cache.keys, cache.values, ids[:13], ids[13:26])
    tokens = [rng.randint(0, block) for _ in range(13)]
    _check(cache.keys, cache.values, ids[:13], ids[13:26], tokens)
    # One page to many, all of a layer's view.
    _check(cache.keys[layers - 1], cache.values[layers - 1], [ids[0]] * 20, ids[20:], [block] * 20)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_chains_swaps_and_cycles(layout):
    cache = _cache(2, 64, 16, 2, 64, torch.bfloat16, layout)
    k, v = cache.keys, cache.values
    _check(k, v, [1, 2, 3, 4], [2, 3, 4, 5])             # shift up
    _check(k, v, [2, 3, 4, 5], [1, 2, 3, 4])             # shift down
    _check(k, v, [7, 8], [8, 7])                         # swap
    _check(k, v, [10, 11, 12], [11, 12, 10])             # cycle
    # A cycle whose pages are read from outside too, and a chain beside it.
    _check(k, v, [20, 21, 22, 21, 30, 31, 20], [21, 22, 20, 30, 31, 32, 33])
    # The same with leading rows only: rows past them break the cycle.
    _check(k, v, [20, 21, 22, 21, 30, 31, 20], [21, 22, 20, 30, 31, 32, 33],
           [16, 5, 9, 0, 16, 3, 1])
    _check(k, v, [7, 8], [8, 7], [3, 16])
    _check(k, v, [9, 9, 14], [9, 13, 14])                # onto itself
    _check(k, v, [40, 40, 41], [41, 42, 40], [0, 16, 16])


@pytest.mark.parametrize("seed", range(6))
def test_any_assignment(seed):
    rng = random.Random(seed)
    blocks = 500
    cache = _cache(2, blocks, 4, 2, 8, torch.float16, LAYOUTS[seed % 3], seed)
    n = rng.choice([3, 100, 450])
    dst = rng.sample(range(blocks), n)
    pool = range(blocks) if seed % 2 else dst
    src = [rng.choice(pool) for _ in range(n)]
    tokens = [rng.randint(0, 4) for _ in range(n)] if seed % 3 else None
    _check(cache.keys, cache.values, src, dst, tokens)


def test_lists_longer_than_a_launch():
    cache = _cache(2, 2100, 4, 1, 8)
    k, v = cache.keys, cache.values
    ids = random.Random(1).sample(range(2100), 2100)
    _check(k, v, ids[:1000], ids[1000:2000])
    _check(k, v, ids[:1000], ids[1:1001])                 # one chain over several launches
    cycle = ids[:255]
    _check(k, v, cycle, cycle[1:] + cycle[:1])            # the longest cycle
    many = ids[:2000]                                     # 400 cycles of five
    _check(k, v, many, [many[i // 5 * 5 + (i + 1) % 5] for i in range(2000)])
    with pytest.raises(RuntimeError, match="cycle"):
        copy_blocks(k, v, ids[:256], ids[1:256] + ids[:1])


def test_refusals_leave_the_pool_alone():
    cache = _cache(2, 8, 16, 2, 64)
    k, v = cache.keys, cache.values
    before = k.clone(), v.clone()
    for src, dst, tokens, what in [([0, 1], [2, 2], None, "twice"), ([0, 8], [2, 3], None, "id"),
                                   ([0, -1], [2, 3], None, "id"), ([0, 1], [2, 8], None, "id"),
                                   ([0, 1], [2, 3], [3, 17], "tokens"),
                                   ([0, 1], [2, 3], [3, -1], "tokens"), ([0], [2, 3], None, "one"),
                                   ([0, 1], [2, 3], [3], "one"), ([0.5], [1], None, "src")]:
        with pytest.raises(ValueError, match=what):
            copy_blocks(k, v, src, dst, tokens=tokens)
    with pytest.raises(ValueError, match="host"):
        copy_blocks(k, v, torch.tensor([0], device=DEV), [1])
    with pytest.raises(ValueError, match="shapes"):
        copy_blocks(k, v[:1], [0], [1])
    with pytest.raises(ValueError, match="layout"):
        copy_blocks(k, v.clone(memory_format=torch.contiguous_format), [0], [1])
    with pytest.raises(ValueError, match="dtype"):
        copy_blocks(k[0], v[0].view(torch.float16), [0], [1])
    copy_blocks(k, v, [], [])
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def test_fork_of_a_model_sized_pool_leaves_the_rest():
    cache = _cache(28, 64, 16, 8, 128)
    _check(cache.keys, cache.values, [5] * 16, list(range(20, 36)), [11] * 16)


def test_more_than_the_last_level_cache():
    cache = _cache(6, 900, 16, 8, 128)
    ids = random.Random(5).sample(range(900), 900)
    _check(cache.keys, cache.values, ids[:440], ids[440:880])


def test_offsets_past_32_bits():
    # A pool of 8 GiB: its last pages lie past 2^32 bytes and 2^31 elements.
    cache = KVCache(1, 65536 * 2, 16, 8, 128, dtype=torch.bfloat16, device=DEV)
    last = cache.num_blocks - 1
    gen = torch.Generator(device=DEV).manual_seed(3)
    for pool in (cache.keys, cache.values):
        pool[0, :2] = torch.randn(2, 16, 8, 128, generator=gen, device=DEV).to(torch.bfloat16)
    copy_blocks(cache.keys, cache.values, [0, 1], [last, last - 1], tokens=[16, 7])
    copy_blocks(cache.keys, cache.values, [last], [2])
    for pool in (cache.keys, cache.values):
        assert torch.equal(pool[0, last], pool[0, 0]) and torch.equal(pool[0, 2], pool[0, 0])
        assert torch.equal(pool[0, last - 1, :7], pool[0, 1, :7])
        assert not pool[0, last - 1, 7:].any()


def test_nan_patterns_survive_and_numpy_lists_are_taken():
    import numpy as np

    cache = _cache(1, 8, 16, 2, 64, torch.bfloat16)
    raw = cache.keys[0, 3].view(torch.int16)
    raw.copy_(torch.randint(-32768, 32767, raw.shape, device=DEV, dtype=torch.int16))
    copy_blocks(cache.keys, cache.values, np.array([3]), np.array([6]))
    assert (bits(cache.keys[0, 6]) == bits(cache.keys[0, 3])).all()


def test_another_stream_and_a_captured_call():
    cache = _cache(4, 32, 16, 8, 128)
    k, v = cache.keys, cache.values
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check(k, v, [1, 2], [3, 4], [16, 5])
    torch.cuda.synchronize()
    src, dst = [1, 1, 2], [8, 9, 10]
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph, stream=side):
        copy_blocks(k, v, src, dst)
    src[:] = [7, 7, 7]                                    # the lists were read at capture
    for replay in range(3):
        gen = torch.Generator(device=DEV).manual_seed(replay)
        k[:, 1:3] = torch.randn(4, 2, 16, 8, 128, generator=gen, device=DEV).to(torch.bfloat16)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for s, d in ((1, 8), (1, 9), (2, 10)):
            assert torch.equal(k[:, d], k[:, s]) and torch.equal(v[:, d], v[:, s])


@pytest.mark.parametrize("seed", range(4))
def test_few_pairs_of_many_blocks(seed):
    rng = random.Random(seed)
    cache = _cache(2, 40000, 4, 2, 8, torch.bfloat16, LAYOUTS[seed % 3], seed)
    k, v = cache.keys, cache.values
    a, b, c, d, e, f, g = rng.sample(range(40000), 7)
    _check(k, v, [a], [b])
    _check(k, v, [a, b], [b, a])
    _check(k, v, [a, b, c, b, d, e, a], [b, c, a, d, e, f, g])
    for n in (2, 17, 38, 124):
        dst = rng.sample(range(40000), n)
        src = [rng.choice(dst) if rng.random() < 0.7 else rng.randrange(40000) for _ in range(n)]
        _check(k, v, src, dst, [rng.randint(0, 4) for _ in range(n)])
