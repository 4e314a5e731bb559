"""Decode and varlen attention over an 8-bit cache against float64."""

import math
import threading

import numpy as np
import pytest
import torch

from microinfer_amd.layer.hip_quantized_attention import (hip_quantized_decode,
                                                          hip_quantized_prefill,
                                                          quantized_decode_plan,
                                                          quantized_prefill_plan)
from microinfer_amd.worker.hip_quantized_kv import quantized_append, quantized_gather
from microinfer_amd.worker.kv_cache import KVCache
from tests.quantized_support import CODES, DTYPES, Twin, check_attention, ints, tables_of

pytestmark = pytest.mark.gpu

# How a softmax weight is held for its product with V (``check_attention``).
# Decode: two bf16 parts for 16-bit queries (half a step of each: 2^-8 of 2^-8),
# three for float32. Varlen: one f16 part for 16-bit queries (half a step, 2^-11),
# three bf16 parts for float32.
DECODE = {"bf16": (16, 0), "f16": (16, 0), "f32": (24, 0)}
VARLEN = {"bf16": (11, 2.0 ** -35), "f16": (11, 2.0 ** -35), "f32": (24, 0)}

SHAPES = [  # Hq, Hkv, D, block, layout
    (16, 8, 128, 16, "paired"), (32, 8, 128, 32, "head_major"), (5, 5, 128, 64, "token_major"),
    (15, 5, 64, 16, "paired"), (8, 1, 64, 32, "token_major"), (16, 1, 128, 16, "paired"),
    (6, 2, 32, 16, "paired"), (34, 2, 128, 16, "paired"), (4, 2, 16, 4, "head_major"),
    (3, 1, 256, 16, "paired"), (2, 2, 128, 8, "token_major")]


def query_of(rng, rows, heads, dim, dtype):
    return torch.from_numpy(rng.standard_normal((rows, heads, dim))).to(DTYPES[dtype]).cuda()


def decode_case(rng, contexts, shape, kind, dtype, blocks=None):
    hq, hkv, dim, block, layout = shape
    blocks = blocks or sum(-(-c // block) for c in contexts) + 2
    twin = Twin(blocks, block, hkv, dim, kind, layout)
    twin.fill(rng)
    return twin, tables_of(rng, contexts, block, blocks), query_of(rng, len(contexts), hq, dim,
                                                                   dtype)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(kind, dtype, shape):
    rng = np.random.default_rng(shape[0] + shape[2])
    contexts = [1, 0, 17, 33, 700, 2, 64, 257]
    twin, tables, query = decode_case(rng, contexts, shape, kind, dtype)
    scale = 1 / math.sqrt(shape[2])
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
    assert got.dtype == query.dtype and not got[1].any()
    check_attention(got, query, twin, tables, contexts, list(range(9)), scale,
                    DECODE[dtype])


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("contexts", [[4000], [2500, 3, 1900], [300] * 40, [1] * 70,
                                      [40 + 7 * i for i in range(90)]])
def test_decode_splits_and_batches(kind, dtype, contexts):
    rng = np.random.default_rng(len(contexts))
    twin, tables, query = decode_case(rng, contexts, (4, 2, 128, 16, "paired"), kind, dtype)
    plan = quantized_decode_plan(ints(contexts), num_q_heads=4, num_kv_heads=2, head_dim=128,
                                 dtype=query.dtype, block_size=16,
                                 block_table_width=len(tables[0]))
    for q in (query, query.flip(0)):
        got = hip_quantized_decode(q, *twin.tensors, ints(tables), ints(contexts), plan=plan,
                                   scale=0.11)
        check_attention(got, q, twin, tables, contexts, list(range(len(contexts) + 1)), 0.11,
                        DECODE[dtype])


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_what_the_context_ends_before_does_not_matter(kind):
    """NaN codes and scales behind the context, in the pages behind it and in
    blocks that the table does not name."""
    rng = np.random.default_rng(2)
    contexts = [19, 5, 160, 513]
    for shape in ((4, 2, 128, 16, "paired"), (4, 2, 64, 32, "paired"), (4, 4, 32, 16, "paired"),
                  (4, 2, 256, 16, "paired")):
        twin, tables, query = decode_case(rng, contexts, shape, kind, "bf16")
        block = shape[3]
        used = {tables[s][j] for s, c in enumerate(contexts) for j in range(-(-c // block))}
        for pool, scales in ((twin.layer.keys, twin.layer.key_scales),
                             (twin.layer.values, twin.layer.value_scales)):
            for page in range(pool.shape[0]):
                if page not in used:
                    scales[page] = float("nan")
                    pool[page].view(torch.uint8).fill_(0x7f)
            if kind == "fp8":
                for s, c in enumerate(contexts):
                    if c % block:
                        pool[tables[s][c // block], c % block:].view(torch.uint8).fill_(0xff)
        wide = [row + [page] * 2 for row, page in zip(tables, (0, 1, 2, 3))]
        got = hip_quantized_decode(query, *twin.tensors, ints(wide), ints(contexts))
        check_attention(got, query, twin, tables, contexts, list(range(5)),
                        1 / math.sqrt(shape[2]), DECODE["bf16"])


@pytest.mark.parametrize("shape", [(4, 2, 128, 16, "paired"), (4, 2, 64, 16, "paired"),
                                   (4, 2, 128, 64, "paired"), (3, 3, 32, 16, "paired"),
                                   (4, 2, 256, 16, "paired")])
def test_blocks_outside_the_pool_are_masked(shape):
    rng = np.random.default_rng(3)
    contexts = [100, 900, 40, 33]
    twin, tables, query = decode_case(rng, contexts, shape, "fp8", "f16")
    blocks = twin.k.shape[0]
    tables[0][0] = -1
    tables[1][1] = blocks
    tables[1][-1] = 2 ** 31 - 1
    tables[2] = [-5] * len(tables[2])
    tables[3][-(-33 // shape[3]) - 1] = -2 ** 31
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
    assert not got[2].any()
    check_attention(got, query, twin, tables, contexts, list(range(5)), 1 / math.sqrt(shape[2]),
                    DECODE["f16"])


@pytest.mark.parametrize("dim", [256, 128, 64, 32])
def test_nan_reaches_the_output(dim):
    """A NaN code or scale inside a context makes its rows NaN, wherever the
    context is split, and no other sequence's."""
    rng = np.random.default_rng(4)
    contexts = [1500, 60, 1500, 900, 20]
    twin, tables, query = decode_case(rng, contexts, (4, 2, dim, 16, "paired"), "fp8", "bf16")
    twin.layer.keys[tables[0][93], 7, 0, 3:4].view(torch.uint8).fill_(0x7f)
    twin.layer.value_scales[tables[2][0], 1] = float("nan")
    twin.layer.key_scales[tables[3][50], 0] = float("nan")
    twin.layer.values[tables[4][0], 19 % 16, 0, 5:6].view(torch.uint8).fill_(0xff)
    twin.layer.values[tables[4][1], 3, 1, 6:7].view(torch.uint8).fill_(0xff)
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts)).float().cpu()
    assert got[0, :2].isnan().all() and not got[0, 2:].isnan().any()
    assert not got[1].isnan().any()
    assert got[2, 2:].isnan().all() and not got[2, :2].isnan().any()
    assert got[3, :2].isnan().all() and not got[3, 2:].isnan().any()
    assert got[4, 2:, 6].isnan().all()
    rows = hip_quantized_prefill(query[:1], *twin.tensors, ints([0, 1]), ints([0, 1500]),
                                 ints(tables[:1]), max_seqlen_q=1).float().cpu()
    assert rows[0, :2].isnan().all() and not rows[0, 2:].isnan().any()


def test_scales_far_apart():
    """Blocks whose values differ by 2^60 in size, and weights that differ as
    much the other way."""
    rng = np.random.default_rng(5)
    for dtype in DTYPES:
        for kind in CODES:
            contexts = [400, 70]
            hq, hkv, dim, block, layout = 4, 2, 128, 16, "paired"
            twin = Twin(40, block, hkv, dim, kind, layout)
            twin.fill(rng, sizes=(-3, 3))
            twin.vs *= np.exp2(rng.integers(-30, 31, twin.vs.shape))
            twin.layer.value_scales.copy_(torch.from_numpy(twin.vs).float())
            if dtype == "f16":  # outputs within its range
                twin.vs *= 2.0 ** -30
                twin.layer.value_scales.copy_(torch.from_numpy(twin.vs).float())
            tables = tables_of(rng, contexts, block, 40)
            query = 3 * query_of(rng, 2, hq, dim, dtype)
            got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
            check_attention(got, query, twin, tables, contexts, [0, 1, 2], dim ** -0.5,
                            DECODE[dtype])
            cu_q = [0, 40, 41]
            query = 3 * query_of(rng, 41, hq, dim, dtype)
            got = hip_quantized_prefill(query, *twin.tensors, ints(cu_q), ints([0, 400, 470]),
                                        ints(tables), max_seqlen_q=40)
            check_attention(got, query, twin, tables, contexts, cu_q, dim ** -0.5,
                            VARLEN[dtype])


def prefill(query, twin, tables, contexts, lengths, planned=False, **kw):
    cu_q = np.cumsum([0] + lengths).tolist()
    cu_k = np.cumsum([0] + contexts).tolist()
    plan = None
    if planned:
        plan = quantized_prefill_plan(
            ints(cu_q), ints(cu_k), num_tokens=query.shape[0], num_q_heads=query.shape[1],
            num_kv_heads=twin.k.shape[2], head_dim=query.shape[2], dtype=query.dtype,
            block_size=twin.k.shape[1], block_table_width=len(tables[0]))
    return hip_quantized_prefill(query, *twin.tensors, ints(cu_q), ints(cu_k), ints(tables),
                                 max_seqlen_q=max(lengths), plan=plan, **kw), cu_q


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_prefill(kind, dtype, shape):
    rng = np.random.default_rng(shape[0] + shape[2] + 1)
    contexts, lengths = [70, 1, 45, 130, 33, 9], [33, 1, 1, 70, 0, 9]
    hq, hkv, dim, block, layout = shape
    twin, tables, _ = decode_case(rng, contexts, shape, kind, dtype)
    query = query_of(rng, sum(lengths), hq, dim, dtype)
    for planned in (False, True):
        got, cu_q = prefill(query, twin, tables, contexts, lengths, planned)
        assert got.dtype == query.dtype
        check_attention(got, query, twin, tables, contexts, cu_q, 1 / math.sqrt(dim),
                        VARLEN[dtype])


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("contexts,lengths", [
    ([1800], [40]), ([1800, 900], [1, 129]), ([300, 310, 320, 330], [5, 4, 3, 2]),
    ([257], [257]), ([600, 1, 500], [64, 1, 65])])
def test_prefill_lengths(kind, contexts, lengths):
    rng = np.random.default_rng(len(contexts))
    twin, tables, _ = decode_case(rng, contexts, (8, 2, 128, 16, "paired"), kind, "bf16")
    query = query_of(rng, sum(lengths), 8, 128, "bf16")
    for planned in (False, True):
        got, cu_q = prefill(query, twin, tables, contexts, lengths, planned, scale=0.07)
        check_attention(got, query, twin, tables, contexts, cu_q, 0.07, VARLEN["bf16"])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("shape,lengths", [
    ((4, 2, 128, 16, "paired"), [3, 0, 1, 8, 2]),  # up to 16 rows
    ((8, 2, 64, 32, "head_major"), [7, 8, 0, 1, 5]),  # 32
    ((12, 2, 128, 16, "paired"), [10, 9, 1, 6, 3]),  # 60, in two groups
    ((3, 1, 64, 16, "token_major"), [11, 21, 5, 16, 13]),  # 63
    ((20, 1, 128, 64, "paired"), [1, 3, 2, 0, 3]),
    ((17, 1, 64, 16, "paired"), [0, 0, 1, 1, 0]),
    ((6, 2, 256, 32, "head_major"), [3, 0, 5, 1, 4])])  # 18, of 256 dims
def test_few_rows_a_request(kind, dtype, shape, lengths):
    """Requests laid out like decode steps: whole and in parts, rows in one
    group and in several, tokens that see less than the last, rows that see
    nothing, blocks outside the pool."""
    rng = np.random.default_rng(sum(lengths))
    hq, hkv, dim, block, _ = shape
    contexts = [1700, 40, 33, 5, 900]
    twin, tables, _ = decode_case(rng, contexts, shape, kind, dtype)
    tables[4][0] = -3
    query = query_of(rng, sum(lengths), hq, dim, dtype)
    cu_q = ints(np.cumsum([0] + lengths).tolist())
    cu_k = ints(np.cumsum([0] + contexts).tolist())
    plan = quantized_prefill_plan(
        cu_q, cu_k, num_tokens=query.shape[0], num_q_heads=hq, num_kv_heads=hkv, head_dim=dim,
        dtype=query.dtype, block_size=block, block_table_width=len(tables[0]),
        max_seqlen_q=max(lengths) + 1)
    for q, how, most in ((query, None, max(lengths)), (query, plan, max(lengths) + 1),
                         (query.flip(0), plan, max(lengths) + 1)):
        got = hip_quantized_prefill(q, *twin.tensors, cu_q, cu_k, ints(tables),
                                    max_seqlen_q=max(lengths), plan=how, scale=0.13)
        few = most * hq // hkv <= 32  # of five requests
        check_attention(got, q, twin, tables, contexts, cu_q.tolist(), 0.13,
                        (DECODE if few else VARLEN)[dtype])
    longer = dict(max_seqlen_q=max(lengths) + 2, plan=plan)
    if sum(lengths) > max(lengths) + 1:  # more rows than tokens there cannot be
        with pytest.raises(ValueError, match="plan"):
            hip_quantized_prefill(query, *twin.tensors, cu_q, cu_k, ints(tables), **longer)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape,length,context", [
    ((8, 2, 128, 16, "paired"), 30, 1900), ((3, 1, 64, 32, "head_major"), 42, 700),
    ((128, 1, 128, 16, "paired"), 1, 2500), ((16, 2, 64, 16, "paired"), 16, 50),
    ((4, 1, 256, 16, "paired"), 61, 900)])
def test_one_request_of_rows_in_several_groups(dtype, shape, length, context):
    rng = np.random.default_rng(length)
    hq, hkv, dim, block, _ = shape
    twin, tables, _ = decode_case(rng, [context], shape, "fp8", dtype)
    query = query_of(rng, length, hq, dim, dtype)
    got = hip_quantized_prefill(query, *twin.tensors, ints([0, length]), ints([0, context]),
                                ints(tables), max_seqlen_q=length)
    check_attention(got, query, twin, tables, [context], [0, length], dim ** -0.5, DECODE[dtype])


@pytest.mark.parametrize("hq,hkv", [(17, 1), (32, 1), (64, 2), (66, 2), (40, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_of_large_groups(hq, hkv, dim):
    rng = np.random.default_rng(hq)
    contexts = [1500, 1, 77]
    shape = (hq, hkv, dim, 16, "paired")
    for dtype in DTYPES:
        twin, tables, query = decode_case(rng, contexts, shape, "fp8", dtype)
        got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
        check_attention(got, query, twin, tables, contexts, [0, 1, 2, 3], dim ** -0.5,
                        DECODE[dtype])


def test_few_rows_in_graphs_and_on_other_streams():
    """A captured plan with its calls and captured calls of an eager plan,
    replayed among eager calls, as the lengths on the device change."""
    rng = np.random.default_rng(21)
    contexts, lengths = [1800, 500, 60], [4, 1, 3]
    shape = (8, 2, 128, 16, "paired")
    twin, tables, _ = decode_case(rng, contexts, shape, "fp8", "bf16")
    query, other = query_of(rng, 8, 8, 128, "bf16"), query_of(rng, 8, 8, 128, "bf16")
    cu_q, cu_k = ints([0, 4, 5, 8]), ints(np.cumsum([0] + contexts).tolist())
    at = ints(tables)

    def planned():
        return quantized_prefill_plan(cu_q, cu_k, num_tokens=8, num_q_heads=8, num_kv_heads=2,
                                      head_dim=128, dtype=query.dtype, block_size=16,
                                      block_table_width=at.shape[1], max_seqlen_q=4)

    def run(q, plan):
        return hip_quantized_prefill(q, *twin.tensors, cu_q, cu_k, at, max_seqlen_q=4, plan=plan)

    eager = planned()
    want = run(query, eager).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = planned()
        first, second = run(query, plan), run(other, plan)
    held = torch.cuda.CUDAGraph()
    with torch.cuda.graph(held):
        third = run(query, eager)
    side = torch.cuda.Stream()
    for step in range(3):
        graph.replay()
        held.replay()
        with torch.cuda.stream(side):
            fourth = run(query, eager)
        torch.cuda.synchronize()
        for got, q in ((first, query), (second, other)):
            check_attention(got, q, twin, tables, contexts, [0, 4, 5, 8], 128 ** -0.5,
                            DECODE["bf16"])
        assert torch.equal(third, want) and torch.equal(fourth, want)
        if step == 1:  # lengths for the captured plan; the eager one keeps its own
            contexts = [1700, 300, 41]
            cu_k.copy_(ints(np.cumsum([0] + contexts).tolist()))
            break
    graph.replay()
    torch.cuda.synchronize()
    check_attention(first, query, twin, tables, contexts, [0, 4, 5, 8], 128 ** -0.5,
                    DECODE["bf16"])


def test_prefill_rows_that_see_nothing_are_zeros():
    """More query rows than positions, contexts of nothing, invalid blocks."""
    rng = np.random.default_rng(7)
    for shape in ((4, 2, 128, 16, "paired"), (4, 2, 64, 16, "paired"), (2, 2, 32, 16, "paired")):
        contexts, lengths = [5, 0, 40, 20], [9, 3, 2, 20]
        twin, tables, _ = decode_case(rng, contexts, shape, "int8", "bf16")
        tables[3] = [-1] * len(tables[3])
        query = query_of(rng, sum(lengths), shape[0], shape[2], "bf16")
        for planned in (False, True):
            got, cu_q = prefill(query, twin, tables, contexts, lengths, planned)
            assert not got[:4].any() and not got[9:12].any() and not got[14:].any()
            check_attention(got, query, twin, tables, contexts, cu_q, 1 / math.sqrt(shape[2]),
                            VARLEN["bf16"])


def test_strides_of_queries():
    rng = np.random.default_rng(8)
    contexts = [90, 31]
    twin, tables, _ = decode_case(rng, contexts, (4, 2, 128, 16, "paired"), "fp8", "bf16")
    fused = query_of(rng, 2, 8, 128, "bf16")
    for query in (fused[:, 2:6], query_of(rng, 2, 4, 130, "bf16")[..., 1:129],
                  query_of(rng, 4, 2, 128, "bf16").transpose(0, 1)):
        got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
        check_attention(got, query, twin, tables, contexts, [0, 1, 2], 128 ** -0.5, DECODE["bf16"])
        got = hip_quantized_prefill(query, *twin.tensors, ints([0, 1, 2]), ints([0, 90, 121]),
                                    ints(tables), max_seqlen_q=1)
        check_attention(got, query, twin, tables, contexts, [0, 1, 2], 128 ** -0.5, VARLEN["bf16"])


def test_decode_graphs_and_eager_calls_share_nothing():
    """Two captured graphs, an eager plan and a plan captured with its calls,
    replayed among eager calls on another stream."""
    rng = np.random.default_rng(9)
    contexts = [1700, 300, 900]
    shape = (8, 2, 128, 16, "paired")
    twin, tables, query = decode_case(rng, contexts, shape, "fp8", "bf16")
    tables, lens = ints(tables), ints(contexts)
    sizes = dict(num_q_heads=8, num_kv_heads=2, head_dim=128, dtype=torch.bfloat16,
                 block_size=16, block_table_width=tables.shape[1])
    eager = quantized_decode_plan(lens, **sizes)
    queries = [query, query.flip(0).contiguous(), (query * 2).contiguous()]
    want = [hip_quantized_decode(q, *twin.tensors, tables, lens, plan=eager) for q in queries]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = eager if i else quantized_decode_plan(lens, **sizes)
            outs.append([hip_quantized_decode(q, *twin.tensors, tables, lens, plan=plan)
                         for q in queries])
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(3):
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        third = torch.cuda.Stream()
        with torch.cuda.stream(third):
            again = hip_quantized_decode(queries[1], *twin.tensors, tables, lens, plan=eager)
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(again, want[1])


def test_decode_replays_with_other_lengths():
    rng = np.random.default_rng(10)
    shape = (4, 2, 128, 16, "paired")
    most = [1200, 700, 64]
    twin, tables, query = decode_case(rng, most, shape, "int8", "f16")
    lens = ints(most)
    where = ints(tables)

    def call():
        return hip_quantized_decode(query, *twin.tensors, where, lens)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for contexts in ([3, 700, 1], [1200, 0, 64], [640, 333, 17]):
        lens.copy_(ints(contexts))
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, query, twin, tables, contexts, [0, 1, 2, 3], 128 ** -0.5,
                        DECODE["f16"])


def test_graphs_do_not_share_a_plans_workspace():
    """A plan that one graph holds, called in the capture of another: both are
    replayed at once, on two streams."""
    rng = np.random.default_rng(23)
    contexts, lengths = [1900, 700, 1200], [3, 200, 4]
    twin, tables, _ = decode_case(rng, contexts, (8, 2, 128, 16, "paired"), "fp8", "bf16")
    at, lens = ints(tables), ints(contexts)
    sizes = dict(num_q_heads=8, num_kv_heads=2, head_dim=128, dtype=torch.bfloat16,
                 block_size=16, block_table_width=at.shape[1])
    cu_k = ints(np.cumsum([0] + contexts).tolist())
    one, other = (query_of(rng, 3, 8, 128, "bf16") for _ in range(2))
    cases = [(one, other, [1, 1, 1], lambda: quantized_decode_plan(lens, **sizes),
              lambda q, plan: hip_quantized_decode(q, *twin.tensors, at, lens, plan=plan))]
    for new in ([3, 2, 4], lengths):
        cu_q = ints(np.cumsum([0] + new).tolist())
        rows, most = sum(new), max(new)
        one, other = (query_of(rng, rows, 8, 128, "bf16") for _ in range(2))
        cases.append((
            one, other, new,
            lambda cu_q=cu_q, rows=rows, most=most: quantized_prefill_plan(
                cu_q, cu_k, num_tokens=rows, max_seqlen_q=most, **sizes),
            lambda q, plan, cu_q=cu_q, most=most: hip_quantized_prefill(
                q, *twin.tensors, cu_q, cu_k, at, max_seqlen_q=most, plan=plan)))
    side = torch.cuda.Stream()
    for one, other, new, planned, run in cases:
        held = planned()
        run(one, held)  # kernels are loaded
        torch.cuda.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            plan = planned()
            mine = run(one, plan)
        first.replay()
        torch.cuda.synchronize()
        with torch.cuda.graph(second):
            theirs = run(other, plan)
        for _ in range(10):
            first.replay()
            with torch.cuda.stream(side):
                second.replay()
        torch.cuda.synchronize()
        cu_q = np.cumsum([0] + new).tolist()
        for got, q in ((mine, one), (theirs, other)):
            check_attention(got, q, twin, tables, contexts, cu_q, 128 ** -0.5, VARLEN["bf16"])


def test_results_repeat():
    rng = np.random.default_rng(11)
    contexts = [3000, 40, 1500]
    twin, tables, query = decode_case(rng, contexts, (8, 2, 128, 16, "paired"), "fp8", "bf16")
    first = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
    for _ in range(5):
        assert torch.equal(first, hip_quantized_decode(query, *twin.tensors, ints(tables),
                                                       ints(contexts)))


def test_two_threads_with_the_same_plans():
    """Plans made by one thread, called by two at once, each on a stream of its
    own: workspaces and counters are not shared."""
    rng = np.random.default_rng(31)
    contexts = [1900, 40, 1300]
    twin, tables, _ = decode_case(rng, contexts, (8, 2, 128, 16, "paired"), "fp8", "bf16")
    at, lens = ints(tables), ints(contexts)
    cu_k = ints(np.cumsum([0] + contexts).tolist())
    sizes = dict(num_q_heads=8, num_kv_heads=2, head_dim=128, dtype=torch.bfloat16,
                 block_size=16, block_table_width=at.shape[1])
    news = [[1, 1, 1], [5, 1, 3], [150, 40, 90]]
    offsets = [ints(np.cumsum([0] + new).tolist()) for new in news]
    plans = [quantized_decode_plan(lens, **sizes)] + [
        quantized_prefill_plan(cu_q, cu_k, num_tokens=sum(new), max_seqlen_q=max(new), **sizes)
        for cu_q, new in zip(offsets[1:], news[1:])]

    def run(i, q):
        if i == 0:
            return hip_quantized_decode(q, *twin.tensors, at, lens, plan=plans[0])
        return hip_quantized_prefill(q, *twin.tensors, offsets[i], cu_k, at,
                                     max_seqlen_q=max(news[i]), plan=plans[i])

    queries = [[query_of(rng, sum(new), 8, 128, "bf16") for new in news] for _ in range(2)]
    torch.cuda.synchronize()
    results, errors = [None, None], []

    def work(who):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    outs = [run(i, q) for i, q in enumerate(queries[who])]
                torch.cuda.current_stream().synchronize()
            results[who] = outs
        except Exception as error:  # reported by the test's own thread
            errors.append(error)

    threads = [threading.Thread(target=work, args=(who,)) for who in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors
    for who in range(2):
        for got, q, cu_q in zip(results[who], queries[who], offsets):
            check_attention(got, q, twin, tables, contexts, cu_q.tolist(), 128 ** -0.5,
                            VARLEN["bf16"])


@pytest.mark.parametrize("layout", ["paired", "token_major"])
def test_offsets_past_32_bits(layout):
    """Blocks that lie more than 2^31 bytes into a pool hold and give what those of
    a small one do."""
    rng = np.random.default_rng(32)
    blocks, heads, dim, block = 150000, 8, 128, 16
    contexts = [500, 37]
    need = [-(-c // block) for c in contexts]
    high = [[blocks - 1 - 7 * j - 1000 * s for j in range(n)] + [-1] * (max(need) - n)
            for s, n in enumerate(need)]
    low = [[j + 40 * s for j in range(n)] + [-1] * (max(need) - n) for s, n in enumerate(need)]
    rows = [torch.from_numpy(rng.standard_normal((sum(contexts), heads, dim))).bfloat16().cuda()
            for _ in range(2)]
    query = query_of(rng, 3, 16, dim, "bf16")
    chunk = query_of(rng, 200, 16, dim, "bf16")
    cu_k = ints([0, contexts[0], sum(contexts)])
    outs = []
    for count, tables in ((blocks, high), (80, low)):
        cache = KVCache(1, count, block, heads, dim, dtype=torch.float8_e4m3fn, device="cuda",
                        layout=layout).layer(0)
        tensors = cache.keys, cache.values, cache.key_scales, cache.value_scales
        slots = [t[p // block] * block + p % block for t, c in zip(tables, contexts)
                 for p in range(c)]
        at = ints(tables)
        for part in (slice(0, 400), slice(400, None)):  # planned, scanned
            quantized_append(*tensors, torch.tensor(slots[part], device="cuda"),
                             rows[0][part], rows[1][part])
        outs.append([
            *quantized_gather(*tensors, at, cu_k, sum(contexts)),
            hip_quantized_decode(query[:2], *tensors, at, ints(contexts)),
            hip_quantized_prefill(query, *tensors, ints([0, 2, 3]), cu_k, at, max_seqlen_q=2),
            hip_quantized_prefill(chunk, *tensors, ints([0, 170, 200]), cu_k, at,
                                  max_seqlen_q=170)])
        del cache, tensors
    for far, near in zip(*outs):
        assert torch.equal(far, near)
    assert not torch.equal(outs[0][0], torch.zeros_like(outs[0][0]))


@pytest.mark.parametrize("shape", [(4, 2, 128, 256, "paired"), (2, 1, 64, 1024, "head_major"),
                                   (3, 1, 256, 128, "paired"), (2, 2, 32, 512, "token_major")])
def test_large_blocks(shape):
    rng = np.random.default_rng(shape[3])
    contexts = [1500, 3, 1024, 700]
    twin, tables, query = decode_case(rng, contexts, shape, "int8", "f16")
    scale = 1 / math.sqrt(shape[2])
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
    check_attention(got, query, twin, tables, contexts, list(range(5)), scale, DECODE["f16"])
    for lengths in ([3, 1, 0, 2], [130, 3, 1, 64]):
        query = query_of(rng, sum(lengths), shape[0], shape[2], "f16")
        got, cu_q = prefill(query, twin, tables, contexts, lengths)
        check_attention(got, query, twin, tables, contexts, cu_q, scale, VARLEN["f16"])


def test_the_most_sequences():
    rng = np.random.default_rng(33)
    contexts = [int(c) for c in rng.integers(0, 40, 4096)]
    shape = (2, 1, 64, 16, "paired")
    twin, tables, query = decode_case(rng, contexts, shape, "fp8", "bf16")
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
    check_attention(got, query, twin, tables, contexts, list(range(4097)), 0.125, DECODE["bf16"])
    plan = quantized_prefill_plan(
        ints(range(4097)), ints(np.cumsum([0] + contexts).tolist()), num_tokens=4096,
        max_seqlen_q=1, num_q_heads=2, num_kv_heads=1, head_dim=64, dtype=query.dtype,
        block_size=16, block_table_width=len(tables[0]))
    got = hip_quantized_prefill(query, *twin.tensors, plan.cu_seqlens_q, plan.cu_seqlens_k,
                                ints(tables), max_seqlen_q=1, plan=plan)
    check_attention(got, query, twin, tables, contexts, list(range(4097)), 0.125, DECODE["bf16"])
    more = [1] * 4097
    with pytest.raises(ValueError, match="4096"):
        hip_quantized_decode(query_of(rng, 4097, 2, 64, "bf16"), *twin.tensors,
                             torch.zeros(4097, 1, dtype=torch.int32, device="cuda"), ints(more))


@pytest.mark.parametrize("shape,dtype", [
    ((4, 2, 128, 16, "paired"), "bf16"), ((16, 2, 128, 16, "paired"), "f16"),
    ((16, 2, 64, 16, "paired"), "f32"), ((32, 2, 64, 16, "head_major"), "bf16")])
def test_many_short_sequences_and_a_few_long_ones(shape, dtype):
    rng = np.random.default_rng(35)
    contexts = [3000, 900] + [int(c) for c in rng.integers(0, 30, 600)] + [1500]
    twin, tables, query = decode_case(rng, contexts, shape, "int8", dtype)
    scale = 1 / math.sqrt(shape[2])
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts))
    check_attention(got, query, twin, tables, contexts, list(range(604)), scale, DECODE[dtype])


@pytest.mark.parametrize("lengths", [[3, 0, 2], [60, 1, 90]])
def test_rows_behind_the_last_request(lengths):
    """Padded queries: the requests' rows are what they are without; tables and
    offsets of other types and strides."""
    rng = np.random.default_rng(34)
    contexts = [300, 70, 95]
    twin, tables, _ = decode_case(rng, contexts, (8, 2, 128, 16, "paired"), "fp8", "bf16")
    rows = sum(lengths)
    query = query_of(rng, rows + 40, 8, 128, "bf16")
    cu_q = np.cumsum([0] + lengths).tolist()
    cu_k = np.cumsum([0] + contexts).tolist()
    wide = torch.full((3, 2 * len(tables[0])), -1, dtype=torch.int64, device="cuda")
    wide[:, ::2] = ints(tables)
    got = hip_quantized_prefill(query, *twin.tensors, torch.tensor(cu_q, device="cuda"),
                                torch.tensor(cu_k, device="cuda"), wide[:, ::2],
                                max_seqlen_q=max(lengths))
    check_attention(got[:rows], query[:rows], twin, tables, contexts, cu_q, 128 ** -0.5,
                    VARLEN["bf16"])
    got = hip_quantized_decode(query[:3], *twin.tensors, wide[:, ::2],
                               torch.tensor(contexts, device="cuda"))
    check_attention(got, query[:3], twin, tables, contexts, [0, 1, 2, 3], 128 ** -0.5,
                    DECODE["bf16"])
