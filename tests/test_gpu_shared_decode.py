"""Decode over shared pages (mi_shared_decode via layer.hip_shared_decode)
against float64 attention over each sequence's own table.

Tolerance: the weights p round to the cache's type before the product with V,
off by at most half a step h = eps / 2 each, and their sum adds the rounded
ones, which moves an output by at most h * sum p |v - out| / sum p <= h (A +
|out|) with A = sum p |v| / sum p; the output rounds once more, h |out|. The
scores are float32 sums of 128 products, a few 2^-24 of values up to some tens,
which move a weight by less than 2^-15 of itself.
"""

import math
import random

import pytest
import torch

from microinfer_amd.layer.hip_paged_attention import hip_paged_decode
from microinfer_amd.layer.hip_shared_decode import (SharedDecodePlan, hip_shared_decode,
                                                    shared_decode_plan)
from microinfer_amd.runner import capture_graph
from microinfer_amd.worker.kv_cache import KVCache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _assert_close(out, q, keys, values, tables, contexts, scale):
    """``out`` against float64 attention, rows of invalid blocks left out."""
    half = torch.finfo(q.dtype).eps / 2
    blocks, block, hkv, dim = keys.shape
    share = q.shape[1] // hkv
    assert out.shape == q.shape and out.dtype == q.dtype
    for s, c in enumerate(contexts):
        ids = tables[s, : -(-c // block)].long()
        there = ((ids >= 0) & (ids < blocks)).repeat_interleave(block)[:c]
        ids = ids.clamp(0, blocks - 1)
        k = keys[ids].flatten(0, 1)[:c][there].double().transpose(0, 1).contiguous()
        v = values[ids].flatten(0, 1)[:c][there].double().transpose(0, 1).contiguous()
        if k.shape[1] == 0:
            assert not out[s].any()
            continue
        p = torch.softmax(torch.matmul(q[s].double().view(hkv, share, dim),
                                       k.transpose(1, 2).contiguous()) * scale, -1)
        want = torch.matmul(p, v).view(-1, dim)
        size = torch.matmul(p, v.abs()).view(-1, dim)
        tol = half * (size + 2 * want.abs()) + 2.0 ** -15 * size
        err = (out[s].double() - want).abs()
        assert (err <= tol).all(), f"sequence {s}: {(err / tol).max()} times the tolerance"


class Batch:
    """Random tables whose groups share their first pages."""

    def __init__(self, groups, *, hq=16, hkv=8, dim=128, block=16, dtype=torch.bfloat16,
                 layout="paired", seed=0, extra=2, width_extra=0):
        rng = random.Random(seed)
        self.block = block
        self.contexts, self.starts, self.shared, rows = [], [0], [], []
        pages = sum(shared + sum(-(-c // block) for c in ctx) for shared, ctx in groups) + extra
        ids = rng.sample(range(pages), pages)
        for shared, ctx in groups:
            head = [ids.pop() for _ in range(shared)]
            for c in ctx:
                need = -(-c // block)
                rows.append((head + [ids.pop() for _ in range(max(0, need - shared))])
                            [:max(need, shared)])
            self.contexts += ctx
            self.starts.append(len(self.contexts))
            self.shared.append(shared)
        width = max(max(map(len, rows)), 1) + width_extra
        self.tables = _ints([r + [-1] * (width - len(r)) for r in rows])
        cache = KVCache(1, pages, block, hkv, dim, dtype=dtype, device=DEV, layout=layout)
        gen = torch.Generator(device=DEV).manual_seed(seed)
        cache.keys.copy_(torch.randn(cache.keys.shape, generator=gen, device=DEV))
        cache.values.copy_(torch.randn(cache.values.shape, generator=gen, device=DEV))
        self.keys, self.values = cache.keys[0], cache.values[0]
        self.q = torch.randn(len(rows), hq, dim, generator=gen, device=DEV).to(dtype)

    def plan(self, starts=None, shared=None, contexts=None):
        return shared_decode_plan(
            _ints(self.contexts) if contexts is None else contexts,
            _ints(self.starts if starts is None else starts),
            _ints(self.shared if shared is None else shared), num_q_heads=self.q.shape[1],
            num_kv_heads=self.keys.shape[2], head_dim=self.q.shape[2], dtype=self.q.dtype,
            block_size=self.block, block_table_width=self.tables.shape[1])

    def run(self, plan=None, scale=None):
        return hip_shared_decode(self.q, self.keys, self.values, self.tables,
                                 _ints(self.contexts), plan=plan or self.plan(), scale=scale)

    def check(self, plan=None, scale=None):
        out = self.run(plan, scale)
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        _assert_close(out, self.q, self.keys, self.values, self.tables, self.contexts, scale)
        return out


def _tails(prefix, n, most, seed):
    rng = random.Random(seed)
    return [prefix + rng.randint(1, most) for _ in range(n)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (32, 8), (8, 8), (12, 4), (64, 4), (40, 8), (2, 1)])
def test_groups_of_every_size(dtype, hq, hkv):
    groups = [(37, _tails(592, 4, 50, 1)), (2, _tails(32, 1, 100, 2)),
              (70, _tails(1120, 21, 90, 3)), (1, _tails(16, 2, 20, 4)),
              (0, _tails(0, 3, 700, 5)), (9, _tails(144, 70, 33, 6))]
    Batch(groups, hq=hq, hkv=hkv, dtype=dtype, seed=hq + hkv).check()


@pytest.mark.parametrize("block", [16, 32, 256])
@pytest.mark.parametrize("layout", ["paired", "head_major", "token_major"])
def test_block_sizes_and_layouts(block, layout):
    groups = [(5, _tails(5 * block, 6, 3 * block, 1)), (1, _tails(block, 3, 5, 2))]
    Batch(groups, block=block, layout=layout, seed=block, width_extra=3).check()


def test_a_long_prefix_and_many_sequences():
    Batch([(500, _tails(8000, 16, 300, 1))], hq=32).check()
    Batch([(40, _tails(640, 3, 9, s)) for s in range(150)], hq=8, seed=3).check()
    Batch([(2, _tails(32, 1000, 3, 9))], hkv=1, hq=2, seed=4).check()


def test_contexts_at_the_ends_of_pages():
    # Nothing behind the shared pages, one position behind, one position in all.
    Batch([(4, [64, 64, 65, 80]), (1, [16, 16]), (0, [1, 1, 2])]).check()


def test_shared_pages_that_do_not_fit_every_context():
    # 10 columns agree, but one sequence ends inside the third page: two count.
    batch = Batch([(10, [400, 45, 161, 160]), (3, [48, 0, 50])])
    out = batch.check()
    assert not out[5].any()  # no position: zeros
    same = batch.check(batch.plan(shared=[2, 0]))
    assert torch.equal(out, same)
    # Fewer columns than agree, negative and none.
    batch.check(batch.plan(shared=[1, -5]))
    batch.check(batch.plan(shared=[0, 2 ** 30]))


def test_sequences_outside_every_group():
    batch = Batch([(6, _tails(96, 5, 40, 1)), (8, _tails(128, 4, 40, 2))])
    batch.check(batch.plan(starts=[5, 9], shared=[8]))
    batch.check(batch.plan(starts=[1, 4], shared=[6]))
    batch.check(batch.plan(starts=[0], shared=[]))
    batch.check(batch.plan(starts=[], shared=[]))
    batch.check(batch.plan(starts=[0, 5, 5, 5, 900], shared=[6, 3, 3, 8]))


def test_invalid_blocks_are_masked_and_stale_rows_never_read():
    batch = Batch([(6, _tails(96, 5, 40, 1)), (2, [40, 40, 33])], extra=3)
    used = {b for row, c in zip(batch.tables.tolist(), batch.contexts)
            for b in row[: -(-c // batch.block)]}
    spare = next(b for b in range(batch.keys.shape[0]) if b not in used)
    for pool in (batch.keys, batch.values):
        pool[spare] = math.nan
        for row, c in zip(batch.tables.tolist(), batch.contexts):
            if c % batch.block:  # rows behind the last position
                pool[row[c // batch.block], c % batch.block:] = math.nan
    batch.tables[:5, 2] = -1                 # inside the shared pages
    batch.tables[1, 6] = batch.keys.shape[0]  # a whole page of one sequence's own
    batch.tables[5:, :] = -1                 # nothing left at all
    batch.check()


def test_large_scores_and_scale():
    batch = Batch([(20, _tails(320, 9, 60, 1))])
    batch.q *= 20
    batch.check(scale=0.11)
    batch.check(scale=0.0)


def test_strided_queries_and_tables():
    batch = Batch([(20, _tails(320, 9, 60, 1))])
    wide = torch.randn(9, 40, 128, device=DEV).to(torch.bfloat16)
    batch.q = wide[:, 4:20]
    wide_tables = torch.full((9, batch.tables.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide_tables[:, :-5] = batch.tables
    batch.tables = wide_tables[:, : batch.tables.shape[1]]
    batch.check()


def test_offsets_past_32_bits():
    batch = Batch([(3, [50, 60, 49])])
    pool = KVCache(1, 2 * 65536, 16, 8, 128, dtype=torch.bfloat16, device=DEV)  # 8 GiB
    shift = pool.num_blocks - batch.keys.shape[0]
    pool.keys[0, shift:] = batch.keys
    pool.values[0, shift:] = batch.values
    want = batch.run()
    batch.keys, batch.values = pool.keys[0], pool.values[0]
    batch.tables = torch.where(batch.tables >= 0, batch.tables + shift, batch.tables)
    assert torch.equal(batch.run(), want)


def test_repeatable_and_on_another_stream():
    batch = Batch([(60, _tails(960, 12, 200, 1))])
    first = batch.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = batch.run()
    torch.cuda.synchronize()
    assert torch.equal(first, again) and torch.equal(first, batch.run())


def test_captured_steps_follow_the_lengths_and_groups():
    batch = Batch([(20, _tails(320, 4, 100, 1)), (4, _tails(64, 4, 100, 2))])
    contexts, starts, shared = (_ints(x) for x in (batch.contexts, batch.starts, batch.shared))
    sizes = dict(num_q_heads=16, num_kv_heads=8, head_dim=128, dtype=torch.bfloat16,
                 block_size=16, block_table_width=batch.tables.shape[1])

    def step():
        plan = shared_decode_plan(contexts, starts, shared, **sizes)
        return hip_shared_decode(batch.q, batch.keys, batch.values, batch.tables, contexts,
                                 plan=plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph, stream=side):
        out = step()
    most = list(batch.contexts)
    for replay, (groups, pages) in enumerate([([0, 4, 8], [20, 4]), ([0, 3, 8], [20, 0]),
                                              ([4, 8, 8], [3, 1]), ([0, 4, 8], [20, 4])]):
        batch.contexts = [c - 7 * replay for c in most]
        contexts.copy_(_ints(batch.contexts))
        starts.copy_(_ints(groups))
        shared.copy_(_ints(pages))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        _assert_close(out, batch.q, batch.keys, batch.values, batch.tables, batch.contexts,
                      128 ** -0.5)


@pytest.mark.parametrize("dtype,dim,block,hq,hkv", [
    (torch.float32, 128, 16, 4, 2), (torch.bfloat16, 64, 16, 4, 2), (torch.float16, 128, 8, 4, 2),
])
def test_other_shapes_take_the_ordinary_kernels(dtype, dim, block, hq, hkv):
    batch = Batch([(6, _tails(6 * block, 5, 40, 1))], dtype=dtype, dim=dim, block=block, hq=hq,
                  hkv=hkv)
    plan = batch.plan()
    assert not plan.shared
    want = hip_paged_decode(batch.q, batch.keys, batch.values, batch.tables,
                            _ints(batch.contexts))
    assert torch.equal(batch.run(plan), want)


def test_no_sequences():
    batch = Batch([(3, [50, 60])])
    plan = shared_decode_plan(_ints([]), _ints([0]), _ints([]), num_q_heads=16, num_kv_heads=8,
                              head_dim=128, dtype=torch.bfloat16, block_size=16,
                              block_table_width=4)
    out = hip_shared_decode(batch.q[:0], batch.keys, batch.values, batch.tables[:0, :4],
                            _ints([]), plan=plan)
    assert out.shape == (0, 16, 128)


def test_refusals():
    batch = Batch([(3, [50, 60])])
    plan = batch.plan()
    for bad in (None, plan.buffer, SharedDecodePlan(plan.buffer, True, ())):
        with pytest.raises(ValueError, match="plan"):
            hip_shared_decode(batch.q, batch.keys, batch.values, batch.tables,
                              _ints(batch.contexts), plan=bad)
    with pytest.raises(ValueError, match="plan"):
        hip_shared_decode(batch.q, batch.keys, batch.values, batch.tables[:, :-1],
                          _ints(batch.contexts), plan=plan)
    with pytest.raises(ValueError, match="one entry"):
        batch.plan(starts=[0, 1, 2])
    with pytest.raises(ValueError, match="entry per request"):
        hip_shared_decode(batch.q, batch.keys, batch.values, batch.tables, _ints([1]), plan=plan)


def test_tables_without_columns():
    # No sequence has a position: zeros, whatever the groups say.
    batch = Batch([(1, [16, 20])])
    contexts, tables = _ints([0, 0]), batch.tables[:, :0]
    plan = shared_decode_plan(contexts, _ints([0, 2]), _ints([1]), num_q_heads=16, num_kv_heads=8,
                              head_dim=128, dtype=torch.bfloat16, block_size=16,
                              block_table_width=0)
    for tab in (tables, tables.clone()):
        out = hip_shared_decode(batch.q, batch.keys, batch.values, tab, contexts, plan=plan)
        assert out.shape == batch.q.shape and not out.any()


def test_the_most_sequences():
    # 4096 sequences: pairs, one group, and groups of one.
    batch = Batch([(1, [17 + i % 5, 18]) for i in range(2048)], hkv=1, hq=2)
    batch.check()
    one = Batch([(1, [16 + i % 7 for i in range(4096)])], hkv=1, hq=2)
    one.check()
    alone = one.plan(starts=list(range(4097)), shared=[1] * 4096)
    one.check(alone)
    with pytest.raises(ValueError, match="at most 4096 groups"):
        one.plan(starts=list(range(4098)), shared=[0] * 4097)


def test_lengths_of_other_types_and_strides():
    batch = Batch([(6, _tails(96, 5, 40, 1))])
    want = batch.check()
    wide = torch.stack([_ints(batch.contexts), _ints([0] * 5)], 1).long()[:, 0]
    tables = batch.tables.t().contiguous().t()  # columns outermost
    got = hip_shared_decode(batch.q, batch.keys, batch.values, tables, wide,
                            plan=batch.plan(contexts=wide))
    assert torch.equal(got, want)


def test_unaligned_queries():
    batch = Batch([(6, _tails(96, 5, 40, 1))])
    want = batch.check()
    wide = torch.zeros(5, 16, 131, device=DEV, dtype=torch.bfloat16)
    wide[:, :, 3:] = batch.q
    flat = torch.zeros(batch.q.numel() + 1, device=DEV, dtype=torch.bfloat16)
    flat[1:] = batch.q.flatten()
    for q in (wide[:, :, 3:], flat[1:].view_as(batch.q)):
        got = hip_shared_decode(q, batch.keys, batch.values, batch.tables, _ints(batch.contexts),
                                plan=batch.plan())
        assert torch.equal(got, want) and got.is_contiguous()


def test_two_graphs_and_eager_calls_share_nothing():
    batches = [Batch([(60, _tails(960, 12, 200, s))], hq=32, seed=s) for s in (1, 2, 3)]
    want = [batch.check() for batch in batches]
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs, kept = [], [], []
    for batch, stream in zip(batches, streams):
        args = [_ints(x) for x in (batch.contexts, batch.starts, batch.shared)]
        kept.append(args)  # the graph reads them
        sizes = dict(num_q_heads=32, num_kv_heads=8, head_dim=128, dtype=torch.bfloat16,
                     block_size=16, block_table_width=batch.tables.shape[1])

        def step(batch=batch, args=args, sizes=sizes):
            return hip_shared_decode(batch.q, batch.keys, batch.values, batch.tables, args[0],
                                     plan=shared_decode_plan(*args, **sizes))

        if len(graphs) == 2:
            break
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with capture_graph(graph, stream=stream):
            outs.append(step())
        graphs.append(graph)
    for _ in range(10):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = [step() for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert all(torch.equal(x, want[2]) for x in eager)


def _exact(batch, s, scale):
    """Sequence s in float64: its output and the same of |v|."""
    c, (_, _, hkv, dim) = batch.contexts[s], batch.keys.shape
    ids = batch.tables[s, : -(-c // batch.block)].long()
    k, v = (x[ids].flatten(0, 1)[:c].double().transpose(0, 1).contiguous()
            for x in (batch.keys, batch.values))
    q = batch.q[s].double().view(hkv, -1, dim)
    p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * scale, -1)
    return torch.matmul(p, v).view(-1, dim), torch.matmul(p, v.abs()).view(-1, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups", [
    [(2, _tails(32, 12, 30, 1)), (1, _tails(16, 7, 9, 2))], [(0, _tails(0, 5, 70, 3))],
    [(30, _tails(480, 16, 90, 4))],
])
def test_an_output_is_off_by_its_own_rounding(dtype, groups):
    # A weight is held to 2^-16 of itself in bf16 and 2^-22 in fp16 (two
    # roundings of half a step each), scores and exponentials to less than 2^-16
    # of a weight (float32 sums of values up to some tens): beyond the output's
    # rounding nothing but that remains.
    batch = Batch(groups, hq=32, dtype=dtype, seed=5)
    out = batch.run().double()
    half = torch.finfo(dtype).eps / 2
    rest = 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -16 + 2.0 ** -22
    for s in range(len(batch.contexts)):
        want, size = _exact(batch, s, 128 ** -0.5)
        over = (out[s] - want).abs() - (half * want.abs() + rest * (1 + half) * size)
        assert (over <= 0).all(), f"sequence {s}: {over.max()} over"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_small_weights_add_up(dtype):
    # One position of value 0 outweighs each of the others 2^26 times: what they
    # leave is the output, within the bounds above.
    batch = Batch([(3, [64, 49, 50])], hq=32, dtype=dtype, seed=6)
    for pool, fill in ((batch.keys, 0.0), (batch.values, 1024.0)):  # outputs stay normal numbers
        pool.fill_(fill)
    batch.q.fill_(1.0)
    scale = 26 * math.log(2) / 128
    at = batch.tables[:, 0].long()  # the first position, shared or not
    batch.keys[at, 0] = 1.0
    batch.values[at, 0] = 0.0
    out = batch.run(scale=scale).double()
    half = torch.finfo(dtype).eps / 2
    for s, c in enumerate(batch.contexts):
        want, size = _exact(batch, s, scale)
        assert (want > 0).all()
        assert ((out[s] - want).abs() <= half * want + 2.0 ** -15 * (1 + half) * size).all()


def _nan_rows(batch, plan=None):
    """Which outputs are NaN, by the kernel and by float64 attention."""
    out = batch.run(plan)
    want = torch.stack([_exact(batch, s, 128 ** -0.5)[0] for s in range(len(batch.contexts))])
    assert bool((out.isnan() == want.isnan()).all())
    fine = want.isfinite()
    half = torch.finfo(out.dtype).eps / 2
    size = want[fine].abs().max()
    assert ((out.double() - want)[fine].abs() <= half * want[fine].abs() + 2 ** -13 * size).all()
    return out.isnan()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("members,hq", [(3, 8), (3, 32), (20, 16), (20, 32)])
def test_nan_reaches_the_output(dtype, members, hq):
    # Groups of few and of many query rows; one sequence has a single position
    # behind the shared pages, one none.
    prefix = 20 * 16
    ctx = [prefix + 1, prefix] + _tails(prefix, members - 2, 40, 3)

    def batch(seed):
        return Batch([(20, ctx), (0, [1, 40])], hq=hq, dtype=dtype, seed=seed)

    one = batch(1)
    one.q[2, 3, 7] = math.nan                        # one head of one sequence
    one.q[members, 1, 0] = math.nan                  # and of one that has a single position
    nan = _nan_rows(one)
    assert nan[2, 3].all() and nan[members, 1].all() and nan.sum() == 2 * 128

    one = batch(2)
    own = int(one.tables[0, 20])                     # a page whose only position is NaN
    one.keys[own, 0] = math.nan
    nan = _nan_rows(one)
    assert nan[0].all() and not nan[1:].any()

    one = batch(3)
    one.keys[int(one.tables[0, 9]), 5, 1] = math.nan  # one KV head of a shared position
    share = hq // 8
    nan = _nan_rows(one)
    assert nan[:members, share:2 * share].all() and nan.sum() == members * share * 128

    one = batch(4)
    one.keys[one.tables[0, :20].long()] = math.nan   # every shared position
    one.values[int(one.tables[members + 1, 1]), 3, 2, 9] = math.nan  # one value elsewhere
    nan = _nan_rows(one)
    assert nan[:members].all() and nan[members:].sum() == share


def test_workspaces_end_with_their_plan():
    # One plan's calls on several streams; nothing stays allocated behind it.
    batch = Batch([(60, _tails(960, 12, 200, 1))], hq=32)
    want = batch.check()
    plan = batch.plan()
    contexts = _ints(batch.contexts)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    streams, outs = [torch.cuda.Stream() for _ in range(6)], []
    for stream in streams:
        with torch.cuda.stream(stream):
            for _ in range(2):
                outs.append(hip_shared_decode(batch.q, batch.keys, batch.values, batch.tables,
                                              contexts, plan=plan))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)
    del plan, outs
    assert torch.cuda.memory_allocated() <= before
