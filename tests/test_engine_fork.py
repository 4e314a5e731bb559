"""Forks, compaction and log probabilities in the engine's host logic, with
stand-in runners (CPU, no kernels): block ownership and copies of a fork, the
moves of a compaction with its prefix cache, what the step loop records, and
the asyncio frontend's forks.
"""

import asyncio
import random

import pytest

from microinfer_amd.engine.async_engine import AsyncEngine, BackpressureError
from microinfer_amd.engine.config import SampleParameter
from microinfer_amd.engine.llm_engine import LLMEngine
from microinfer_amd.engine.sequence import SequenceStatus, TokenLogprob
from microinfer_amd.layer.hip_shared_decode import (least_shared_positions,
                                                    prefer_shared_decode, shared_groups,
                                                    shared_order)


class PoolRunner:
    """Samples a function of the tokens and keeps a pool of them: row ``p`` of a
    sequence's table holds ``(tokens up to p)``, checked for every cached row."""

    def __init__(self, block_size, width=97):
        self.block_size, self.width = block_size, width
        self.pool = {}
        self.copies = []
        self.asked = {}
        self.fail_copy = False

    def run(self, seqs, is_prefill):
        out = []
        for s in seqs:
            start = s.num_cached_tokens if is_prefill else len(s) - 1
            for p in range(start):
                assert self.pool[self._slot(s, p)] == tuple(s[:p + 1]), "a cached row is wrong"
            for p in range(start, start + s.num_scheduled_tokens):
                self.pool[self._slot(s, p)] = tuple(s[:p + 1])
            token = 100 + (sum(s.token_ids) * 7 + s.seq_id) % self.width
            out.append(token)
            if s.sampling.logprobs is not None:
                self.asked[s.seq_id] = TokenLogprob(token, -float(len(s)), ())
        return out

    def _slot(self, s, p):
        return s.block_table[p // self.block_size], p % self.block_size

    def copy_blocks(self, src, dst, tokens=None):
        if self.fail_copy:
            raise RuntimeError("copy failed")
        tokens = tokens or [self.block_size] * len(src)
        self.copies.append((src, dst, tokens))
        before = dict(self.pool)
        for s, d, n in zip(src, dst, tokens):
            for r in range(n):
                self.pool[d, r] = before.get((s, r))

    def take_logprobs(self):
        taken, self.asked = self.asked, {}
        return taken


def make(scheduler_factory, **limits):
    values = dict(num_blocks=16, max_num_seqs=8, max_num_batched_tokens=16, max_model_len=60)
    values.update(limits)
    scheduler, manager = scheduler_factory(**values)
    runner = PoolRunner(manager.block_size)
    return LLMEngine(scheduler, runner), runner, manager


def params(n, **values):
    return SampleParameter(max_tokens=n, ignore_eos=True, **values)


def run_out(engine):
    while not engine.is_finished():
        engine.step()


def refs(manager):
    return {b.block_id: b.ref_count for b in manager.blocks if b.ref_count}


@pytest.mark.parametrize("prompt,steps", [(6, 1), (8, 1), (9, 1), (3, 5), (4, 1), (4, 2), (1, 1)])
def test_fork_shares_full_blocks_and_copies_the_last(scheduler_factory, sequence_cls, prompt,
                                                     steps):
    engine, runner, manager = make(scheduler_factory)
    seq = sequence_cls(list(range(1, prompt + 1)), params(20))
    engine.add_request(seq)
    for _ in range(steps):
        engine.step()
    cached = seq.num_cached_tokens
    assert cached == len(seq) - 1
    full, rest = divmod(cached, 4)
    children = engine.fork(seq.seq_id, 3)
    assert len({c.seq_id for c in children} | {seq.seq_id}) == 4
    for c in children:
        assert c.token_ids == seq.token_ids and c.token_ids is not seq.token_ids
        assert c.num_prompt_tokens == prompt and c.num_cached_tokens == cached
        assert c.status is SequenceStatus.RUNNING and not c.is_prefill and c.block_size == 4
        assert c.block_table[:full] == seq.block_table[:full]
        assert len(c.block_table) == full + (rest > 0)
    last = [s.block_table[full] for s in [seq, *children] if rest]
    assert len(set(last)) == len(last)
    if rest:
        assert runner.copies == [([seq.block_table[full]] * 3, last[1:], [rest] * 3)]
    else:
        assert runner.copies == []
    for b in seq.block_table[:full]:
        assert manager.blocks[b].ref_count == 4
    run_out(engine)  # the runner checks every cached row of every step
    outs = [s.completion_token_ids for s in [seq, *children]]
    assert all(len(o) == 20 and o[:steps] == outs[0][:steps] for o in outs)
    assert len({tuple(o) for o in outs}) > 1
    assert not manager.used_block_ids and refs(manager) == {}


def test_fork_refusals_change_nothing(scheduler_factory, sequence_cls):
    engine, runner, manager = make(scheduler_factory, num_blocks=3)
    seq = sequence_cls([1, 2, 3, 4, 5], params(6))
    engine.add_request(seq)
    with pytest.raises(ValueError, match="not running"):
        engine.fork(seq.seq_id)
    engine.step()
    before = refs(manager), set(manager.free_block_ids)
    with pytest.raises(RuntimeError, match="no free blocks"):
        engine.fork(seq.seq_id, 2)  # one block is free, two would be needed
    for n in (0, -1, 1.5, True and 0):
        with pytest.raises(ValueError):
            engine.fork(seq.seq_id, n)
    with pytest.raises(ValueError, match="not running"):
        engine.fork(seq.seq_id + 1000)
    with pytest.raises(ValueError, match="max_tokens"):
        engine.fork(seq.seq_id, 1, params(1))  # it has one token already
    runner.fail_copy = True
    with pytest.raises(RuntimeError, match="copy failed"):
        engine.fork(seq.seq_id)
    runner.fail_copy = False
    assert (refs(manager), set(manager.free_block_ids)) == before
    assert list(engine.scheduler.running) == [seq] and runner.copies == []
    engine.scheduler.schedule()
    with pytest.raises(RuntimeError, match="between steps"):
        engine.fork(seq.seq_id)
    with pytest.raises(RuntimeError, match="between steps"):
        engine.compact()


def test_forks_survive_preemption_and_abort(scheduler_factory, sequence_cls):
    engine, runner, manager = make(scheduler_factory, num_blocks=7, max_num_batched_tokens=30)
    seq = sequence_cls([1, 2, 3, 4, 5, 6], params(12))
    engine.add_request(seq)
    engine.step()
    children = engine.fork(seq.seq_id, 2) + engine.fork(seq.seq_id, 1, params(5))
    assert engine.abort(seq.seq_id)
    run_out(engine)
    assert engine.stats()["num_preemptions"] > 0
    assert [len(c.completion_token_ids) for c in children] == [12, 12, 5]
    assert not manager.used_block_ids


@pytest.mark.parametrize("seed", range(8))
def test_random_forks_aborts_and_compactions(scheduler_factory, sequence_cls, seed):
    rng = random.Random(seed)
    # Either preemptions or prompts in chunks: with both, a preempted request can
    # wait for ever behind the blocks of a chunked prompt, with or without forks.
    blocks, budget = rng.choice([(12, 400), (24, 400), (160, 5), (160, 16)])
    engine, runner, manager = make(scheduler_factory, num_blocks=blocks,
                                   max_num_batched_tokens=budget,
                                   mixed_batch=rng.random() < 0.7)
    shared = [rng.randrange(1, 9) for _ in range(9)]
    made = []
    for step in range(120):
        if len(made) < 14 and rng.random() < 0.3:
            prompt = shared[:rng.randrange(9)] + [rng.randrange(1, 9)
                                                  for _ in range(rng.randrange(1, 8))]
            made.append(sequence_cls(prompt, params(rng.randrange(1, 14))))
            engine.add_request(made[-1])
        running = [s.seq_id for s in engine.scheduler.running]
        if running and len(made) < 14 and rng.random() < 0.3:
            n = rng.randrange(1, 4)
            try:
                made += engine.fork(rng.choice(running), n, params(rng.randrange(14, 20)))
            except RuntimeError:
                pass
        if running and rng.random() < 0.05:
            engine.abort(rng.choice(running))
        if rng.random() < 0.3:
            moved = engine.compact()
            used = sorted(manager.used_block_ids)
            assert used == list(range(len(used))) and moved >= 0
        if not engine.is_finished():
            engine.step()
        tables = [s.block_table for s in [*engine.scheduler.waiting, *engine.scheduler.running]]
        counted = {}
        for b in (b for t in tables for b in t):
            counted[b] = counted.get(b, 0) + 1
        assert counted == refs(manager) and set(counted) == manager.used_block_ids
        assert set(manager.free_block_ids) | set(counted) == set(range(len(manager.blocks)))
        assert not set(manager.free_block_ids) & set(counted)
        for h, b in manager.hash_to_block_id.items():  # what is cached is findable and right
            assert h in manager._published[b]
    run_out(engine)
    assert not manager.used_block_ids and refs(manager) == {}


def test_compaction_keeps_published_prefixes(scheduler_factory, sequence_cls):
    engine, runner, manager = make(scheduler_factory, num_blocks=12)
    low = sequence_cls([9, 9, 9, 9, 9], params(1))
    keep = sequence_cls(list(range(1, 10)), params(8))
    engine.add_request(low)
    engine.add_request(keep)
    engine.step()  # `low` is done; its blocks 0 and 1 are free, and cached
    assert low.is_finished and min(keep.block_table) >= 2
    cached = len(manager.hash_to_block_id)
    table = list(keep.block_table)
    assert engine.compact() == 2
    assert sorted(keep.block_table) == list(range(len(keep.block_table)))
    assert runner.copies[-1] == (table[-2:], [0, 1], [4, 4]) or \
        sorted(runner.copies[-1][1]) == [0, 1]
    assert len(manager.hash_to_block_id) == cached - 1  # low's prefix went, keep's stays
    assert engine.compact() == 0
    follow = sequence_cls(list(range(1, 10)) + [5], params(2))
    engine.add_request(follow)
    engine.step()
    assert manager.prefix_cache_hit_blocks == 2
    run_out(engine)


def test_a_failing_compaction_leaves_nothing_behind(scheduler_factory, sequence_cls):
    engine, runner, manager = make(scheduler_factory, num_blocks=12)
    low = sequence_cls([9, 9, 9, 9, 9], params(1))
    keep = sequence_cls(list(range(1, 10)), params(8))
    for seq in (low, keep):
        engine.add_request(seq)
    engine.step()
    late = sequence_cls(list(range(1, 10)), params(2))
    engine.add_request(late)  # holds no blocks
    runner.fail_copy = True
    with pytest.raises(RuntimeError, match="copy failed"):
        engine.compact()
    assert keep.is_finished and keep.finish_reason == "abort" and not manager.used_block_ids
    assert not manager.hash_to_block_id
    run_out(engine)  # the runner would see a wrong block
    assert len(late.completion_token_ids) == 2 and manager.prefix_cache_hit_blocks == 0


def test_logprobs_follow_the_kept_tokens(scheduler_factory, sequence_cls):
    engine, runner, _ = make(scheduler_factory, max_num_batched_tokens=4)
    a = sequence_cls([1, 2, 3, 4, 5, 6, 7], params(3, logprobs=2))  # two prompt chunks
    b = sequence_cls([1], params(3))
    engine.add_request(a)
    engine.add_request(b)
    engine.step()
    assert a.logprobs == []  # the first chunk's sample is dropped
    for _ in range(2):
        engine.step()
    child, = engine.fork(a.seq_id)
    assert child.logprobs == a.logprobs and child.logprobs is not a.logprobs
    run_out(engine)
    for s in (a, child):
        assert [x.token_id for x in s.logprobs] == s.completion_token_ids
        assert [x.logprob for x in s.logprobs] == [-7.0, -8.0, -9.0]
    assert b.logprobs == []


def test_sampling_values_are_checked():
    for bad in (-1, 33, 1.0, True, "3"):
        with pytest.raises(ValueError, match="logprobs"):
            SampleParameter(logprobs=bad)
    assert SampleParameter(logprobs=0).logprobs == 0
    assert SampleParameter().logprobs is None


def test_async_forks_stream_from_the_tokens_so_far(scheduler_factory, sequence_cls):
    engine, runner, manager = make(scheduler_factory)

    async def scenario():
        frontend = AsyncEngine(engine, max_waiting=3)
        request = await frontend.add_request([1, 2, 3], params(12))
        stream = frontend.stream(request)
        first = await anext(stream)
        with pytest.raises(BackpressureError):
            await frontend.fork(request, 3)
        forks = await frontend.fork(request, 2, params(15))
        with pytest.raises(BackpressureError):
            await frontend.add_request([4], params(1))
        with pytest.raises(TypeError):
            await frontend.fork(request, 1, {"max_tokens": 1})
        with pytest.raises(ValueError):
            await frontend.fork(request, 0)
        outs = [await frontend.collect(f) for f in forks]
        async for event in stream:
            last = event
        assert len(last.token_ids) == 12 and all(len(o.token_ids) == 15 for o in outs)
        assert all(o.token_ids[:1] == first.token_ids[:1] for o in outs)
        with pytest.raises(ValueError, match="not running"):
            await frontend.fork(request)  # it has finished
        assert frontend.stats()["active_requests"] == 0
        again = await frontend.generate([1, 2], params(2))  # the room came back
        request = await frontend.add_request([1, 2, 3], params(30))
        stream = frontend.stream(request)
        await anext(stream)
        task = asyncio.ensure_future(frontend.fork(request, 2))
        await asyncio.sleep(0)
        task.cancel()
        with pytest.raises(asyncio.CancelledError):
            await task
        async for event in stream:
            pass
        assert len(event.token_ids) == 30
        assert frontend._reserved == 0 and not frontend._channels
        assert len(again.token_ids) == 2
        await frontend.stop()
        assert not manager.used_block_ids

    asyncio.run(scenario())


def test_async_requests_carry_their_logprobs(scheduler_factory):
    engine, _, _ = make(scheduler_factory)

    async def scenario():
        frontend = AsyncEngine(engine)
        plain = await frontend.generate([1, 2], params(3))
        assert plain.logprobs == ()
        request = await frontend.add_request([1, 2, 3], params(6, logprobs=0))
        stream = frontend.stream(request)
        event = await anext(stream)
        assert len(request.logprobs) >= len(event.token_ids)
        fork, = await frontend.fork(request)
        for out in (await frontend.collect(fork), request):
            async for event in stream:
                pass
            assert [e.token_id for e in out.logprobs] == list(out.token_ids)
            assert [e.logprob for e in out.logprobs] == [-3.0, -4.0, -5.0, -6.0, -7.0, -8.0]
        await frontend.stop()

    asyncio.run(scenario())


def test_shared_groups_of_neighbours():
    a = list(range(10))
    tables = [a + [20], a + [21, 22], a[:8] + [23, 24], [50, 51], [50, 52], [60]]
    lens = [4 * len(t) for t in tables]
    # Ten blocks shared by two, eight by three; a single block by the next
    # two; nothing by the last.
    assert shared_groups(tables, lens, 4) == ([0, 3, 5, 6], [8, 1, 0])
    # Blocks must be whole in every context.
    assert shared_groups(tables[:2], [40, 39], 4) == ([0, 2], [9])
    assert shared_groups(tables[:2], [3, 44], 4) == ([0, 1, 2], [0, 0])
    # A sequence that shares little does not take it from the others.
    assert shared_groups([a, a, a[:3] + [9]], [40, 40, 16], 4) == ([0, 2, 3], [10, 0])
    # Long contexts behind a short common beginning.
    b, c = [1, 2] + list(range(100, 140)), [1, 2] + list(range(200, 230))
    assert shared_groups([b, c], [168, 128], 4) == ([0, 2], [2])
    # The next neighbour shares more.
    assert shared_groups([b, c, c + [7]], [168, 128, 132], 4) == ([0, 1, 3], [0, 32])
    assert shared_groups([], [], 4) == ([0], [])
    assert shared_groups([a], [40], 4) == ([0, 1], [0])


def test_shared_order_puts_common_beginnings_together():
    a = list(range(30))
    tables = [a[:20] + [40], [50], a[:5] + [60, 61], [], a[:20] + [41, 42], [50, 51],
              a[:5] + [70], a[:5] + [60, 62], a[:12] + [80]]
    order = shared_order(tables)
    assert sorted(order) == list(range(9))
    assert order[:6] in ([0, 4, 8, 2, 7, 6], [0, 4, 8, 6, 2, 7]) and set(order[6:8]) == {1, 5}
    starts, shared = shared_groups([tables[i] for i in order], [4 * len(tables[i]) for i in order],
                                   4)
    members = [set(order[s:e]) for s, e in zip(starts, starts[1:])]
    assert [(m, n) for m, n in zip(members, shared) if n] == [
        ({0, 4, 8}, 12), ({2, 7, 6}, 5), ({1, 5}, 1)]
    assert shared_order([]) == []


@pytest.mark.parametrize("seed", range(20))
def test_groups_share_what_they_say(seed):
    rng = random.Random(seed)
    tables = [[rng.randrange(3) for _ in range(rng.randrange(9))] for _ in range(12)]
    contexts = [rng.randrange(max(0, 4 * len(t) - 3), 4 * len(t) + 1) for t in tables]
    order = shared_order(tables)
    assert sorted(order) == list(range(12))
    tables, contexts = [tables[i] for i in order], [contexts[i] for i in order]
    starts, shared = shared_groups(tables, contexts, 4)
    assert starts[0] == 0 and starts[-1] == 12 and sorted(set(starts)) == starts
    for g, n in enumerate(shared):
        members = range(starts[g], starts[g + 1])
        assert (n == 0) == (len(members) == 1)
        assert len({tuple(tables[i][:n]) for i in members}) == 1
        assert all(4 * n <= contexts[i] and n <= len(tables[i]) for i in members)


def test_groups_are_used_where_they_pay():
    assert not prefer_shared_decode([0], [], 16, 8)
    assert not prefer_shared_decode([0, 1, 2], [0, 0], 16, 8)
    assert not prefer_shared_decode([0, 2], [1 << 20], 16, 8)  # pairs never
    least = -(-((1 << 17) + 8192 * 6) // (8 * 16 * 2))  # blocks, two sequences counted
    assert prefer_shared_decode([0, 4, 6], [least, 0], 16, 8)
    assert not prefer_shared_decode([0, 4, 6], [least - 1, 9999], 16, 8)


def test_a_fork_cancelled_when_its_requests_exist_drops_them(scheduler_factory):
    engine, runner, manager = make(scheduler_factory, num_blocks=24)

    async def scenario():
        frontend = AsyncEngine(engine, max_waiting=3)
        request = await frontend.add_request([1, 2, 3], params(40))
        stream = frontend.stream(request)
        await anext(stream)
        settle, tasks = frontend._settle_fork, []

        def settle_and_cancel(*args):
            settle(*args)
            tasks[0].cancel()  # the answer is there, its caller has not run yet

        frontend._settle_fork = settle_and_cancel
        tasks.append(asyncio.ensure_future(frontend.fork(request, 2)))
        with pytest.raises(asyncio.CancelledError):
            await tasks[0]
        frontend._settle_fork = settle
        assert list(frontend._channels) == [request.seq_id] and frontend._reserved == 0
        forks = await frontend.fork(request, 2)  # the room is there at once
        assert len(engine.scheduler.running) == 3  # the dropped ones run no more
        tokens = [len((await frontend.collect(f)).token_ids) for f in forks]
        async for event in stream:
            pass
        assert tokens == [40, 40] and len(event.token_ids) == 40
        assert not frontend._channels
        await frontend.stop()
        assert not manager.used_block_ids

    asyncio.run(scenario())


def test_a_failed_fork_cancelled_by_then_leaves_nothing(scheduler_factory):
    engine, runner, manager = make(scheduler_factory)

    async def scenario():
        frontend = AsyncEngine(engine, max_waiting=3)
        request = await frontend.add_request([1, 2, 3], params(20))
        stream = frontend.stream(request)
        await anext(stream)
        settle, tasks = frontend._settle_fork, []

        def settle_and_cancel(*args):
            settle(*args)
            tasks[0].cancel()

        frontend._settle_fork = settle_and_cancel
        tasks.append(asyncio.ensure_future(frontend.fork(request, 1, params(1))))  # refused
        with pytest.raises(asyncio.CancelledError):
            await tasks[0]
        assert list(frontend._channels) == [request.seq_id] and frontend._reserved == 0
        await frontend.stop()

    asyncio.run(scenario())


def test_preempted_forks_pass_a_chunked_prompt_that_holds_blocks(scheduler_factory, sequence_cls):
    engine, runner, manager = make(scheduler_factory, num_blocks=9, max_num_prefill_tokens=4)
    seq = sequence_cls(list(range(1, 11)), params(24))
    engine.add_request(seq)
    while not seq.num_completion_tokens:
        engine.step()
    forks = engine.fork(seq.seq_id, 4)
    run_out(engine)  # the runner checks every cached row of every step
    assert [len(s.completion_token_ids) for s in [seq, *forks]] == [24] * 5
    assert engine.stats()["num_preemptions"] > 0
    assert not manager.used_block_ids and refs(manager) == {}


@pytest.mark.parametrize("seed", range(40))
def test_preemptions_and_chunked_prompts_together(scheduler_factory, sequence_cls, seed):
    rng = random.Random(seed)
    engine, runner, manager = make(scheduler_factory, num_blocks=rng.choice([9, 12]),
                                   max_num_batched_tokens=rng.choice([5, 16]), max_model_len=36,
                                   max_num_prefill_tokens=rng.choice([3, 400]),
                                   mixed_batch=rng.random() < 0.7)
    made = []
    for _ in range(14):
        prompt = [rng.randrange(1, 9) for _ in range(rng.randrange(1, 15))]
        made.append(sequence_cls(prompt, params(rng.randrange(1, 20))))
        engine.add_request(made[-1])
    for step in range(4000):
        if engine.is_finished():
            break
        engine.step()
        running = [s.seq_id for s in engine.scheduler.running]
        if running and len(made) < 20 and rng.random() < 0.2:
            try:
                made += engine.fork(rng.choice(running), rng.randrange(1, 3), params(20))
            except RuntimeError:
                pass
        held = {b for s in [*engine.scheduler.waiting, *engine.scheduler.running]
                for b in s.block_table}
        assert held == manager.used_block_ids
    assert engine.is_finished()
    assert all(len(s.completion_token_ids) == s.max_tokens or len(s) >= 36 for s in made)
    assert not manager.used_block_ids and refs(manager) == {}


@pytest.mark.parametrize("sequences,hq,hkv,prefix,worth", [
    # Whole steps that were measured (28 layers, block 16): those that gain more
    # than a twentieth, and those that lose.
    (4, 16, 8, 20496, True), (8, 16, 8, 8208, True), (16, 16, 8, 4688, True),
    (64, 16, 8, 2656, True), (8, 16, 8, 2064, False), (64, 16, 8, 672, False),
    (64, 32, 8, 1328, False), (64, 32, 8, 2656, True), (16, 32, 8, 4688, True),
    (64, 64, 8, 1328, False), (64, 64, 8, 5296, True), (16, 64, 8, 1184, False),
    (64, 64, 4, 2656, False), (64, 64, 4, 5296, False), (64, 64, 4, 10576, True),
    (64, 32, 2, 5296, False), (64, 32, 2, 10576, True), (4, 32, 2, 81936, True),
    (4, 64, 4, 20496, True), (4, 32, 2, 40976, True), (64, 16, 16, 1328, True),
    (16, 16, 16, 592, False), (8, 16, 16, 1040, False),
])
def test_the_rule_follows_the_measured_steps(sequences, hq, hkv, prefix, worth):
    assert prefer_shared_decode([0, sequences], [prefix // 16], 16, hkv, hq) is worth
    # Sequences that share nothing beside them only raise what has to be gained.
    if not worth:
        assert not prefer_shared_decode([0, sequences, sequences + 9], [prefix // 16, 0], 16,
                                        hkv, hq)


def test_the_rule_counts_reads_of_row_tiles():
    # 64 rows meet a page at once: 16 sequences of four query heads a KV head.
    def least(sequences, counted):
        return -(-least_shared_positions(sequences, 8, 32) // (16 * counted))

    for sequences, counted in ((3, 1), (16, 14), (17, 14), (32, 29), (33, 29)):
        blocks = least(sequences, counted)
        assert prefer_shared_decode([0, sequences], [blocks], 16, 8, 32)
        assert not prefer_shared_decode([0, sequences], [blocks - 1], 16, 8, 32)
    assert not prefer_shared_decode([0, 2], [1 << 20], 16, 8, 32)
    assert not prefer_shared_decode([0, 1], [1 << 20], 16, 8, 32)
