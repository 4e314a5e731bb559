"""Forked requests on the device, as a program uses them: page copies at the
fork, decode that reads the shared pages once, the log probability of every
kept token, and compaction between steps, in one engine.

Checked against the dense float64 oracle, teacher-forced: greedy tokens as in
the engine's other tests, and each recorded log probability against the
oracle's log-softmax at its position. If a logit is off by at most e, the
deficit of a greedy token (a difference of two logits) and a log probability
(a logit and a log-sum-exp) are off by at most 2e, so both take the bounds that
the engine's tests set on the deficits: 1e-4 in float32, 0.1 for bfloat16.
"""

import numpy as np
import pytest
import torch

from microinfer_amd.engine import model_runner as runner_module
from microinfer_amd.engine.blockmanager import BlockManager
from microinfer_amd.engine.config import EngineConfig, SampleParameter
from microinfer_amd.engine.llm_engine import LLMEngine
from microinfer_amd.engine.model import QwenConfig, Qwen3Model
from microinfer_amd.engine.model_runner import ModelRunner
from microinfer_amd.engine.scheduler import Scheduler
from microinfer_amd.engine.sequence import Sequence
from microinfer_amd.layer import paged_attention
from oracle.qwen3_dense import forward_logits, weights_f64

pytestmark = pytest.mark.gpu

TINY = QwenConfig(vocab_size=512, hidden_dim=128, MLP_inter_dim=256, num_q_head=4,
                  num_kv_head=2, head_dim=32, num_hidden_layer=2, max_pos_embed=512)
WIDE = QwenConfig(vocab_size=4096, hidden_dim=1024, MLP_inter_dim=2048, num_q_head=16,
                  num_kv_head=8, head_dim=128, num_hidden_layer=2, max_pos_embed=1024)


@pytest.fixture(scope="module")
def tiny_model():
    return Qwen3Model(TINY, dtype=torch.float32, device="cuda", seed=0, init_std=0.1)


@pytest.fixture(scope="module")
def wide_model():
    return Qwen3Model(WIDE, dtype=torch.bfloat16, device="cuda", seed=7, init_std=0.05)


@pytest.fixture
def shared_calls(monkeypatch):
    """Every sharing step is worth it; counts the launches' Python calls."""
    calls = []
    launch = paged_attention.hip_shared_decode

    def counted(query, *args, **kwargs):
        calls.append(query.shape[0])
        return launch(query, *args, **kwargs)

    monkeypatch.setattr(paged_attention, "hip_shared_decode", counted)
    monkeypatch.setattr(runner_module, "least_shared_positions", lambda *sizes: 0)
    monkeypatch.setattr(runner_module, "prefer_shared_decode",
                        lambda starts, shared, *sizes: any(shared))
    return calls


def make_engine(model, *, num_blocks=96, block_size=16, **limits):
    values = dict(max_num_seqs=8, max_num_batched_tokens=128, max_num_prefill_tokens=64,
                  max_model_len=512, use_cuda_graph=True)
    values.update(limits)
    config = EngineConfig(**values)
    runner = ModelRunner(model, config, num_blocks=num_blocks, block_size=block_size)
    return LLMEngine(Scheduler(config, BlockManager(num_blocks, block_size)), runner)


def count_replays(runner):
    """A list that grows with every replay of the graphs for shared blocks."""
    replay, batches = runner.shared_graphs.run, []

    def counted(seqs, groups=None):
        batches.append(len(seqs))
        return replay(seqs, groups)

    runner.shared_graphs.run = counted
    return batches


def params(n, greedy=True, **values):
    return SampleParameter(max_tokens=n, greedy=greedy, ignore_eos=True, **values)


def prompt(seed, n, config):
    return np.random.default_rng(seed).integers(0, config.vocab_size, n).tolist()


def check(model, seqs, tolerance):
    """Each sequence's tokens and recorded log probabilities against the oracle."""
    weights = weights_f64(model.host_weights())
    for seq in seqs:
        done = seq.completion_token_ids
        rows = forward_logits(weights, model.config, seq.token_ids[:-1], last_rows=len(done))
        top = rows.max(-1, keepdims=True)
        want = rows - top - np.log(np.exp(rows - top).sum(-1, keepdims=True))
        if seq.sampling.greedy:
            deficits = (top[:, 0] - rows[range(len(done)), done]).tolist()
            assert max(deficits) <= tolerance, deficits
        if seq.sampling.logprobs is None:
            assert seq.logprobs == []
            continue
        assert [entry.token_id for entry in seq.logprobs] == done
        for entry, row in zip(seq.logprobs, want):
            assert abs(entry.logprob - row[entry.token_id]) <= tolerance
            assert len(entry.alternatives) == seq.sampling.logprobs
            best = np.sort(row)[::-1]
            for rank, (token, value) in enumerate(entry.alternatives):
                assert abs(value - row[token]) <= tolerance
                assert abs(value - best[rank]) <= tolerance
            values = [value for _, value in entry.alternatives]
            assert values == sorted(values, reverse=True)
            assert len({token for token, _ in entry.alternatives}) == len(values)


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("length", [15, 16, 17, 40])
def test_forks_continue_as_the_oracle(tiny_model, graph, length):
    # Forked with the cached tokens in a partial block, a full one, the first
    # token of the next, and in the middle.
    engine = make_engine(tiny_model, use_cuda_graph=graph, debug_mode=True)
    seq = Sequence(prompt(1, length, TINY), params(10, logprobs=3))
    engine.add_request(seq)
    engine.step()
    forks = engine.fork(seq.seq_id, 2) + engine.fork(
        seq.seq_id, 2, params(10, greedy=False, logprobs=5, temperature=1.5))
    engine.step()
    forks += engine.fork(forks[2].seq_id, 1, params(12, logprobs=0))
    while not engine.is_finished():
        engine.step()
    greedy = [seq, *forks[:2]]
    assert len({tuple(s.completion_token_ids) for s in greedy}) == 1
    check(tiny_model, greedy, 1e-4)
    check_late(tiny_model, forks[2:4], 1, 1e-4)
    check_late(tiny_model, forks[4:], 2, 1e-4)
    assert engine.stats()["used_blocks"] == 0


def check_late(model, seqs, inherited, tolerance):
    """``check`` for what sequences added after the tokens they were forked with."""
    for seq in seqs:
        tail = Sequence(seq.token_ids[:seq.num_prompt_tokens + inherited], seq.sampling)
        for token in seq.completion_token_ids[inherited:]:
            tail.append_token(token)
        tail.logprobs = seq.logprobs[inherited:]
        check(model, [tail], tolerance)


@pytest.mark.parametrize("graph", [True, False])
def test_a_run_of_the_three_together(wide_model, graph, shared_calls):
    # Two prompts (140 and 97 tokens), one forked into four and one into two,
    # beside a third that shares nothing; scored, compacted as requests leave.
    engine = make_engine(wide_model, use_cuda_graph=graph, shared_prefix_decode=True,
                         debug_mode=True)
    captured = len(shared_calls)
    seqs = [Sequence(prompt(s, n, WIDE), params(m, logprobs=t))
            for s, n, m, t in ((2, 140, 24, 2), (3, 97, 20, None), (4, 31, 30, 0))]
    for seq in seqs:
        engine.add_request(seq)
    while any(not s.num_completion_tokens for s in seqs):
        engine.step()
    forks = engine.fork(seqs[0].seq_id, 3, params(40, logprobs=4, greedy=False))
    late, = engine.fork(seqs[1].seq_id, 1, params(33, logprobs=1))
    tokens = [s.num_completion_tokens for s in seqs]  # that the forks began with
    replays = count_replays(engine.model_runner) if graph else None
    moved = steps = 0
    while not engine.is_finished():
        engine.step()
        steps += 1
        if steps % 5 == 0:
            moved += engine.compact()
    calls = len(replays) if graph else (len(shared_calls) - captured) // WIDE.num_hidden_layer
    assert calls >= 25 and moved > 0
    check(wide_model, seqs, 0.1)
    check_late(wide_model, forks, tokens[0], 0.1)
    # Its parent kept no scores, so its own begin with its own tokens.
    late.logprobs = [None] * tokens[1] + late.logprobs
    check_late(wide_model, [late], tokens[1], 0.1)
    assert engine.stats()["used_blocks"] == 0


def test_shared_and_plain_decode_agree(wide_model, shared_calls):
    # Greedy completions with and without the shared reads, each within the
    # oracle's bound, from equal prompts that the prefix cache shares.
    outs = []
    for share in (True, False):
        engine = make_engine(wide_model, shared_prefix_decode=share)
        replays = count_replays(engine.model_runner) if share else []
        first = Sequence(prompt(5, 100, WIDE), params(12, logprobs=1))
        engine.add_request(first)
        while not first.num_completion_tokens:
            engine.step()
        rest = [Sequence(first.token_ids[:100] + prompt(6 + i, 3 + i, WIDE),
                         params(12, logprobs=1)) for i in range(5)]
        for seq in rest:
            engine.add_request(seq)
        while not engine.is_finished():
            engine.step()
        check(wide_model, [first, *rest], 0.1)
        outs.append([first, *rest])
        assert len(replays) >= 8 if share else not replays
    same = sum(a == b for x, y in zip(*outs)
               for a, b in zip(x.completion_token_ids, y.completion_token_ids))
    print(f"{same} of 72 tokens equal")


def test_shapes_without_shared_decode_run_plainly(tiny_model, shared_calls):
    engine = make_engine(tiny_model, shared_prefix_decode=True)
    seq = Sequence(prompt(9, 40, TINY), params(6))
    engine.add_request(seq)
    while not seq.num_completion_tokens:
        engine.step()
    forks = engine.fork(seq.seq_id, 2)
    while not engine.is_finished():
        engine.step()
    assert not shared_calls and engine.model_runner.shared_graphs is None
    check(tiny_model, [seq, *forks], 1e-4)


def test_preempted_forks_keep_their_tokens(tiny_model):
    # Whole prompts at once: a chunk of one could wait behind another's blocks.
    engine = make_engine(tiny_model, num_blocks=9, max_num_batched_tokens=512,
                         max_num_prefill_tokens=512)
    seq = Sequence(prompt(10, 60, TINY), params(30, logprobs=2))
    engine.add_request(seq)
    while not seq.num_completion_tokens:
        engine.step()
    forks = engine.fork(seq.seq_id, 3)
    while not engine.is_finished():
        engine.step()
    assert engine.stats()["num_preemptions"] > 0
    check(tiny_model, [seq, *forks], 1e-4)


def test_scores_of_requests_that_do_not_ask_cost_nothing(tiny_model, monkeypatch):
    def refuse(*args, **kwargs):
        raise AssertionError("not asked for")

    monkeypatch.setattr(runner_module, "token_logprobs", refuse)
    engine = make_engine(tiny_model)
    out = engine.generate([prompt(11, 20, TINY)], params(4))
    assert len(out[0]) == 4


def test_preempted_forks_with_prompts_in_chunks(tiny_model):
    # A preempted fork waits in front of another's prompt, of which a chunk is done.
    engine = make_engine(tiny_model, num_blocks=9, max_num_prefill_tokens=16)
    seq = Sequence(prompt(10, 60, TINY), params(40, logprobs=2))
    engine.add_request(seq)
    while not seq.num_completion_tokens:
        engine.step()
    forks = engine.fork(seq.seq_id, 4)
    while not engine.is_finished():
        engine.step()
    assert engine.stats()["num_preemptions"] > 0
    check(tiny_model, [seq, *forks], 1e-4)


@pytest.mark.parametrize("graph", [True, False])
def test_shared_and_plain_steps_give_the_same_logits(wide_model, shared_calls, graph):
    # The same tokens in both, those of the plain run. Each run's logits are within
    # half the oracle's bound on deficits (0.1) of the oracle's, as `check` shows for
    # the tokens it sees, so their difference is within that bound.
    forced, logits = {}, []
    for share in (False, True):
        engine = make_engine(wide_model, shared_prefix_decode=share, use_cuda_graph=graph)
        runner, seen, index = engine.model_runner, {}, {}
        plain_run, record = runner.run, runner._record_logprobs

        def run(seqs, is_prefill):
            tokens = plain_run(seqs, is_prefill)
            for i, seq in enumerate(seqs):
                if seq.num_cached_tokens + seq.num_scheduled_tokens < len(seq):
                    continue  # a prompt's chunk: its sample is dropped
                key = index[seq.seq_id], len(seq)
                tokens[i] = forced.setdefault(key, tokens[i])
            return tokens

        def recorded(seqs, rows, tokens):
            for seq, row in zip(seqs, rows):
                seen[index[seq.seq_id], len(seq)] = row.float().cpu()
            record(seqs, rows, tokens)

        runner.run, runner._record_logprobs = run, recorded
        calls = len(shared_calls)
        base = prompt(5, 100, WIDE)
        seqs = [Sequence(base, params(14))]
        seqs += [Sequence(base + prompt(6 + i, 3 + 5 * i, WIDE), params(14)) for i in range(5)]
        for i, seq in enumerate(seqs):
            index[seq.seq_id] = i
            engine.add_request(seq)
            while not seq.num_completion_tokens:
                engine.step()
        replays = count_replays(runner) if share and graph else None
        while not engine.is_finished():
            engine.step()
        steps = len(replays) if replays is not None else \
            (len(shared_calls) - calls) // WIDE.num_hidden_layer
        assert steps >= 8 if share else steps == 0
        logits.append(seen)
        outs = [seq.completion_token_ids for seq in seqs]
        if not share:
            check(wide_model, seqs, 0.1)
    plain, shared = logits
    assert plain.keys() == shared.keys() and len(plain) >= 6 * 14
    for key, row in plain.items():
        off = (shared[key] - row).abs().max()
        assert off <= 0.1, f"sequence {key[0]}, {key[1]} tokens: {off}"
    assert outs == [[forced[i, len(s.token_ids) - 14 + k] for k in range(14)]
                    for i, s in enumerate(seqs)]
