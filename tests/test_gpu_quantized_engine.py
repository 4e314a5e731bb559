"""The 8-bit cache as a program uses it: writes, chunks and decode through
``CachedAttention`` and the engine.

``CachedAttention`` is checked against the float64 oracle of the same writes.
The engine's steps are checked against the same model over a float32 cache that
holds what the 8-bit one stands for: both attend over the same values, so their
logits differ by float32 rounding alone, for which the engine's float32 tests
take 1e-4. What an engine does with its blocks (graphs, forks, compaction) must
not change a token.
"""

import numpy as np
import pytest
import torch

from microinfer_amd.engine.blockmanager import BlockManager
from microinfer_amd.engine.config import KV_CACHE_DTYPES, EngineConfig, SampleParameter
from microinfer_amd.engine.llm_engine import LLMEngine
from microinfer_amd.engine.model import QwenConfig, Qwen3Model
from microinfer_amd.engine.model_runner import ModelRunner
from microinfer_amd.engine.scheduler import Scheduler
from microinfer_amd.engine.sequence import Sequence
from microinfer_amd.layer.cached_attention import CachedAttention
from microinfer_amd.layer.metadata import AttentionMetadata
from microinfer_amd.layer.paged_attention import gather_paged_kv, paged_attention_meta
from microinfer_amd.worker.kv_cache import KVCache
from oracle import quantized as oracle
from tests.quantized_support import Twin, check_attention, ints

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


def prompts(seed, lengths, vocab=512):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, vocab, n).tolist() for n in lengths]


def make_engine(model, *, num_blocks=64, block_size=16, **limits):
    values = dict(max_num_seqs=8, max_num_batched_tokens=48, max_num_prefill_tokens=32,
                  max_model_len=256, use_cuda_graph=True, kv_cache_dtype="int8")
    values.update(limits)
    config = EngineConfig(**values)
    runner = ModelRunner(model, config, num_blocks=num_blocks, block_size=block_size)
    return LLMEngine(Scheduler(config, BlockManager(num_blocks, block_size)), runner)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("checked", [True, False])
def test_chunks_and_decode_through_cached_attention(kind, checked):
    gen = torch.Generator().manual_seed(0)
    total, block = 90, 16
    q, k, v = (torch.randn(total, h, 64, generator=gen).to(torch.bfloat16).cuda()
               for h in (4, 2, 2))
    pool = KVCache(2, 9, block, 2, 64, dtype=KV_CACHE_DTYPES[kind], device="cuda")
    backend = CachedAttention()
    backend.bind_cache(pool.layer(1))
    twin = Twin(9, block, 2, 64, kind, device="cpu")
    table = [7, 2, 0, 8, 1, 5]
    slots = [table[p // block] * block + p % block for p in range(total)]
    for start, end in [(0, 20), (20, 21), (21, 75), (75, 88), (88, 89), (89, 90)]:
        decode = start >= 88
        common = dict(slot_mapping=ints(slots[start:end]), validate_cache_write=checked)
        if decode:
            metadata = AttentionMetadata.build(is_prefill=False, context_lens=ints([end]),
                                               block_tables=ints([table]), **common)
        else:
            metadata = AttentionMetadata.build(
                is_prefill=True, cu_seqlens_q=ints([0, end - start]),
                cu_seqlens_k=ints([0, end]), max_seqlen_q=end - start, max_seqlen_k=end,
                block_tables=ints([table]) if start else None, **common)
        got = backend(q[start:end], k[start:end], v[start:end], metadata)
        twin.expect(slots[start:end], k[start:end], v[start:end])
        if start == 0:  # no cached prefix: over the rows as they came
            want = CachedAttention()(q[:end], k[:end], v[:end], metadata)
            assert torch.equal(got, want)
            continue
        check_attention(got, q[start:end], twin, [table], [end], [0, end - start], 64 ** -0.5,
                        (16, 0) if decode else (11, 2.0 ** -35))
    for got, want in zip((pool.keys, pool.values, pool.key_scales, pool.value_scales),
                         (twin.k, twin.v, twin.ks, twin.vs)):
        np.testing.assert_array_equal(got[1].cpu().double().numpy(), want)
        assert not got[0].float().any()
    layer = pool.layer(1)
    rows = gather_paged_kv(layer.keys, layer.values, ints([table]), [total], block,
                           key_scales=layer.key_scales, value_scales=layer.value_scales,
                           dtype=torch.float32)
    for got, codes, scales in zip(rows, (twin.k, twin.v), (twin.ks, twin.vs)):
        want = oracle.gather(codes, scales, [table], [total])
        np.testing.assert_array_equal(got.cpu().double().numpy(), want)


def test_groups_of_sequences_and_missing_scales():
    gen = torch.Generator().manual_seed(1)
    cache = KVCache(1, 8, 16, 2, 128, dtype=torch.float8_e4m3fn, device="cuda").layer(0)
    rows = torch.randn(2, 100, 2, 128, generator=gen).to(torch.bfloat16).cuda()
    cache.write_slots(ints(list(range(100))), *rows)
    query = torch.randn(3, 4, 128, generator=gen).to(torch.bfloat16).cuda()
    tables = ints([[0, 1, 2], [0, 1, 4], [0, 3, 5]])
    scales = dict(key_scales=cache.key_scales, value_scales=cache.value_scales)

    def metadata(**kw):
        return AttentionMetadata(is_prefill=False, context_lens=ints([40, 37, 48]),
                                 block_tables=tables, **kw)

    plain = paged_attention_meta(query, cache.keys, cache.values, metadata(), **scales)
    grouped = metadata(group_starts=ints([0, 2, 3]), shared_blocks=ints([2, 0]))
    assert torch.equal(plain, paged_attention_meta(query, cache.keys, cache.values, grouped,
                                                   **scales))
    with pytest.raises(ValueError, match="scales"):
        paged_attention_meta(query, cache.keys, cache.values, metadata())
    with pytest.raises(ValueError, match="scales"):
        gather_paged_kv(cache.keys, cache.values, tables, [3, 3, 3], 16)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_steps_are_those_of_a_cache_with_the_same_values(tiny_model, kind):
    """Chunks and decode steps of a batch, each run a second time over a float32
    cache that was given what the 8-bit one stands for after the step."""
    model = tiny_model
    engine = make_engine(model, kv_cache_dtype=kind, use_cuda_graph=False)
    runner = engine.model_runner
    plain = KVCache(TINY.num_hidden_layer, 65, 16, 2, 32, dtype=torch.float32, device="cuda")
    codes = runner.kv_cache
    run_model, seen = runner.run_model, []

    def both(input_ids, positions, metadata):
        logits = run_model(input_ids, positions, metadata)
        if metadata.is_prefill and metadata.direct_prefill:
            return logits
        for got, scales, into in ((codes.keys, codes.key_scales, plain.keys),
                                  (codes.values, codes.value_scales, plain.values)):
            into.copy_(got.float() * scales[:, :, None, :, None])
        model.bind_caches([plain.layer(i) for i in range(TINY.num_hidden_layer)])
        slots, metadata.slot_mapping = metadata.slot_mapping, ints([-1] * len(input_ids))
        at_end, metadata.slots_at_end = metadata.slots_at_end, False
        want = run_model(input_ids, positions, metadata)
        metadata.slot_mapping, metadata.slots_at_end = slots, at_end
        model.bind_caches([codes.layer(i) for i in range(TINY.num_hidden_layer)])
        torch.testing.assert_close(logits, want, atol=1e-4, rtol=1e-4)
        seen.append(metadata.is_prefill)
        return logits

    runner.run_model = both
    outputs = engine.generate(prompts(3, [1, 7, 40, 33, 70]),
                              SampleParameter(max_tokens=9, greedy=True))
    assert [len(o) for o in outputs] == [9] * 5
    assert seen.count(True) >= 2 and seen.count(False) >= 8


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_graphs_change_no_token(wide_model, kind):
    batch = prompts(4, [5, 64, 33, 100], WIDE.vocab_size)
    ask = SampleParameter(max_tokens=20, greedy=True, logprobs=3)
    runs = []
    for graph in (True, False):
        engine = make_engine(wide_model, use_cuda_graph=graph, kv_cache_dtype=kind)
        seqs = [Sequence(list(p), ask) for p in batch]
        for seq in seqs:
            engine.add_request(seq)
        while not engine.is_finished():
            engine.step()
        assert all(len(s.logprobs) == 20 for s in seqs)
        runs.append([s.completion_token_ids for s in seqs])
        assert engine.stats()["used_blocks"] == 0
    assert runs[0] == runs[1]


def test_forks_and_compaction_change_no_token(tiny_model):
    """Greedy forks of a request go on as it does, from copied pages with their
    scales; compaction moves pages with theirs. Both runs take their prompts in
    the same chunks: a prompt's first chunk attends over its rows as they came,
    the others over what the cache holds."""
    ask = SampleParameter(max_tokens=24, greedy=True)
    batch = prompts(5, [21, 40, 9])

    def run(disturbed):
        engine = make_engine(tiny_model)
        early = Sequence(prompts(6, [50])[0], SampleParameter(max_tokens=2, greedy=True))
        engine.add_request(early)  # its blocks are free when the others have some
        seqs = [Sequence(list(p), ask) for p in batch]
        for seq in seqs:
            engine.add_request(seq)
        children, moved, steps = [], 0, 0
        while not engine.is_finished():
            engine.step()
            steps += 1
            if disturbed and steps == 9:
                assert len(seqs[1]) % 16 != 0 and len(seqs[1]) < 64
                assert not any(s.num_cached_tokens < len(p) for s, p in zip(seqs, batch))
                children = engine.fork(seqs[1].seq_id, 2)
            if disturbed and steps in (8, 12):
                moved += engine.compact()
        return [s.completion_token_ids for s in seqs], children, moved

    want, _, _ = run(False)
    got, children, moved = run(True)
    assert moved > 0 and len(children) == 2
    assert got == want
    for child in children:
        assert child.completion_token_ids[-5:] == want[1][-5:]


def test_an_8_bit_pool_is_half_of_a_16_bit_one(wide_model):
    pools = {}
    for kind in (None, "fp8"):
        pools[kind] = make_engine(wide_model, use_cuda_graph=False, shared_prefix_decode=True,
                                  kv_cache_dtype=kind).model_runner
    assert pools[None].share and not pools["fp8"].share
    eight, sixteen = (pools[k].kv_cache.num_bytes for k in ("fp8", None))
    assert eight == sixteen // 2 + 2 * 2 * 65 * 8 * 4
