"""Runs one scheduled step of the model and returns the sampled tokens.

Mirrors ``ModelRunner.run`` / ``run_model`` / ``_run_decode``
(microinfer/runner.py:555-626): prefill steps build their metadata on the
device and run eagerly; decode steps replay the smallest captured hipGraph
bucket that holds the batch (greedy tokens selected inside the graph) or run
eagerly when no bucket fits or graphs are off; greedy rows take the argmax,
the others the temperature sampler, mixed per row as the reference does.

The KV pool has one block more than the block manager hands out: the pad
rows of graph buckets write their K/V there. With ``EngineConfig.debug_mode``
each step's metadata is validated before launch (``runner.validate_step``).

With ``EngineConfig.shared_prefix_decode`` a decode batch whose sequences
share enough blocks (forks of a request, common prompts) reads them together
(``hip_shared_decode``), from a second set of graphs; sequences that ask for
``logprobs`` get those of each token they keep (``token_logprobs`` of the
step's logits).
"""

from __future__ import annotations

import torch

from microinfer_amd.engine.config import EngineConfig
from microinfer_amd.engine.sequence import TokenLogprob
from microinfer_amd.layer.hip_logprobs import token_logprobs
from microinfer_amd.layer.hip_sampler import Sampler, greedy_argmax
from microinfer_amd.layer.hip_shared_decode import (least_shared_positions,
                                                    prefer_shared_decode, shared_groups,
                                                    shared_order, supported_shared_decode)
from microinfer_amd.runner import DecodeGraphRunner, StepMetadataBuilder
from microinfer_amd.worker.kv_cache import KVCache


class ModelRunner:
    def __init__(self, model, config: EngineConfig, *, num_blocks: int, block_size: int,
                 layout: str = "paired"):
        c = model.config
        self.model, self.config = model, config
        self.num_blocks, self.block_size = num_blocks, block_size
        self.kv_cache = KVCache(c.num_hidden_layer, num_blocks + 1, block_size, c.num_kv_head,
                                c.head_dim, dtype=model.dtype, device=model.device,
                                layout=layout)
        model.bind_caches([self.kv_cache.layer(i) for i in range(c.num_hidden_layer)])
        self.builder = StepMetadataBuilder(block_size, model.device, pad_block_id=num_blocks,
                                           debug_mode=config.debug_mode, num_blocks=num_blocks,
                                           max_pos_embed=c.max_pos_embed,
                                           vocab_size=c.vocab_size)
        self.sampler = Sampler()
        self.share = config.shared_prefix_decode and supported_shared_decode(
            c.num_q_head, c.num_kv_head, c.head_dim, model.dtype, block_size,
            config.max_num_seqs)
        self.graphs = self.shared_graphs = None
        if config.use_cuda_graph:
            buckets = dict(max_num_seqs=config.max_num_seqs, table_width=num_blocks + 1,
                           greedy=True)
            self.graphs = DecodeGraphRunner(self.builder, self.run_model, **buckets)
            if self.share:
                self.shared_graphs = DecodeGraphRunner(self.builder, self.run_model, shared=True,
                                                       **buckets)
        self._logprobs: dict[int, TokenLogprob] = {}

    def run_model(self, input_ids, positions, metadata):
        return self.model.compute_logits(self.model.forward(input_ids, positions, metadata),
                                         metadata)

    def copy_blocks(self, src, dst, tokens=None) -> None:
        """Copy cache blocks in every layer (forks, compaction)."""
        self.kv_cache.copy_blocks(src, dst, tokens)

    def take_logprobs(self) -> dict[int, TokenLogprob]:
        """The log probabilities of the tokens sampled since the last call, by
        sequence id, for the sequences that ask for them."""
        taken, self._logprobs = self._logprobs, {}
        return taken

    def _shared_groups(self, seqs):
        """The decode batch ordered so that sequences with a common beginning
        are neighbours, and its groups; None where they are not worth it."""
        contexts = [len(s) for s in seqs]
        heads = self.kv_cache.num_kv_heads, self.model.config.num_q_head
        if sum(contexts) < least_shared_positions(len(seqs), *heads):
            return seqs, None
        tables = [s.block_table for s in seqs]
        order = shared_order(tables)
        starts, shared = shared_groups([tables[i] for i in order], [contexts[i] for i in order],
                                       self.block_size)
        if not prefer_shared_decode(starts, shared, self.block_size, *heads):
            return seqs, None
        return [seqs[i] for i in order], (starts, shared)

    @torch.inference_mode()
    def run(self, seqs, is_prefill: bool) -> list[int]:
        if not seqs:
            return []
        greedy_tokens = None
        asked = seqs
        if is_prefill:
            logits = self.run_model(*self.builder.prepare_prefill(seqs))
        else:
            groups = None
            if self.share and len(seqs) > 1:
                seqs, groups = self._shared_groups(seqs)
            replayed = None
            if groups is not None and self.shared_graphs is not None:
                replayed = self.shared_graphs.run(seqs, groups)
            elif self.graphs is not None:
                replayed = self.graphs.run(seqs)
            if replayed is not None:
                logits, greedy_tokens = replayed
            else:
                logits = self.run_model(*self.builder.prepare_decode(seqs, groups))
        flags = [seq.greedy for seq in seqs]
        if all(flags):
            tokens = greedy_tokens if greedy_tokens is not None else greedy_argmax(logits)
        else:
            temperatures = torch.tensor([seq.temperature for seq in seqs],
                                        dtype=torch.float32, device=logits.device)
            tokens = self.sampler(logits, temperatures)
            if any(flags):
                greedy = greedy_tokens if greedy_tokens is not None else greedy_argmax(logits)
                mask = torch.tensor(flags, dtype=torch.bool, device=logits.device)
                tokens = torch.where(mask, greedy, tokens)
        self._record_logprobs(seqs, logits, tokens)
        sampled = tokens.tolist()
        if seqs is asked:
            return sampled
        by_id = dict(zip((seq.seq_id for seq in seqs), sampled))
        return [by_id[seq.seq_id] for seq in asked]

    def _record_logprobs(self, seqs, logits, tokens) -> None:
        wanted = [seq.sampling.logprobs for seq in seqs]
        if all(n is None for n in wanted):
            return
        top = min(max(n for n in wanted if n is not None), logits.shape[1])
        got = token_logprobs(logits, tokens, top=top)
        sampled, logprobs = tokens.tolist(), got.logprobs.tolist()
        best = [()] * len(seqs)
        if top:
            best = [tuple(zip(ids, values)) for ids, values in
                    zip(got.top_tokens.tolist(), got.top_logprobs.tolist())]
        for seq, n, token, logprob, alternatives in zip(seqs, wanted, sampled, logprobs, best):
            if n is not None:
                self._logprobs[seq.seq_id] = TokenLogprob(token, logprob, alternatives[:n])
