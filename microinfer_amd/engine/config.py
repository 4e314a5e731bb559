"""Engine limits and per-request sampling values.

Mirrors ``SampleParameter`` (microinfer/config/samplepara.py:5-17) and the
fields of ``EngineConfig`` (microinfer/config/engine.py:6-68) that this
engine acts on, with the same validation errors. The reference's switches
for torch.compile and n-gram speculative decoding have no counterpart here:
decode runs from hipGraphs of the HIP kernels, and speculation is not part
of the attention path. ``SampleParameter.logprobs``,
``EngineConfig.shared_prefix_decode`` and ``EngineConfig.kv_cache_dtype`` have no
counterpart in the reference.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

# What EngineConfig.kv_cache_dtype may be (None: the model's type).
KV_CACHE_DTYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
MAX_LOGPROBS = 32  # alternatives that mi_token_logprobs gives


@dataclass(slots=True)
class SampleParameter:
    temperature: float = 1.0
    max_tokens: int = 64
    ignore_eos: bool = False
    greedy: bool = False
    # Record each sampled token's log probability with this many alternatives
    # (0: the token alone; None: nothing), of the model's own distribution.
    logprobs: int | None = None

    def __post_init__(self):
        # A temperature near zero is rejected: greedy decoding is asked for
        # with ``greedy=True`` instead (samplepara.py:12-14).
        assert math.isfinite(self.temperature) and self.temperature > 1e-10, (
            "greedy sampling is not permitted"
        )
        if type(self.max_tokens) is not int or self.max_tokens <= 0:
            raise ValueError("max_tokens must be a positive integer")
        if self.logprobs is not None and (
                type(self.logprobs) is not int or not 0 <= self.logprobs <= MAX_LOGPROBS):
            raise ValueError(f"logprobs must be None or an integer between 0 and {MAX_LOGPROBS}")


@dataclass(frozen=True)
class EngineConfig:
    max_num_seqs: int = 16
    max_num_batched_tokens: int = 512
    max_num_prefill_tokens: int = 512  # cap of one prefill chunk
    max_model_len: int = 4096
    eos_token_id: int | None = None
    debug_mode: bool = False
    use_cuda_graph: bool = False  # decode buckets replayed from hipGraphs
    mixed_batch: bool = True  # fill the budget with prefill after running decode
    # Decode batches whose sequences share enough cache blocks (forks, common
    # prompts) read them together; captures a second graph per bucket.
    shared_prefix_decode: bool = False
    # "fp8" or "int8": the K/V cache in 8 bits, half of a 16-bit one's memory,
    # with a scale for each block and KV head. Decode steps get faster; chunks of
    # prompts behind cached tokens may get slower (half precision, uneven lengths:
    # by a quarter). Sequences read shared blocks each for itself:
    # ``shared_prefix_decode`` has no effect.
    kv_cache_dtype: str | None = None

    def __post_init__(self):
        for name in ("max_num_seqs", "max_num_batched_tokens", "max_num_prefill_tokens",
                     "max_model_len"):
            value = getattr(self, name)
            if type(value) is not int or value <= 0:
                raise ValueError(f"{name} must be a positive integer")
        if self.eos_token_id is not None and (
                type(self.eos_token_id) is not int or self.eos_token_id < 0):
            raise ValueError("eos_token_id must be a nonnegative integer or None")
        for name in ("debug_mode", "use_cuda_graph", "mixed_batch", "shared_prefix_decode"):
            if type(getattr(self, name)) is not bool:
                raise ValueError(f"{name} must be a boolean")
        if self.kv_cache_dtype is not None and self.kv_cache_dtype not in KV_CACHE_DTYPES:
            raise ValueError(f"kv_cache_dtype must be None or one of {tuple(KV_CACHE_DTYPES)}")
