"""Paged attention over an 8-bit KV cache, on the HIP library.

``hip_quantized_decode`` and ``hip_quantized_prefill`` are ``hip_paged_decode``
and ``hip_paged_prefill`` for a cache that holds each value as ``code * scale``
(``hip_quantized_kv``): the query keeps its own type, codes are widened as they
are read, the scales of each block of tokens and KV head meet the scores (K)
and the softmax weights (V) in float32.
"""

from __future__ import annotations

import ctypes
import threading
from dataclasses import dataclass, field

import torch

from microinfer_amd import _lib
from microinfer_amd.worker.hip_quantized_kv import (check_quantized_cache, index32,
                                                    whole_vectors)

MAX_SEQS = 4096
_FLOAT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _call_place(stream: int) -> tuple:
    """What calls that run one after the other have in common: thread, stream (the
    current one) and the capture that they are in, if any."""
    capture = 0
    if torch.cuda.is_current_stream_capturing():
        number = ctypes.c_uint64()
        _lib.check(_lib.load().mi_stream_capture_id(stream, ctypes.addressof(number)),
                   "mi_stream_capture_id")
        capture = number.value
    return threading.get_ident(), stream, capture


@dataclass(frozen=True)
class QuantizedDecodePlan:
    """One step's work (``quantized_decode_plan``), for calls of its sizes."""

    buffer: torch.Tensor  # the plan, and a workspace for where it was made
    sizes: tuple  # sequences, Hq, Hkv, head_dim, dtype, block size, table width
    bytes: int
    workspace_bytes: int
    _workspaces: dict = field(repr=False, compare=False)  # place -> addresses, memory

    def workspace(self, stream: int) -> tuple:
        """Addresses of the partials and counters of a call from here (then what
        keeps them): its thread's and stream's own, a call's own where a graph
        holds it but not the plan."""
        place = _call_place(stream)
        have = self._workspaces.get(place)
        if have is None:
            device = self.buffer.device
            partials = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=device)
            counters = torch.zeros(self.sizes[0] * self.sizes[2], dtype=torch.int32,
                                   device=device)
            have = partials.data_ptr(), counters.data_ptr(), partials, counters
            if not place[2]:
                self._workspaces[place] = have
        return have


def quantized_decode_plan(context_lens: torch.Tensor, *, num_q_heads: int, num_kv_heads: int,
                          head_dim: int, dtype: torch.dtype, block_size: int,
                          block_table_width: int) -> QuantizedDecodePlan:
    """The plan of one decode step over an 8-bit cache (shared by its layers),
    from the lengths on the device alone (capture-safe). ``dtype``: the
    query's."""
    _lib.require_device(context_lens, what="quantized_decode_plan")
    if num_kv_heads <= 0 or num_q_heads <= 0 or num_q_heads % num_kv_heads:
        raise ValueError("Hq must be divisible by Hkv")
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("unsupported query dtype")
    if block_size <= 0 or block_size & (block_size - 1):
        raise ValueError("paged kernels require a power-of-two block size")
    if context_lens.ndim != 1:
        raise ValueError("context_lens must be 1-D")
    num_seqs, device = context_lens.numel(), context_lens.device
    if num_seqs > MAX_SEQS:
        raise ValueError(f"at most {MAX_SEQS} sequences")
    context_lens = index32(context_lens)
    lib = _lib.load()
    with _lib.on_device(device):
        nbytes = lib.mi_quant_decode_plan_bytes(num_seqs, num_kv_heads)
        partial_bytes = lib.mi_quant_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads,
                                                            head_dim)
        # One allocation: plan, partials, counters.
        partials = -(-nbytes // 256) * 256
        counters = partials + -(-partial_bytes // 256) * 256
        buffer = torch.empty(counters + 4 * num_seqs * num_kv_heads, dtype=torch.uint8,
                             device=device)
        at, stream = buffer.data_ptr(), _lib.stream_handle(device)
        status = lib.mi_quant_decode_plan(
            context_lens.data_ptr(), num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
            block_table_width, _lib.DTYPE_CODES[dtype], at, nbytes, at + counters, stream)
        _lib.check(status, "mi_quant_decode_plan")
        place = _call_place(stream)
    return QuantizedDecodePlan(
        buffer, (num_seqs, num_q_heads, num_kv_heads, head_dim, dtype, block_size,
                 block_table_width), nbytes, partial_bytes,
        {place: (at + partials, at + counters)})


def _check_query(query: torch.Tensor, key_cache: torch.Tensor, device: int, rows: str):
    """ValueError unless the query fits the cache; its shape and the cache's."""
    shape, cache = query.shape, key_cache.shape
    if len(shape) != 3:
        raise ValueError(f"query must have shape [{rows}, Hq, D]")
    if query.dtype not in _FLOAT_DTYPES:
        raise ValueError("unsupported query dtype")
    if query.get_device() != device:
        raise ValueError("query and cache must share a device")
    if cache[3] != shape[2]:
        raise ValueError("query and cache head dimensions differ")
    if shape[1] == 0 or shape[1] % cache[2]:
        raise ValueError("Hq must be divisible by Hkv")
    return shape, cache


def hip_quantized_decode(query: torch.Tensor, key_cache: torch.Tensor,
                         value_cache: torch.Tensor, key_scales: torch.Tensor,
                         value_scales: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, *, scale: float | None = None,
                         plan: QuantizedDecodePlan | None = None) -> torch.Tensor:
    """Decode one query row per request over an 8-bit paged cache.

    ``query [R, Hq, D]`` (float16, bfloat16 or float32), caches
    ``[N, B, Hkv, D]``, scales ``[N, Hkv]``, ``block_tables [R, W]`` and
    ``context_lens [R]`` on the device. Returns ``[R, Hq, D]`` in the query's
    dtype. The caches hold the step's rows already. ``plan``: of
    ``quantized_decode_plan`` for these lengths; without it the call makes its
    own. Sequences of length 0 give zeros, block ids outside the pool are
    masked.
    """
    cache, code, device = check_quantized_cache(key_cache, value_cache, key_scales,
                                                value_scales, "hip_quantized_decode")
    ((num_seqs, num_q_heads, head_dim),
     (num_blocks, block_size, num_kv_heads, _)) = _check_query(query, key_cache, device,
                                                               "requests")
    if device != _lib.raw_device():
        with torch.cuda.device(device):
            return hip_quantized_decode(query, key_cache, value_cache, key_scales, value_scales,
                                        block_tables, context_lens, scale=scale, plan=plan)
    if block_tables.ndim != 2 or block_tables.shape[0] != num_seqs:
        raise ValueError("block_tables must have one row per request")
    if context_lens.numel() != num_seqs:
        raise ValueError("context_lens must have one entry per request")
    if block_tables.get_device() != device or context_lens.get_device() != device:
        _lib.require_device(block_tables, context_lens, what="hip_quantized_decode")
        raise ValueError("block_tables and context_lens must be on the query's device")
    width, dtype = block_tables.shape[1], query.dtype
    if plan is None:
        plan = quantized_decode_plan(
            context_lens.reshape(-1), num_q_heads=num_q_heads, num_kv_heads=num_kv_heads,
            head_dim=head_dim, dtype=dtype, block_size=block_size, block_table_width=width)
    elif not isinstance(plan, QuantizedDecodePlan) or plan.sizes != (
            num_seqs, num_q_heads, num_kv_heads, head_dim, dtype, block_size, width):
        raise ValueError("plan must come from quantized_decode_plan() for this call's sizes")
    elif plan.buffer.get_device() != device:
        raise ValueError("plan must be on the query's device")
    query, tables = whole_vectors(query), index32(block_tables)
    out = query.new_empty((num_seqs, num_q_heads, head_dim))
    if num_seqs == 0:
        return out
    strides, stream = query.stride(), _lib.raw_stream(device)
    workspace = plan.workspace(stream)
    status = _lib.load().mi_quant_decode(
        query.data_ptr(), strides[0], strides[1], *cache, tables.data_ptr(), width, width,
        plan.buffer.data_ptr(), plan.bytes, out.data_ptr(), num_q_heads * head_dim, head_dim,
        workspace[0], plan.workspace_bytes, workspace[1], num_seqs, num_q_heads, num_kv_heads,
        head_dim, block_size, num_blocks, head_dim ** -0.5 if scale is None else float(scale),
        _lib.DTYPE_CODES[dtype], code, stream)
    if status:
        _lib.check(status, "mi_quant_decode")
    return out


@dataclass(frozen=True)
class QuantizedPrefillPlan:
    """One step's work (``quantized_prefill_plan``), for calls of its sizes."""

    cu_seqlens_q: torch.Tensor
    cu_seqlens_k: torch.Tensor
    sizes: tuple  # tokens, requests, Hq, Hkv, head_dim, block size, table width
    max_seqlen_q: int
    workspace_bytes: int
    _workspaces: dict = field(default_factory=dict, repr=False, compare=False)

    def workspace(self, stream: int) -> torch.Tensor:
        """The plan with room for the partials of a call from here: its
        thread's and stream's own, a call's own where a graph holds it but not
        the plan."""
        place = _call_place(stream)
        have = self._workspaces.get(place)
        if have is None:
            have = torch.empty(self.workspace_bytes, dtype=torch.uint8,
                               device=self.cu_seqlens_q.device)
            tokens, requests, *sizes = self.sizes
            status = _lib.load().mi_quant_prefill_plan(
                self.cu_seqlens_q.data_ptr(), self.cu_seqlens_k.data_ptr(), tokens, requests,
                self.max_seqlen_q, *sizes, have.data_ptr(), self.workspace_bytes, place[1])
            _lib.check(status, "mi_quant_prefill_plan")
            # A graph keeps what is made in its capture: only the plan's own does
            # for further calls.
            if not place[2] or not self._workspaces:
                self._workspaces[place] = have
        return have


def quantized_prefill_plan(cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, *,
                           num_tokens: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                           dtype: torch.dtype, block_size: int, block_table_width: int,
                           max_seqlen_q: int | None = None) -> QuantizedPrefillPlan | None:
    """The plan of one step's ``hip_quantized_prefill`` calls (shared by its
    layers), from the cu_seqlens on the device (capture-safe). None: calls of
    these sizes run without one, row by row and many times slower (head sizes other
    than 64 and 128, blocks of less than 16, the largest groups and steps:
    ``mi_quant.h`` has the limits). ``max_seqlen_q`` bounds the new tokens of any
    request (``num_tokens`` by default): where it is small, the step is laid out
    for few rows a request. Plans of longer requests hold 38 MB (heads of 64) or
    71 MB (128) of partials."""
    _lib.require_device(cu_seqlens_q, cu_seqlens_k, what="quantized_prefill_plan")
    if num_kv_heads <= 0 or num_q_heads <= 0 or num_q_heads % num_kv_heads:
        raise ValueError("Hq must be divisible by Hkv")
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("unsupported query dtype")
    requests, device = cu_seqlens_q.numel() - 1, cu_seqlens_q.device
    if requests < 0 or cu_seqlens_k.numel() != requests + 1:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have num_requests + 1 entries")
    if cu_seqlens_k.device != device:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must share a device")
    longest = num_tokens if max_seqlen_q is None else min(max_seqlen_q, num_tokens)
    if longest <= 0 and num_tokens:
        raise ValueError("max_seqlen_q must be positive")
    sizes = num_q_heads, num_kv_heads, head_dim, block_size
    nbytes = _lib.load().mi_quant_prefill_workspace_bytes(num_tokens, requests, longest, *sizes)
    if nbytes == 0:
        return None
    plan = QuantizedPrefillPlan(index32(cu_seqlens_q), index32(cu_seqlens_k),
                                (num_tokens, requests, *sizes, block_table_width), longest,
                                nbytes)
    with _lib.on_device(device):
        plan.workspace(_lib.stream_handle(device))
    return plan


def hip_quantized_prefill(query: torch.Tensor, key_cache: torch.Tensor,
                          value_cache: torch.Tensor, key_scales: torch.Tensor,
                          value_scales: torch.Tensor, cu_seqlens_q: torch.Tensor,
                          cu_seqlens_k: torch.Tensor, block_tables: torch.Tensor, *,
                          max_seqlen_q: int, scale: float | None = None,
                          plan: QuantizedPrefillPlan | None = None) -> torch.Tensor:
    """Causal varlen attention over an 8-bit paged cache (bottom-right mask).

    ``query [T, Hq, D]``; request r owns query rows ``cu_seqlens_q[r]..`` and
    context ``cu_seqlens_k[r+1] - cu_seqlens_k[r]`` (it includes the new rows,
    which the caller appended first). ``max_seqlen_q`` bounds the query rows of
    any request. ``plan``: of ``quantized_prefill_plan`` for these lengths and
    sizes; without it the call makes its own. Rows that see nothing give zeros;
    rows of no request (behind the last one) are not computed: theirs is
    uninitialised memory.
    """
    cache, code, device = check_quantized_cache(key_cache, value_cache, key_scales,
                                                value_scales, "hip_quantized_prefill")
    ((num_tokens, num_q_heads, head_dim),
     (num_blocks, block_size, num_kv_heads, _)) = _check_query(query, key_cache, device, "tokens")
    if device != _lib.raw_device():
        with torch.cuda.device(device):
            return hip_quantized_prefill(query, key_cache, value_cache, key_scales, value_scales,
                                         cu_seqlens_q, cu_seqlens_k, block_tables,
                                         max_seqlen_q=max_seqlen_q, scale=scale, plan=plan)
    if block_tables.ndim != 2:
        raise ValueError("block_tables must have one row per request")
    num_requests, width = block_tables.shape
    for name, offsets in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        if offsets.numel() != num_requests + 1:
            raise ValueError(f"{name} must have num_requests + 1 entries")
    if max_seqlen_q <= 0 and num_tokens:
        raise ValueError("max_seqlen_q must be positive")
    if any(t.get_device() != device for t in (cu_seqlens_q, cu_seqlens_k, block_tables)):
        _lib.require_device(cu_seqlens_q, cu_seqlens_k, block_tables,
                            what="hip_quantized_prefill")
        raise ValueError("cu_seqlens and block_tables must be on the query's device")
    sizes = num_tokens, num_requests, num_q_heads, num_kv_heads, head_dim, block_size, width
    longest = min(max_seqlen_q, num_tokens)
    if plan is not None and (not isinstance(plan, QuantizedPrefillPlan) or plan.sizes != sizes
                             or plan.max_seqlen_q < longest):
        raise ValueError("plan must come from quantized_prefill_plan() for this call's sizes")
    if plan is not None and plan.cu_seqlens_q.get_device() != device:
        raise ValueError("plan must be on the query's device")
    if num_tokens and not num_requests:
        raise ValueError("tokens without requests")
    query, tables = whole_vectors(query), index32(block_tables)
    cu_q, cu_k = index32(cu_seqlens_q), index32(cu_seqlens_k)
    out = query.new_empty((num_tokens, num_q_heads, head_dim))
    if num_tokens == 0:
        return out
    if plan is None:
        plan = quantized_prefill_plan(
            cu_q, cu_k, num_tokens=num_tokens, num_q_heads=num_q_heads,
            num_kv_heads=num_kv_heads, head_dim=head_dim, dtype=query.dtype,
            block_size=block_size, block_table_width=width, max_seqlen_q=max_seqlen_q)
    strides, stream = query.stride(), _lib.raw_stream(device)
    workspace, nbytes = None, 0
    if plan is not None:
        workspace, nbytes = plan.workspace(stream), plan.workspace_bytes
        longest = plan.max_seqlen_q
    status = _lib.load().mi_quant_prefill(
        query.data_ptr(), strides[0], strides[1], *cache, cu_q.data_ptr(), cu_k.data_ptr(),
        tables.data_ptr(), width, width, out.data_ptr(), num_q_heads * head_dim, head_dim,
        None if workspace is None else workspace.data_ptr(), nbytes, num_tokens, num_requests,
        longest, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks,
        head_dim ** -0.5 if scale is None else float(scale), _lib.DTYPE_CODES[query.dtype], code,
        stream)
    if status:
        _lib.check(status, "mi_quant_prefill")
    return out
