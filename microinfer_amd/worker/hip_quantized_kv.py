"""Writes into and reads out of an 8-bit KV cache through the HIP library.

A pool of ``torch.float8_e4m3fn`` or ``torch.int8`` holds each value as
``code * scale`` with one float32 scale for each block of tokens and KV head, K
and V apart (``KVCache(dtype=...)`` makes one). ``quantized_append`` is
``append_slots`` for such a pool, ``quantized_gather`` is ``hip_gather_kv``:
rows go in and come out as float32, float16 or bfloat16.

A block's scale is the least power of two that brings its rows into the type's
range. A row at offset 0 begins its block anew; rows at later offsets leave the
scale or raise it, and then the rows before them are rounded again (in e4m3
without loss, until they leave its normal range). So the rows of a block are
written in the order of their offsets, as an engine does. What is not finite is
held as NaN; int8 has none, there the block's scale becomes NaN.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from microinfer_amd import _lib

QUANTIZED_DTYPES = (torch.float8_e4m3fn, torch.int8)
# Calls of so many rows find a block's rows in the slot list themselves; larger
# ones have them from a plan.
MAX_SCANNED_TOKENS = 256

_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}
_FLOAT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_INDEX_DTYPES = (torch.int32, torch.int64)


def check_quantized_cache(key_cache, value_cache, key_scales, value_scales, what: str):
    """ValueError / RuntimeError unless the four are an 8-bit cache on the GPU;
    the arguments that describe it to the library, its code and its device's
    index. One look at each property: this is most of a small call's time."""
    shape, strides, dtype = key_cache.shape, key_cache.stride(), key_cache.dtype
    scale_strides, device = key_scales.stride(), key_cache.get_device()
    keys, values = key_cache.data_ptr(), value_cache.data_ptr()
    if (len(shape) != 4 or dtype not in _CODES or value_cache.shape != shape
            or value_cache.dtype != dtype or value_cache.stride() != strides
            or strides[3] != 1 or key_scales.shape != (shape[0], shape[2])
            or value_scales.shape != key_scales.shape or key_scales.dtype != torch.float32
            or value_scales.dtype != torch.float32 or value_scales.stride() != scale_strides
            or device < 0 or value_cache.get_device() != device
            or key_scales.get_device() != device or value_scales.get_device() != device
            or shape[1] & (shape[1] - 1) or not shape[1]
            or shape[3] & (shape[3] - 1) or not 16 <= shape[3] <= 256
            or (keys | values | strides[0] | strides[1] | strides[2]) & 7):
        _refuse(key_cache, value_cache, key_scales, value_scales, what)
    return (keys, values, strides[0], strides[1], strides[2], key_scales.data_ptr(),
            value_scales.data_ptr(), *scale_strides), _CODES[dtype], device


def _refuse(key_cache, value_cache, key_scales, value_scales, what: str):
    """Raises what ``check_quantized_cache`` found."""
    _lib.require_device(key_cache, value_cache, key_scales, value_scales, what=what)
    if key_cache.ndim != 4 or value_cache.shape != key_cache.shape:
        raise ValueError("key/value caches must have matching [blocks, B, Hkv, D] shapes")
    if key_cache.dtype not in _CODES or value_cache.dtype != key_cache.dtype:
        raise ValueError("8-bit caches are float8_e4m3fn or int8, K and V alike")
    num_blocks, block_size, num_kv_heads, head_dim = key_cache.shape
    for scales in (key_scales, value_scales):
        if scales.shape != (num_blocks, num_kv_heads) or scales.dtype != torch.float32:
            raise ValueError("scales must be float32 [blocks, Hkv]")
    if key_cache.stride() != value_cache.stride() or key_scales.stride() != value_scales.stride():
        raise ValueError("K/V caches must share one layout")
    if key_cache.stride(-1) != 1:
        raise ValueError("cache head_dim must be contiguous")
    if any(t.device != key_cache.device for t in (value_cache, key_scales, value_scales)):
        raise ValueError("caches and scales must share a device")
    if block_size <= 0 or block_size & (block_size - 1):
        raise ValueError("paged kernels require a power-of-two block size")
    if head_dim & (head_dim - 1) or not 16 <= head_dim <= 256:
        raise ValueError("8-bit caches need a power-of-two head_dim from 16 to 256")
    raise ValueError("8-bit cache rows must be 8-byte aligned")


def index32(tensor: torch.Tensor) -> torch.Tensor:
    """An index tensor as the kernels read it."""
    if tensor.dtype != torch.int32:
        tensor = tensor.to(torch.int32)
    return tensor if tensor.is_contiguous() else tensor.contiguous()


def whole_vectors(rows: torch.Tensor) -> torch.Tensor:
    """``rows [T, H, D]``, or a copy, with 16-byte aligned head rows."""
    size = rows.element_size()
    token_stride, head_stride, inner = rows.stride()
    if inner != 1 or (rows.data_ptr() | size * token_stride | size * head_stride) & 15:
        return rows.clone(memory_format=torch.contiguous_format)
    return rows


def _slots(slot_mapping: torch.Tensor) -> torch.Tensor:
    if slot_mapping.ndim != 1 or slot_mapping.dtype not in _INDEX_DTYPES:
        raise ValueError("slots must be a 1-D integer tensor")
    return slot_mapping if slot_mapping.is_contiguous() else slot_mapping.contiguous()


@dataclass(frozen=True)
class QuantizedAppendPlan:
    """Where a step's rows go (``quantized_append_plan``), for every layer."""

    buffer: torch.Tensor | None  # None: few rows, which need no plan
    sizes: tuple  # tokens, block size, blocks
    bytes: int


def quantized_append_plan(slot_mapping: torch.Tensor, *, block_size: int,
                          num_blocks: int) -> QuantizedAppendPlan:
    """The plan of ``quantized_append`` calls with these slots, made on the
    device (capture-safe). It holds 4 bytes for each position of the pool."""
    slots = _slots(slot_mapping)
    if not slots.is_cuda:
        _lib.require_device(slots, what="quantized_append_plan")
    if block_size <= 0 or block_size & (block_size - 1):
        raise ValueError("paged kernels require a power-of-two block size")
    if num_blocks <= 0:
        raise ValueError("num_blocks must be positive")
    sizes = slots.numel(), block_size, num_blocks
    if sizes[0] <= MAX_SCANNED_TOKENS:
        return QuantizedAppendPlan(None, sizes, 0)
    lib, device = _lib.load(), slots.device
    nbytes = lib.mi_quant_append_plan_bytes(*sizes)
    buffer = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with _lib.on_device(device):
        status = lib.mi_quant_append_plan(slots.data_ptr(), slots.dtype == torch.int64, *sizes,
                                          buffer.data_ptr(), nbytes, _lib.stream_handle(device))
    _lib.check(status, "mi_quant_append_plan")
    return QuantizedAppendPlan(buffer, sizes, nbytes)


def quantized_append(key_cache: torch.Tensor, value_cache: torch.Tensor,
                     key_scales: torch.Tensor, value_scales: torch.Tensor,
                     slot_mapping: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, *,
                     plan: QuantizedAppendPlan | None = None) -> None:
    """Quantise ``keys``/``values [T, Hkv, D]`` into the cache at
    ``slot_mapping [T]`` (int32/int64; negative or too large ones are skipped).

    Caches ``[N, B, Hkv, D]``, scales ``[N, Hkv]``, all written in place. In a
    block, rows below the lowest offset written stay (rounded again where the
    scale rises); the others stand for something only once they are written.
    Of rows with equal slots one is written, whichever. ``plan``: of
    ``quantized_append_plan`` for these slots; without it a call of many rows
    makes its own.
    """
    cache, code, device = check_quantized_cache(key_cache, value_cache, key_scales,
                                                value_scales, "quantized_append")
    num_blocks, block_size, num_kv_heads, head_dim = key_cache.shape
    shape, dtype = keys.shape, keys.dtype
    if len(shape) != 3 or values.shape != shape:
        raise ValueError("K/V must have matching [tokens, Hkv, D] shapes")
    tokens = shape[0]
    if shape[1] != num_kv_heads or shape[2] != head_dim:
        raise ValueError("K/V heads must match the cache")
    if dtype not in _FLOAT_DTYPES or values.dtype != dtype:
        raise ValueError("K/V must be float16, bfloat16 or float32, both alike")
    slots = _slots(slot_mapping)
    if slots.numel() != tokens:
        raise ValueError("one slot per token is required")
    if (slots.get_device() != device or keys.get_device() != device
            or values.get_device() != device):
        _lib.require_device(slots, keys, values, what="quantized_append")
        raise ValueError("slots and K/V must be on the cache device")
    if block_size > 1024:
        raise ValueError("8-bit caches are written in blocks of at most 1024 tokens")
    if tokens == 0:
        return
    if device != _lib.raw_device():
        with torch.cuda.device(device):
            return quantized_append(key_cache, value_cache, key_scales, value_scales, slots,
                                    keys, values, plan=plan)
    if plan is None:
        plan = quantized_append_plan(slots, block_size=block_size, num_blocks=num_blocks)
    elif not isinstance(plan, QuantizedAppendPlan) or plan.sizes != (tokens, block_size,
                                                                     num_blocks):
        raise ValueError("plan must come from quantized_append_plan() for this call's sizes")
    elif plan.buffer is not None and plan.buffer.get_device() != device:
        raise ValueError("plan must be on the cache device")
    keys, values = whole_vectors(keys), whole_vectors(values)
    k_strides, v_strides = keys.stride(), values.stride()
    status = _lib.load().mi_quant_append(
        keys.data_ptr(), k_strides[0], k_strides[1], values.data_ptr(), v_strides[0],
        v_strides[1], *cache, slots.data_ptr(), slots.dtype == torch.int64,
        None if plan.buffer is None else plan.buffer.data_ptr(), plan.bytes, tokens,
        num_kv_heads, head_dim, block_size, num_blocks, _lib.DTYPE_CODES[dtype], code,
        _lib.raw_stream(device))
    if status:
        _lib.check(status, "mi_quant_append")


def quantized_gather(key_cache: torch.Tensor, value_cache: torch.Tensor,
                     key_scales: torch.Tensor, value_scales: torch.Tensor,
                     block_tables: torch.Tensor, cu_seqlens_k: torch.Tensor, total_rows: int, *,
                     dtype: torch.dtype = torch.bfloat16):
    """Each request's first rows as contiguous K/V ``[total_rows, Hkv, D]`` of
    ``dtype``: request r's are rows ``cu_seqlens_k[r] : cu_seqlens_k[r + 1]``.
    Rows of blocks outside the pool or the table are zeros."""
    cache, code, device = check_quantized_cache(key_cache, value_cache, key_scales,
                                                value_scales, "quantized_gather")
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("rows are read as float16, bfloat16 or float32")
    if block_tables.ndim != 2 or cu_seqlens_k.numel() != block_tables.shape[0] + 1:
        raise ValueError("cu_seqlens_k must have one entry more than block_tables has rows")
    if block_tables.get_device() != device or cu_seqlens_k.get_device() != device:
        _lib.require_device(block_tables, cu_seqlens_k, what="quantized_gather")
        raise ValueError("block_tables and cu_seqlens_k must be on the cache device")
    if type(total_rows) is not int or total_rows < 0:
        raise ValueError("total_rows must be a nonnegative integer")
    if device != _lib.raw_device():
        with torch.cuda.device(device):
            return quantized_gather(key_cache, value_cache, key_scales, value_scales,
                                    block_tables, cu_seqlens_k, total_rows, dtype=dtype)
    num_blocks, block_size, num_kv_heads, head_dim = key_cache.shape
    keys = key_cache.new_empty((total_rows, num_kv_heads, head_dim), dtype=dtype)
    values = torch.empty_like(keys)
    if total_rows == 0:
        return keys, values
    if block_tables.shape[0] == 0:
        raise ValueError("rows without requests")
    tables, offsets = index32(block_tables), index32(cu_seqlens_k)
    requests, width = tables.shape
    status = _lib.load().mi_quant_gather(
        *cache, tables.data_ptr(), width, width, offsets.data_ptr(), requests, total_rows,
        keys.data_ptr(), values.data_ptr(), num_kv_heads, head_dim, block_size, num_blocks,
        _lib.DTYPE_CODES[dtype], code, _lib.raw_stream(device))
    if status:
        _lib.check(status, "mi_quant_gather")
    return keys, values
