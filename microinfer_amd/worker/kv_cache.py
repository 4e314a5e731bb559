"""Runner-owned paged KV storage and zero-copy per-layer views.

Mirrors ``LayerKVCache`` / ``KVCache`` (microinfer/worker/kv_cache.py:10-118):
same constructor, ``layer(i)``, ``num_bytes``, ``keys``/``values`` and
``write_checked``/``write_fast`` contracts. Two things differ by design:

* Physical layout. By default one allocation holds both pools, paired per
  block and KV head: ``[L, N, Hkv, 2, B, D]`` with K at index 0 and V at 1,
  so one KV head's 16-token block of K and of V is one contiguous 8 KiB run
  (bf16, D=128) -- measured 2-4 % faster than separate pools on long decode
  contexts, equal on short ones. ``layout="head_major"`` keeps separate
  ``[L, N, Hkv, B, D]`` pools (4 KiB runs); ``layout="token_major"`` is the
  reference's contiguous ``[L, N, B, Hkv, D]``. In every layout
  ``keys``/``values`` are views with the reference's logical shape
  ``[L, N, B, Hkv, D]`` and equal strides, so indexing
  (``cache.keys[l, blk, off]``) reads exactly what the reference would; the
  kernels take the view's strides.
* 8-bit pools. ``dtype=torch.float8_e4m3fn`` or ``torch.int8`` makes a pool of
  codes with a float32 scale for each block and KV head (``key_scales`` /
  ``value_scales``, logical shape ``[L, N, Hkv]``, K's beside V's); writes
  quantise (``hip_quantized_kv``).
* Writes run on the GPU only (no advanced-indexing CPU fallback,
  kv_cache.py:78-79); a CPU cache can be built and validated but not written.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from microinfer_amd.worker.hip_kv_blocks import _host_ints as host_ints
from microinfer_amd.worker.hip_kv_blocks import copy_blocks
from microinfer_amd.worker.hip_kv_store import launch_append
from microinfer_amd.worker.hip_quantized_kv import (QUANTIZED_DTYPES, QuantizedAppendPlan,
                                                    quantized_append)

LAYOUTS = ("paired", "head_major", "token_major")


@dataclass(frozen=True)
class LayerKVCache:
    """One layer's logical ``[blocks, B, Hkv, D]`` K/V views; no pool or layer id.
    8-bit ones have their scales ``[blocks, Hkv]`` beside them."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor | None = None
    value_scales: torch.Tensor | None = None

    def __post_init__(self):
        if self.keys.ndim != 4 or self.keys.shape != self.values.shape:
            raise ValueError("K/V must have matching [blocks, B, Hkv, D] shapes")
        if self.keys.dtype != self.values.dtype or self.keys.device != self.values.device:
            raise ValueError("K/V must have matching dtype and device")
        if self.quantized:
            for scales in (self.key_scales, self.value_scales):
                if scales is None or scales.shape != (self.keys.shape[0], self.keys.shape[2]):
                    raise ValueError("8-bit K/V need scales of shape [blocks, Hkv]")
        elif self.key_scales is not None or self.value_scales is not None:
            raise ValueError("only 8-bit K/V have scales")

    @property
    def block_size(self):
        return self.keys.shape[1]

    @property
    def quantized(self) -> bool:
        return self.keys.dtype in QUANTIZED_DTYPES

    def _write(self, index0, index1, keys, values, plan=None):
        if not self.quantized:
            launch_append(self.keys, self.values, index0, index1, keys, values)
            return
        slots = index0
        if index1 is not None:
            if index0.shape != index1.shape:
                raise ValueError("one offset per block is required")
            inside = (index0 >= 0) & (index1 >= 0) & (index1 < self.block_size)
            slots = torch.where(inside, index0 * self.block_size + index1, -1)
        quantized_append(self.keys, self.values, self.key_scales, self.value_scales, slots,
                         keys, values, plan=plan)

    def write_checked(self, slots, keys, values):
        """Checked write (kv_cache.py:30-50): -1 skips padding; validates first.

        Every check runs before any storage changes, so an invalid write leaves
        the cache untouched.
        """
        if slots.ndim != 1 or slots.dtype not in (torch.int32, torch.int64):
            raise ValueError("slots must be a 1-D integer tensor")
        expected = (slots.numel(), *self.keys.shape[2:])
        if keys.shape != expected or values.shape != expected:
            raise ValueError("K/V shape must match slots and cache heads")
        if any(t.device != self.keys.device for t in (slots, keys, values)):
            raise ValueError("slots and K/V must be on the cache device")
        capacity = self.keys.shape[0] * self.block_size
        if bool(torch.any(slots < -1)) or bool(torch.any(slots >= capacity)):
            raise ValueError("slot outside cache")
        used = slots[slots >= 0].long()
        if used.unique().numel() != used.numel():
            raise ValueError("duplicate slot")
        if slots.numel() == 0:
            return
        if not self.quantized:
            keys = keys.to(self.keys.dtype)
            values = values.to(self.values.dtype)
        self._write(slots, None, keys, values)

    def write_fast(self, blocks, offsets, keys, values):
        """Hot path (kv_cache.py:52-79): caller guarantees valid, unique slots."""
        self._write(blocks, offsets, keys, values)

    def write_slots(self, slot_mapping, keys, values, plan: QuantizedAppendPlan | None = None):
        """Hot path with the step's int32 slot map; -1 entries are skipped.

        Duplicate slots are allowed (graph pad rows share the pad block);
        which duplicate lands is unspecified. ``plan``: the step's
        ``quantized_append_plan``, for 8-bit caches.
        """
        if plan is not None and not self.quantized:
            raise ValueError("only 8-bit caches are written by a plan")
        self._write(slot_mapping, None, keys, values, plan)


class KVCache:
    """KV pool for every layer, logical shape ``[L, N, B, Hkv, D]`` (zeros)."""

    def __init__(
        self,
        num_layers,
        num_blocks,
        block_size,
        num_kv_heads,
        head_dim,
        *,
        dtype=torch.float32,
        device="cpu",
        layout: str = "paired",
    ):
        dimensions = (num_layers, num_blocks, block_size, num_kv_heads, head_dim)
        if any(d <= 0 for d in dimensions):
            raise ValueError("cache dimensions must be positive")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = torch.device(device)
        self.layout = layout
        if layout == "paired":
            physical = (num_layers, num_blocks, num_kv_heads, 2, block_size, head_dim)
            self._storage = torch.zeros(physical, dtype=dtype, device=device)
            self._key_storage = self._storage[:, :, :, 0]
            self._value_storage = self._storage[:, :, :, 1]
            self.keys = self._key_storage.permute(0, 1, 3, 2, 4)
            self.values = self._value_storage.permute(0, 1, 3, 2, 4)
        elif layout == "head_major":
            physical = (num_layers, num_blocks, num_kv_heads, block_size, head_dim)
            self._key_storage = torch.zeros(physical, dtype=dtype, device=device)
            self._value_storage = torch.zeros_like(self._key_storage)
            self.keys = self._key_storage.permute(0, 1, 3, 2, 4)
            self.values = self._value_storage.permute(0, 1, 3, 2, 4)
        else:
            self._key_storage = torch.zeros(dimensions, dtype=dtype, device=device)
            self._value_storage = torch.zeros_like(self._key_storage)
            self.keys = self._key_storage
            self.values = self._value_storage
        self.key_scales = self.value_scales = None
        if self.quantized:
            self._scale_storage = torch.zeros(num_layers, num_blocks, num_kv_heads, 2,
                                              device=device)
            self.key_scales = self._scale_storage[..., 0]
            self.value_scales = self._scale_storage[..., 1]

    @property
    def quantized(self) -> bool:
        return self.dtype in QUANTIZED_DTYPES

    @property
    def num_bytes(self):
        pools = [self.keys, self.values]
        if self.quantized:
            pools += [self.key_scales, self.value_scales]
        return sum(p.numel() * p.element_size() for p in pools)

    def copy_blocks(self, src, dst, tokens=None) -> None:
        """Copy blocks (or their first ``tokens[i]`` rows) to other blocks in
        every layer: ``hip_kv_blocks.copy_blocks`` over the whole pool. In an
        8-bit pool a destination takes its source's scales too, so that its
        other rows no longer stand for what they did."""
        if not self.quantized:
            copy_blocks(self.keys, self.values, src, dst, tokens=tokens)
            return
        # The copies move bytes: pairs of codes as 16-bit words, a block's
        # scales as one row of a head each.
        src, dst = host_ints(src, "src"), host_ints(dst, "dst")
        moved = range(len(src))
        if tokens is not None:
            # A pair that copies nothing leaves its destination's scales too.
            tokens = host_ints(tokens, "tokens")
            moved = [i for i, n in enumerate(tokens) if n != 0]
        copy_blocks(self.keys.view(torch.float16), self.values.view(torch.float16), src, dst,
                    tokens=tokens)
        scales = [s[:, :, None, :, None] for s in (self.key_scales, self.value_scales)]
        copy_blocks(*scales, [src[i] for i in moved], [dst[i] for i in moved])

    def layer(self, index: int) -> LayerKVCache:
        """Basic indexing shares storage; binding does not copy the cache."""
        if not 0 <= index < self.num_layers:
            raise ValueError("layer outside cache")
        if not self.quantized:
            return LayerKVCache(self.keys[index], self.values[index])
        return LayerKVCache(self.keys[index], self.values[index], self.key_scales[index],
                            self.value_scales[index])
