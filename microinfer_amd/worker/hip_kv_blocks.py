"""Copies of cache pages (blocks) through the HIP library.

``copy_blocks`` is what forked sequences, beams that change parents and a
compacted pool need of the cache: whole pages, or their first rows, copied to
other pages in every layer by one launch. The block manager's host lists go
with the launch, so there is no upload.
"""

from __future__ import annotations

from array import array

import torch

from microinfer_amd import _lib


def _host_ints(values, name: str) -> array:
    """An int32 host array of a list, tuple, range or integer numpy array."""
    if isinstance(values, torch.Tensor):
        if values.is_cuda:
            raise ValueError(f"{name} must be on the host: the block manager's lists")
        values = values.tolist()
    try:
        return array("i", values)
    except (TypeError, OverflowError) as exc:
        raise ValueError(f"{name} must be a list of integers: {exc}") from None


def copy_blocks(key_cache: torch.Tensor, value_cache: torch.Tensor, src, dst, *,
                tokens=None) -> None:
    """``K[..., dst[i], :tokens[i]] = K[..., src[i], :tokens[i]]`` for every
    pair, and the same for V, with all sources as they were before the call:
    ``pool[:, dst] = pool[:, src]`` of torch's indexing.

    ``key_cache``/``value_cache`` are one layer's ``[blocks, B, Hkv, D]`` views
    or all layers' ``[L, blocks, B, Hkv, D]``, of equal strides. ``src``, ``dst``
    and ``tokens`` (default: whole blocks) are host lists of equal length; no
    block is written twice (ValueError, like an id outside the cache, before
    anything is copied). A block may be read by several pairs and be written
    by another one (chains, swaps and cycles of up to 255 blocks). Runs on the
    current stream; a captured call replays the pairs of its capture.
    """
    _lib.require_device(key_cache, value_cache, what="block copy")
    if key_cache.ndim not in (4, 5) or key_cache.shape != value_cache.shape:
        raise ValueError("K/V caches must have matching [blocks, B, Hkv, D] or "
                         "[L, blocks, B, Hkv, D] shapes")
    if key_cache.stride() != value_cache.stride():
        raise ValueError("K/V caches must share one layout")
    if key_cache.dtype != value_cache.dtype or key_cache.device != value_cache.device:
        raise ValueError("K/V caches must have matching dtype and device")
    if key_cache.stride(-1) != 1:
        raise ValueError("cache head_dim must be contiguous")
    sources, targets = _host_ints(src, "src"), _host_ints(dst, "dst")
    rows = None if tokens is None else _host_ints(tokens, "tokens")
    pairs = len(sources)
    if len(targets) != pairs or (rows is not None and len(rows) != pairs):
        raise ValueError("src, dst and tokens must have one entry per pair")
    num_blocks, block_size = key_cache.shape[-4], key_cache.shape[-3]
    layers = key_cache.shape[0] if key_cache.ndim == 5 else 1
    if pairs == 0 or layers == 0:
        return
    layer_stride = key_cache.stride(0) if key_cache.ndim == 5 else 0
    with _lib.on_device(key_cache.device):
        status = _lib.load().mi_kv_copy_blocks(
            key_cache.data_ptr(), value_cache.data_ptr(), layer_stride, *key_cache.stride()[-4:-1],
            sources.buffer_info()[0], targets.buffer_info()[0],
            None if rows is None else rows.buffer_info()[0], pairs, layers,
            key_cache.shape[-2], key_cache.shape[-1], block_size, num_blocks,
            _lib.dtype_code(key_cache.dtype), _lib.stream_handle(key_cache.device))
    if status == _lib.MI_ERR_INVALID_ARGUMENT:  # the lists, before anything is copied
        raise ValueError(_lib.last_error())
    _lib.check(status, "mi_kv_copy_blocks")
