"""Host side of the 8-bit cache (no GPU): CPU tensors raise RuntimeError; the C
entries reject bad sizes, strides and pointers before launching anything.
"""

import pytest
import torch

from microinfer_amd import _lib
from microinfer_amd.layer.hip_quantized_attention import (hip_quantized_decode,
                                                          hip_quantized_prefill,
                                                          quantized_decode_plan,
                                                          quantized_prefill_plan)
from microinfer_amd.worker.hip_quantized_kv import (quantized_append, quantized_append_plan,
                                                    quantized_gather)
from microinfer_amd.worker.kv_cache import KVCache, LayerKVCache


def test_cpu_tensors_raise_runtime_error():
    cache = KVCache(1, 4, 16, 2, 64, dtype=torch.int8).layer(0)
    tensors = cache.keys, cache.values, cache.key_scales, cache.value_scales
    rows = torch.zeros(3, 2, 64)
    index = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(3, 2, dtype=torch.int32)
    cu = torch.zeros(4, dtype=torch.int32)
    sizes = dict(num_q_heads=2, num_kv_heads=2, head_dim=64, dtype=torch.float32, block_size=16,
                 block_table_width=2)
    for call in (lambda: quantized_append(*tensors, index, rows, rows),
                 lambda: cache.write_slots(index, rows, rows),
                 lambda: quantized_append_plan(index, block_size=16, num_blocks=4),
                 lambda: quantized_gather(*tensors, table, cu, 3),
                 lambda: hip_quantized_decode(rows, *tensors, table, index),
                 lambda: quantized_decode_plan(index, **sizes),
                 lambda: quantized_prefill_plan(cu, cu, num_tokens=3, **sizes),
                 lambda: hip_quantized_prefill(rows, *tensors, cu, cu, table, max_seqlen_q=1)):
        with pytest.raises(RuntimeError, match="HIP device only"):
            call()


@pytest.mark.parametrize("layout", ["paired", "head_major", "token_major"])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_caches_of_8_bits_have_scales(layout, dtype):
    cache = KVCache(2, 5, 16, 3, 64, dtype=dtype, layout=layout)
    assert cache.quantized and cache.keys.shape == (2, 5, 16, 3, 64)
    assert cache.key_scales.shape == cache.value_scales.shape == (2, 5, 3)
    assert cache.num_bytes == 2 * 2 * 5 * 3 * (16 * 64 + 4)
    layer = cache.layer(1)
    layer.value_scales[4, 2] = 3.0
    assert cache.value_scales[1, 4, 2] == 3 and cache.key_scales[1, 4, 2] == 0
    plain = KVCache(1, 5, 16, 3, 64)
    assert not plain.quantized and plain.key_scales is None and plain.layer(0).key_scales is None


def test_layers_refuse_scales_that_do_not_fit():
    codes = torch.zeros(4, 16, 2, 64, dtype=torch.int8)
    scales = torch.zeros(4, 2)
    LayerKVCache(codes, codes, scales, scales)
    for bad in ((None, None), (scales, None), (scales, torch.zeros(4, 3))):
        with pytest.raises(ValueError, match="scales"):
            LayerKVCache(codes, codes, *bad)
    with pytest.raises(ValueError, match="scales"):
        LayerKVCache(codes.float(), codes.float(), scales, scales)


CACHE = dict(keys=4096, values=8192, bs=4096, ts=128, hs=2048, ks=4096, vs=4100, sbs=4, shs=2)


def _args(order, over):
    unknown = set(over) - set(order)
    assert not unknown, unknown
    return [over.get(k, v) for k, v in order.items()]


def _append(lib, **over):
    order = dict(rows_k=4096, kts=256, khs=128, rows_v=8192, vts=256, vhs=128, **CACHE, slots=4096,
                 is64=0, plan=None, plan_bytes=0, tokens=3, heads=2, dim=128, block=16, blocks=8,
                 dtype=2, code=0)
    return lib.mi_quant_append(*_args(order, over), None)


def _gather(lib, **over):
    order = dict(**CACHE, tables=4096, tstride=4, width=4, cu=4096, requests=2, total=5, ko=4096,
                 vo=4096, heads=2, dim=128, block=16, blocks=8, dtype=2, code=1)
    return lib.mi_quant_gather(*_args(order, over), None)


def _decode(lib, **over):
    order = dict(q=4096, qts=512, qhs=128, **CACHE, tables=4096, tstride=4, width=4, plan=4096,
                 plan_bytes=1 << 20, out=4096, ots=512, ohs=128, ws=4096, ws_bytes=1 << 30,
                 counters=4096, seqs=2, hq=4, heads=2, dim=128, block=16, blocks=8, scale=0.1,
                 dtype=2, code=0)
    return lib.mi_quant_decode(*_args(order, over), None)


def _prefill(lib, **over):
    order = dict(q=4096, qts=512, qhs=128, **CACHE, cu_q=4096, cu_k=4096, tables=4096, tstride=4,
                 width=4, out=4096, ots=512, ohs=128, ws=4096, ws_bytes=1 << 30, tokens=9,
                 requests=2, longest=9, hq=4, heads=2, dim=128, block=16, blocks=8, scale=0.1,
                 dtype=2, code=0)
    return lib.mi_quant_prefill(*_args(order, over), None)


@pytest.mark.parametrize("call", [_append, _gather, _decode, _prefill])
def test_c_entries_validate_the_cache(call):
    lib = _lib.load()
    assert call(lib, dtype=7) == 1 and "dtype" in _lib.last_error()
    assert call(lib, code=2) == 1 and "code" in _lib.last_error()
    for name in ("heads", "blocks", "dim"):
        assert call(lib, **{name: 0}) == 1
    for dim in (8, 96, 512):
        assert call(lib, dim=dim) == 2 and "head_dim" in _lib.last_error()
    assert call(lib, block=12) == 1 and "block_size" in _lib.last_error()
    for name in ("keys", "values", "ks", "vs"):
        assert call(lib, **{name: None}) == 1 and "null" in _lib.last_error()
    for name in ("bs", "ts", "hs", "sbs", "shs"):
        assert call(lib, **{name: -8}) == 1 and "stride" in _lib.last_error()
    for name in ("keys", "values", "bs", "ts", "hs"):
        assert call(lib, **{name: 4100}) == 1 and "misaligned" in _lib.last_error()
    for name in ("ks", "vs"):
        assert call(lib, **{name: 4098}) == 1 and "misaligned" in _lib.last_error()


def test_c_append_validates_the_rows():
    lib = _lib.load()
    for name in ("rows_k", "rows_v", "slots"):
        assert _append(lib, **{name: None}) == 1 and "null" in _lib.last_error()
    for name in ("rows_k", "kts", "khs", "rows_v", "vts", "vhs"):
        assert _append(lib, **{name: 4100}) == 1 and "misaligned" in _lib.last_error()
    assert _append(lib, tokens=-1) == 1
    assert _append(lib, tokens=1025) == 2 and "plan" in _lib.last_error()
    assert _append(lib, block=2048) == 2
    assert _append(lib, tokens=0, rows_k=None) == 0
    need = lib.mi_quant_append_plan_bytes(2000, 16, 8)
    assert need > 8 * 16 * 4 and lib.mi_quant_append_plan_bytes(0, 16, 8) == 0
    assert _append(lib, tokens=2000, plan=4096, plan_bytes=need - 1) == 3
    assert _append(lib, tokens=2000, plan=4100, plan_bytes=need) == 3

    def plan(slots=4096, tokens=2000, block=16, blocks=8, buffer=4096, nbytes=need):
        return lib.mi_quant_append_plan(slots, 0, tokens, block, blocks, buffer, nbytes, None)

    assert plan(block=12) == 1 and plan(tokens=-3) == 1 and plan(blocks=0) == 1
    assert plan(slots=None) == 1 and plan(buffer=None) == 1
    assert plan(nbytes=need - 1) == 3 and plan(buffer=4100) == 3
    assert plan(tokens=0, slots=None, buffer=None) == 0


def test_c_gather_validates_its_rows():
    lib = _lib.load()
    for name in ("requests", "total", "width"):
        assert _gather(lib, **{name: -1}) == 1
    assert _gather(lib, requests=0) == 1 and "requests" in _lib.last_error()
    for name in ("cu", "ko", "vo", "tables"):
        assert _gather(lib, **{name: None}) == 1 and "null" in _lib.last_error()
    for name in ("ko", "vo"):
        assert _gather(lib, **{name: 4104}) == 1 and "misaligned" in _lib.last_error()
    assert _gather(lib, total=0, cu=None) == 0


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_c_attention_validates_its_rows(call):
    lib = _lib.load()
    for bad in (dict(hq=0), dict(hq=3), dict(hq=-2)):
        assert call(lib, **bad) == 1 and "multiple" in _lib.last_error()
    assert call(lib, width=-1) == 1
    assert call(lib, tables=None) == 1 and "null" in _lib.last_error()
    assert call(lib, width=1 << 27) == 2 and "2^30" in _lib.last_error()
    for name in ("q", "out"):
        assert call(lib, **{name: None}) == 1 and "null" in _lib.last_error()
    for name in ("q", "qts", "qhs", "out", "ots", "ohs"):
        assert call(lib, **{name: 4100}) == 1 and "misaligned" in _lib.last_error()


def test_c_decode_validates_plan_and_workspace():
    lib = _lib.load()
    assert _decode(lib, plan=None) == 1
    assert _decode(lib, plan=4112) == 3 and _decode(lib, plan_bytes=31) == 3
    need = lib.mi_quant_decode_workspace_bytes(2, 4, 2, 128)
    assert _decode(lib, ws_bytes=need - 1) == 3 and str(need) in _lib.last_error()
    assert _decode(lib, ws=None) == 3 and _decode(lib, counters=None) == 3
    assert _decode(lib, seqs=-1) == 1 and _decode(lib, seqs=4097) == 2
    assert _decode(lib, seqs=0, q=None) == 0

    def plan(ctx=4096, seqs=2, hq=4, hkv=2, dim=128, block=16, width=4, dtype=2, buf=4096,
             nbytes=1 << 20, counters=4096):
        return lib.mi_quant_decode_plan(ctx, seqs, hq, hkv, dim, block, width, dtype, buf, nbytes,
                                        counters, None)

    assert plan(dtype=9) == 1 and plan(hq=3) == 1 and plan(seqs=-1) == 1 and plan(width=-1) == 1
    assert plan(block=3) == 1 and plan(width=1 << 27) == 2 and plan(seqs=4097) == 2
    assert plan(ctx=None) == 1 and plan(buf=None) == 1 and plan(counters=None) == 1
    assert plan(nbytes=8) == 3 and plan(buf=4100) == 3 and plan(seqs=0) == 0


def test_c_prefill_validates_its_requests():
    lib = _lib.load()
    assert _prefill(lib, tokens=-1) == 1 and _prefill(lib, requests=-1) == 1
    assert _prefill(lib, requests=0) == 1 and "requests" in _lib.last_error()
    for name in ("cu_q", "cu_k"):
        assert _prefill(lib, **{name: None}) == 1 and "null" in _lib.last_error()
    assert _prefill(lib, tokens=0, q=None) == 0
    assert _prefill(lib, longest=0) == 1 and "max_seqlen_q" in _lib.last_error()
    # Few rows a request, and many.
    for tokens, longest in ((9, 9), (900, 2), (900, 900)):
        need = lib.mi_quant_prefill_workspace_bytes(tokens, 2, longest, 4, 2, 128, 16)
        sizes = dict(tokens=tokens, longest=longest)
        assert need > 0 and _prefill(lib, ws_bytes=need - 1, **sizes) == 3
        assert str(need) in _lib.last_error()
        assert _prefill(lib, ws=None, **sizes) == 3 and _prefill(lib, ws=4112, **sizes) == 3
    for sizes in ((0, 2, 9, 4, 2, 128, 16), (9, 0, 9, 4, 2, 128, 16), (9, 2, 9, 3, 2, 128, 16),
                  (9, 2, 0, 4, 2, 128, 16), (9, 2, 9, 4, 2, 32, 16), (9, 2, 9, 4, 2, 128, 8),
                  (9, 2, 9, 258, 2, 128, 16)):
        assert lib.mi_quant_prefill_workspace_bytes(*sizes) == 0
    need = lib.mi_quant_prefill_workspace_bytes(9, 2, 9, 4, 2, 128, 16)

    def plan(cu_q=4096, cu_k=4096, tokens=9, requests=2, longest=9, hq=4, hkv=2, dim=128,
             block=16, width=4, ws=4096, nbytes=1 << 30):
        return lib.mi_quant_prefill_plan(cu_q, cu_k, tokens, requests, longest, hq, hkv, dim,
                                         block, width, ws, nbytes, None)

    assert plan(hq=3) == 1 and plan(dim=32) == 2 and plan(tokens=0) == 2
    assert plan(block=24) == 1 and plan(width=-1) == 1 and plan(width=1 << 27) == 2
    assert plan(cu_q=None) == 1 and plan(cu_k=None) == 1
    assert plan(ws=None) == 3 and plan(nbytes=need - 1) == 3 and plan(ws=4104) == 3


def test_capture_id_wants_somewhere_to_put_it():
    lib = _lib.load()
    assert lib.mi_stream_capture_id(None, None) == 1 and "null" in _lib.last_error()
