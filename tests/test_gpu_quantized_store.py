"""Quantised writes and reads on the GPU against the float64 oracle: codes and
scales bit for bit, whatever the order of the slots and the way they are found.
"""

import numpy as np
import pytest
import torch

from microinfer_amd import _lib
from microinfer_amd.worker import hip_quantized_kv
from microinfer_amd.worker.hip_quantized_kv import (QuantizedAppendPlan, quantized_append,
                                                    quantized_append_plan, quantized_gather)
from tests.quantized_support import CODES, DTYPES, Twin, ints, tables_of
from oracle import quantized as oracle

pytestmark = pytest.mark.gpu


def rows_of(gen, tokens, heads, dim, dtype, size=1.0):
    x = size * torch.randn(2, tokens, heads, dim, generator=gen)
    return [t.to(dtype).cuda() for t in x]


@pytest.fixture(params=[False, True], ids=["scanned", "planned"])
def planned(request, monkeypatch):
    """Small calls find their rows in the list, or have them from a plan."""
    monkeypatch.setattr(hip_quantized_kv, "MAX_SCANNED_TOKENS", 0 if request.param else 1024)
    return request.param


def write(twin, slots, keys, values, plan=True, index=torch.int32):
    """Through the library and through the twin."""
    where = torch.tensor(slots, dtype=index, device="cuda")
    blocks, block = twin.k.shape[:2]
    quantized_append(*twin.tensors, where, keys, values,
                     plan=quantized_append_plan(where, block_size=block, num_blocks=blocks)
                     if plan else None)
    twin.expect(slots, keys, values)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,dim,block,layout", [
    (8, 128, 16, "paired"), (3, 64, 32, "head_major"), (2, 16, 4, "token_major"),
    (1, 256, 64, "paired"), (5, 32, 1, "token_major"), (2, 128, 256, "paired")])
def test_blocks_fill_over_several_calls(kind, dtype, heads, dim, block, layout, planned):
    gen = torch.Generator().manual_seed(heads + dim)
    blocks = 12
    twin = Twin(blocks, block, heads, dim, kind, layout)
    order = np.random.default_rng(1).permutation(blocks).tolist()

    def slots(seq, begin, end):
        return [order[4 * seq + p // block] * block + p % block for p in range(begin, end)]

    lengths = [0, 0, 0]
    # Chunks, then single rows, of magnitudes that rise and fall.
    for step, (news, size) in enumerate([((1, 5, block), 1.0), ((2, 0, 3), 0.01), ((1, 1, 1), 3.0),
                                         ((block, 2, 1), 40.0), ((1, 1, 0), 1e-3),
                                         ((0, 1, 1), 5000.0)]):
        news = [min(n, 4 * block - length) for n, length in zip(news, lengths)]
        where = [s for seq, n in enumerate(news)
                 for s in slots(seq, lengths[seq], lengths[seq] + n)]
        keys, values = rows_of(gen, len(where), heads, dim, DTYPES[dtype], size)
        write(twin, where, keys, values, plan=step % 2,
              index=torch.int64 if step == 2 else torch.int32)
        lengths = [length + n for length, n in zip(lengths, news)]
        twin.check()


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("tokens", [1, 7, 64, 1024, 1025, 3000])
def test_any_order_of_slots(kind, tokens, planned):
    """Scanned and planned calls find a block's rows wherever they stand."""
    gen = torch.Generator().manual_seed(tokens)
    rng = np.random.default_rng(tokens)
    blocks, block = max(2 * tokens // 16, 4), 16
    twin = Twin(blocks, block, 2, 64, kind)
    slots = rng.permutation(blocks * block)[:tokens]
    slots[rng.random(tokens) < 0.05] = -1
    slots[rng.random(tokens) < 0.05] = blocks * block + 3
    keys, values = rows_of(gen, tokens, 2, 64, torch.bfloat16)
    write(twin, slots.tolist(), keys, values, index=torch.int64 if tokens == 64 else torch.int32)
    twin.check()


def test_every_16_bit_value():
    """Every finite 16-bit input that the scale of its row's block leaves in
    range rounds as the oracle does; rows of one block each."""
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
        keys = x.reshape(256, 2, 128).cuda()
        for kind in CODES:
            twin = Twin(256, 2, 2, 128, kind)
            write(twin, [2 * i for i in range(256)], keys, keys.flip(0).contiguous())
            twin.check()


def test_extreme_float32_rows():
    values = [0.0, 1e-45, 1.2e-38, 448 * 2.0 ** -126, 3.4e38, -3.4e38, 448.0, 127.0, 449.0, 127.5]
    rows = torch.tensor(values).repeat_interleave(16).view(10, 1, 16)
    rows[:, 0, 1:] *= torch.linspace(-1, 1, 15)
    rows = rows.cuda()
    for kind in CODES:
        twin = Twin(10, 4, 1, 16, kind)
        write(twin, [4 * i for i in range(10)], rows, -rows)
        write(twin, [4 * i + 2 for i in range(10)], rows.flip(0), rows)
        twin.check()


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_values_that_are_not_finite(kind, planned):
    gen = torch.Generator().manual_seed(5)
    twin = Twin(8, 16, 2, 128, kind)
    keys, values = rows_of(gen, 20, 2, 128, torch.bfloat16)
    keys[3, 1, 7] = float("nan")
    values[18, 0, 0] = float("-inf")
    values[2] = float("inf")
    write(twin, list(range(30, 50)), keys, values)
    twin.check()
    write(twin, [50], keys[:1], values[:1])  # a block that holds NaN
    write(twin, [32], keys[5:6], values[5:6])  # and one that begins anew
    twin.check()


def test_rows_with_equal_slots_are_not_mixed(planned):
    gen = torch.Generator().manual_seed(6)
    keys, values = rows_of(gen, 40, 2, 128, torch.float16)
    got = Twin(2, 16, 2, 128, "fp8")
    quantized_append(*got.tensors, ints([5] * 30 + [6] * 10), keys, values)
    codes = [t.cpu().double().numpy() for t in got.tensors]
    found = 0
    for i in range(30):
        for j in range(30, 40):
            want = Twin(2, 16, 2, 128, "fp8", device="cpu")
            want.expect([5, 6], keys[[i, j]], values[[i, j]])
            found += all(np.array_equal(a, b) for a, b in
                         zip(codes, (want.k, want.v, want.ks, want.vs)))
    assert found >= 1


def test_fused_rows_and_strides():
    """K and V out of one fused projection's rows, and unaligned ones."""
    gen = torch.Generator().manual_seed(7)
    fused = torch.randn(9, (4 + 2 + 2) * 64, generator=gen).to(torch.bfloat16).cuda()
    keys = fused[:, 4 * 64:6 * 64].view(9, 2, 64)
    values = fused[:, 6 * 64:].view(9, 2, 64)
    for kind in CODES:
        twin = Twin(3, 8, 2, 64, kind)
        write(twin, list(range(4, 13)), keys, values)
        odd = torch.randn(9, 2, 65, generator=gen).to(torch.bfloat16).cuda()[..., 1:]
        write(twin, list(range(12, 21)), odd, values)
        twin.check()


def test_checked_and_fast_writes_of_a_cache():
    gen = torch.Generator().manual_seed(8)
    twin = Twin(4, 16, 2, 32, "fp8")
    keys, values = rows_of(gen, 6, 2, 32, torch.float32)
    slots = [3, 4, 5, 16, 17, -1]
    twin.layer.write_checked(ints(slots), keys, values)
    twin.expect(slots, keys, values)
    twin.layer.write_fast(ints([2, 2, 3, 0, 9, -1]), ints([0, 1, 16, 6, 0, 1]), keys, values)
    twin.expect([32, 33, -1, 6, -1, -1], keys, values)
    twin.check()
    with pytest.raises(ValueError, match="duplicate"):
        twin.layer.write_checked(ints([3, 3, 1, 2, 4, 5]), keys, values)
    with pytest.raises(ValueError, match="outside"):
        twin.layer.write_checked(ints([64, 3, 1, 2, 4, 5]), keys, values)
    twin.check()


def test_what_a_plan_held_before_does_not_matter(monkeypatch):
    """A plan's memory of an earlier step, and of anything else."""
    monkeypatch.setattr(hip_quantized_kv, "MAX_SCANNED_TOKENS", 0)
    gen = torch.Generator().manual_seed(9)
    rng = np.random.default_rng(0)
    twin = Twin(6, 16, 2, 64, "int8")
    keys, values = rows_of(gen, 20, 2, 64, torch.bfloat16)
    lib = _lib.load()
    nbytes = lib.mi_quant_append_plan_bytes(20, 16, 6)
    noise = torch.from_numpy(rng.integers(-9, 30, nbytes // 4).astype(np.int32)).cuda()
    for begin in (40, 33, 61):
        where = list(range(begin, begin + 20))
        slots = ints(where)
        lib.mi_quant_append_plan(slots.data_ptr(), 0, 20, 16, 6, noise.data_ptr(), nbytes,
                                 _lib.stream_handle(slots.device))
        plan = QuantizedAppendPlan(noise.view(torch.uint8), (20, 16, 6), nbytes)
        quantized_append(*twin.tensors, slots, keys, values, plan=plan)
        twin.expect(where, keys, values)
        twin.check()


def test_calls_refuse_plans_of_other_sizes():
    gen = torch.Generator().manual_seed(9)
    twin = Twin(6, 16, 2, 64, "int8")
    keys, values = rows_of(gen, 20, 2, 64, torch.bfloat16)
    slots = ints(list(range(20)))
    for sizes in ((19, 16, 6), (20, 32, 6), (20, 16, 5)):
        plan = quantized_append_plan(slots[:sizes[0]], block_size=sizes[1], num_blocks=sizes[2])
        with pytest.raises(ValueError, match="plan"):
            quantized_append(*twin.tensors, slots, keys, values, plan=plan)
    with pytest.raises(ValueError, match="one slot"):
        quantized_append(*twin.tensors, slots[1:], keys, values)
    with pytest.raises(ValueError, match="alike"):
        quantized_append(*twin.tensors, slots, keys, values.float())
    with pytest.raises(ValueError, match="heads"):
        quantized_append(*twin.tensors, slots, keys[:, :1], values[:, :1])
    with pytest.raises(ValueError, match="layout"):
        quantized_append(twin.layer.keys, twin.layer.values.contiguous(), *twin.tensors[2:],
                         slots, keys, values)
    with pytest.raises(ValueError, match="scales"):
        quantized_append(*twin.tensors[:2], *(t.double() for t in twin.tensors[2:]), slots, keys,
                         values)
    twin.check()


def test_captured_writes_replay_with_other_rows(planned):
    gen = torch.Generator().manual_seed(10)
    twin = Twin(16, 16, 2, 128, "fp8")
    slots = ints([0] * 40)
    keys, values = rows_of(gen, 40, 2, 128, torch.bfloat16)

    def call():
        plan = quantized_append_plan(slots, block_size=16, num_blocks=16)
        quantized_append(*twin.tensors, slots, keys, values, plan=plan)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for t in twin.tensors:
        t.view(torch.uint8 if t.element_size() == 1 else torch.float32).zero_()
    at = 0
    for step in range(3):
        where = list(range(at, at + 38)) + [-1, -1]
        at += 38
        new = rows_of(gen, 40, 2, 128, torch.bfloat16, 10.0 ** step)
        slots.copy_(ints(where))
        keys.copy_(new[0])
        values.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        twin.expect(where, keys, values)
        twin.check()


def test_another_stream():
    gen = torch.Generator().manual_seed(11)
    stream = torch.cuda.Stream()
    twin = Twin(80, 16, 4, 128, "int8")
    keys, values = rows_of(gen, 1200, 4, 128, torch.float16)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        quantized_append(*twin.tensors, ints(list(range(7, 1207))), keys, values)
    stream.synchronize()
    twin.expect(list(range(7, 1207)), keys, values)
    twin.check()


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,dim,block,layout", [
    (8, 128, 16, "paired"), (3, 64, 32, "head_major"), (5, 16, 4, "token_major"),
    (1, 256, 1, "paired"), (12, 32, 64, "token_major")])
def test_reads_are_what_the_cache_stands_for(kind, dtype, heads, dim, block, layout):
    rng = np.random.default_rng(heads)
    twin = Twin(60, block, heads, dim, kind, layout)
    twin.fill(rng)
    contexts = [1, 0, 5 * block, 3 * block - 1, 0, block // 2 + 1]
    tables = tables_of(rng, contexts, block, 60)
    tables[3][1] = -1 if len(tables[3]) > 1 else tables[3][0]
    tables[2][0] = 60
    cu = np.cumsum([0] + contexts).tolist()
    got = quantized_gather(*twin.tensors, ints(tables), ints(cu), cu[-1], dtype=DTYPES[dtype])
    for x, codes, scales in zip(got, (twin.k, twin.v), (twin.ks, twin.vs)):
        want = torch.from_numpy(oracle.gather(codes, scales, tables, contexts)).to(DTYPES[dtype])
        assert torch.equal(x.cpu(), want)


def test_reads_of_any_scale_round_once():
    """Scales that are no powers of two, and NaN ones."""
    rng = np.random.default_rng(3)
    twin = Twin(6, 16, 2, 64, "fp8")
    twin.fill(rng)
    twin.ks[:] = rng.random(twin.ks.shape).astype(np.float32)
    twin.ks[2, 1] = np.nan
    twin.layer.key_scales.copy_(torch.from_numpy(twin.ks).float())
    tables = [[2, 0, 5]]
    got, _ = quantized_gather(*twin.tensors, ints(tables), ints([0, 40]), 40, dtype=torch.float32)
    want = torch.from_numpy(oracle.gather(twin.k, twin.ks, tables, [40])).float()
    assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))


def test_a_written_cache_reads_back_within_half_a_step():
    gen = torch.Generator().manual_seed(12)
    keys, values = rows_of(gen, 100, 8, 128, torch.float32)
    for kind in CODES:
        twin = Twin(8, 16, 8, 128, kind)
        quantized_append(*twin.tensors, ints(list(range(100))), keys, values)
        got = quantized_gather(*twin.tensors, ints([list(range(7))]), ints([0, 100]), 100,
                               dtype=torch.float32)
        for x, y, scales in zip(got, (keys, values), twin.tensors[2:]):
            s = scales[torch.arange(100, device="cuda") // 16][..., None]
            # int8: half a step of the scale; e4m3: 2^-4 of the value, half of
            # 2^-9 of the scale below its normal range.
            bound = s / 2 if kind == "int8" else torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10)
            assert bool(((x - y).abs() <= bound).all())


@pytest.mark.parametrize("layout", ["paired", "head_major", "token_major"])
def test_copied_blocks_take_their_scales(layout):
    rng = np.random.default_rng(4)
    twin = Twin(10, 16, 3, 64, "int8", layout)
    twin.fill(rng)
    twin.cache.copy_blocks([1, 2, 3, 7], [4, 1, 2, 8], tokens=[16, 16, 5, 0])
    for codes, scales in ((twin.k, twin.ks), (twin.v, twin.vs)):
        before = codes.copy()
        codes[4], codes[1] = before[1], before[2]
        codes[2, :5] = before[3, :5]
        scales[[4, 1, 2]] = scales[[1, 2, 3]]
    twin.check()
