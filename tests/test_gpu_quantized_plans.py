"""Plans of attention over an 8-bit cache that are not what a call made: memory that
holds anything, as a plan does whose graph has not been replayed yet."""

import numpy as np
import pytest
import torch

from microinfer_amd.layer.hip_quantized_attention import (hip_quantized_decode,
                                                          quantized_decode_plan)
from tests.quantized_support import Twin, check_attention, ints, tables_of

pytestmark = pytest.mark.gpu

LAST = 2 ** 31 - 1
# Sequences, Hq, Hkv, D, block; the last two are the vector kernel's.
SHAPES = [(8, 2, 128, 16), (8, 2, 64, 32), (4, 1, 256, 16), (6, 2, 32, 16), (8, 2, 128, 8)]


@pytest.mark.parametrize("shape", SHAPES)
def test_items_that_name_nothing_are_left_out(shape):
    """Items whose numbers overflow when they are added or scaled, and random
    ones: each is left out, or reads and writes what is the call's."""
    hq, hkv, dim, block = shape
    rng = np.random.default_rng(dim + block)
    contexts = [70, 90, 50, 40]
    blocks = sum(-(-c // block) for c in contexts)
    twin = Twin(blocks, block, hkv, dim, "fp8")
    twin.fill(rng)
    tables = tables_of(rng, contexts, block, blocks)
    width = len(tables[0])
    query = torch.from_numpy(rng.standard_normal((4, hq, dim))).bfloat16().cuda()
    plan = quantized_decode_plan(ints(contexts), num_q_heads=hq, num_kv_heads=hkv, head_dim=dim,
                                 dtype=query.dtype, block_size=block, block_table_width=width)
    items = np.full((plan.bytes // 32, 8), -1, dtype=np.int32)
    # Sequence, first and last block, parts, first item, context, part, nothing.
    crafted = [
        (0, 0, width, 1, 0, contexts[0], 0, 0),
        # A first block whose position is past 31 bits: nothing of the sequence.
        (1, 2 ** 31 // block, width, 1, 1, contexts[1], 0, 0),
        (2, 0, width, LAST, 5, contexts[2], LAST - 1, 0),
        (2, 0, width, LAST, LAST, contexts[2], 3, 0),
        (2, 0, width, 1, LAST, contexts[2], 0, 0),
        (2, 0, width, 2, len(items) - 1, contexts[2], 0, 0),
        (2, 0, width, 0, 0, contexts[2], 0, 0), (2, 0, width, 2, 0, contexts[2], 2, 0),
        (2, 0, width, 2, 0, contexts[2], -1, 0), (2, 0, width, 1, -1, contexts[2], 0, 0),
        (4, 0, width, 1, 0, contexts[2], 0, 0), (LAST, 0, width, 1, 0, contexts[2], 0, 0)]
    items[:len(crafted)] = crafted
    noise = items[len(crafted):]
    noise[:] = rng.integers(-2 ** 31, 2 ** 31, noise.shape)
    noise[:, 0] = 3
    small = rng.random(noise.shape) < 0.5
    small[:, 0] = False
    noise[small] = rng.integers(-2, 9, noise.shape)[small]
    plan.buffer[:plan.bytes].copy_(torch.from_numpy(items.reshape(-1).view(np.uint8)).cuda())
    got = hip_quantized_decode(query, *twin.tensors, ints(tables), ints(contexts), plan=plan)
    torch.cuda.synchronize()
    assert not got[1].any()
    check_attention(got[:1], query[:1], twin, tables[:1], contexts[:1], [0, 1], dim ** -0.5,
                    (16, 0))
