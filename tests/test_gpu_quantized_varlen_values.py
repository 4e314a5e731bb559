"""Varlen attention over an 8-bit cache where values of V are zero for whole
blocks: such a block's scale is the least there is, 2^-126, beside ordinary ones.

The requests have more than 32 query rows a KV head, so they run on the kernel of
long requests. Bounds are those of ``check_attention`` with the weights of that
kernel (one f16 part for 16-bit queries, three bf16 parts for float32).
"""

import numpy as np
import pytest
import torch

from microinfer_amd.layer.hip_quantized_attention import hip_quantized_prefill
from microinfer_amd.worker.hip_quantized_kv import quantized_append
from tests.quantized_support import DTYPES, Twin, check_attention, ints

pytestmark = pytest.mark.gpu

VARLEN = {"bf16": (11, 2.0 ** -35), "f16": (11, 2.0 ** -35), "f32": (24, 0)}
HEADS = 8, 2


def written(rng, keys, values, kind, block):
    """A cache that holds these rows (numpy, float64), and its table."""
    tokens, heads, dim = keys.shape
    blocks = -(-tokens // block)
    twin = Twin(blocks + 1, block, heads, dim, kind)
    table = rng.permutation(blocks + 1)[:blocks].tolist()
    slots = [table[p // block] * block + p % block for p in range(tokens)]
    rows = [torch.from_numpy(x).to(torch.bfloat16).cuda() for x in (keys, values)]
    quantized_append(*twin.tensors, ints(slots), *rows)
    twin.expect(slots, *rows)
    twin.check()
    return twin, table


def attend(query, twin, table, context):
    new = query.shape[0]
    return hip_quantized_prefill(query, *twin.tensors, ints([0, new]), ints([0, context]),
                                 ints([table]), max_seqlen_q=new)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context,new,zeros", [
    (60, 60, range(16)),  # the first block: rows that see nothing else
    (1800, 60, range(1760)),  # a part of the keys, up to the middle of the new rows
    (1800, 60, range(1600, 1760)),
    (200, 60, range(200)),  # everywhere
    (150, 90, range(64, 80))])
def test_blocks_of_zeros_in_v(kind, dtype, dim, context, new, zeros):
    rng = np.random.default_rng(dim + context + len(zeros))
    hq, hkv = HEADS
    keys, values = rng.standard_normal((2, context, hkv, dim))
    values[list(zeros)] = 0
    twin, table = written(rng, keys, values, kind, 16)
    query = torch.from_numpy(rng.standard_normal((new, hq, dim))).to(DTYPES[dtype]).cuda()
    got = attend(query, twin, table, context)
    for i in range(new):
        if set(range(context - new + i + 1)) <= set(zeros):
            assert not got[i].any()
    check_attention(got, query, twin, [table], [context], [0, new], dim ** -0.5, VARLEN[dtype])


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lead", [90, 118, 124, 200])
def test_a_block_of_zeros_that_leads(kind, dtype, dim, lead):
    """Softmax weights of a block whose V is zero are 2^lead times the others': what
    those add is that much smaller, and counts all the same."""
    rng = np.random.default_rng(lead + dim)
    hq, hkv = HEADS
    context, new = 90, 40
    keys, values = 0.05 * rng.standard_normal((2, context, hkv, dim))
    keys[:, :, 0] = -4
    keys[16:32, :, 0] = 4  # exact in both types
    values *= 40
    values[16:32] = 0
    twin, table = written(rng, keys, values, kind, 16)
    query = 0.05 * rng.standard_normal((new, hq, dim))
    scale = dim ** -0.5
    query[:, :, 0] = lead * np.log(2) / (8 * scale)
    query = torch.from_numpy(query).to(DTYPES[dtype]).cuda()
    got = attend(query, twin, table, context)
    check_attention(got, query, twin, [table], [context], [0, new], scale, VARLEN[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lead,first", [(60, 0), (118, 896), (118, 1744), (200, 400)])
def test_blocks_of_zeros_that_lead_in_one_part(dtype, dim, lead, first):
    """The same among keys that are split, whose parts are merged: 60 rows on 1800."""
    rng = np.random.default_rng(lead + dim + first)
    hq, hkv = HEADS
    context, new = 1800, 60
    keys, values = 0.05 * rng.standard_normal((2, context, hkv, dim))
    keys[:, :, 0] = -4
    keys[first:first + 32, :, 0] = 4
    values *= 40
    values[first:first + 32] = 0
    twin, table = written(rng, keys, values, "fp8", 16)
    query = 0.05 * rng.standard_normal((new, hq, dim))
    scale = dim ** -0.5
    query[:, :, 0] = lead * np.log(2) / (8 * scale)
    query = torch.from_numpy(query).to(DTYPES[dtype]).cuda()
    got = attend(query, twin, table, context)
    check_attention(got, query, twin, [table], [context], [0, new], scale, VARLEN[dtype])
