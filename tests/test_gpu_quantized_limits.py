"""Attention over an 8-bit cache at the ends of what its arguments may be: more
partitions than a merge takes at once, softmax scales of any sign, contexts that reach
behind their tables."""

import numpy as np
import pytest
import torch

from microinfer_amd.layer.hip_quantized_attention import (hip_quantized_decode,
                                                          hip_quantized_prefill)
from tests.quantized_support import DTYPES, Twin, check_attention, ints, tables_of

pytestmark = pytest.mark.gpu

DECODE = {"bf16": (16, 0), "f16": (16, 0), "f32": (24, 0)}
VARLEN = {"bf16": (11, 2.0 ** -35), "f16": (11, 2.0 ** -35), "f32": (24, 0)}


def case(rng, contexts, heads, dim, kind, dtype, rows, block=16):
    hq, hkv = heads
    blocks = sum(-(-c // block) for c in contexts)
    twin = Twin(blocks + 1, block, hkv, dim, kind)
    twin.fill(rng)
    query = torch.from_numpy(rng.standard_normal((rows, hq, dim))).to(DTYPES[dtype]).cuda()
    return twin, tables_of(rng, contexts, block, blocks + 1), query


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,dim,rows", [
    (1, 128, 1), (8, 128, 3), (24, 128, 1), (30, 64, 1), (8, 128, 13), (3, 64, 41), (5, 256, 11)])
def test_many_partitions(dtype, hq, dim, rows):
    """One KV head and a long context: more than 32 partitions to merge."""
    rng = np.random.default_rng(dim + rows)
    context = 9000
    twin, tables, query = case(rng, [context], (hq, 1), dim, "fp8", dtype, rows)
    got = hip_quantized_prefill(query, *twin.tensors, ints([0, rows]), ints([0, context]),
                                ints(tables), max_seqlen_q=rows)
    check_attention(got, query, twin, tables, [context], [0, rows], dim ** -0.5, DECODE[dtype])
    got = hip_quantized_decode(query[:1], *twin.tensors, ints(tables), ints([context]))
    check_attention(got, query[:1], twin, tables, [context], [0, 1], dim ** -0.5, DECODE[dtype])


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0, -5.0])
@pytest.mark.parametrize("dim,block", [(128, 16), (64, 32), (256, 16), (32, 16)])
def test_scales_of_any_sign(kind, scale, dim, block):
    """Scores up to some hundred apart. A weight below 2^-126 of the largest is lost: it
    is no normal float32 number. Where all that leads has codes of 0 in a dim, that is
    what counts there. Such a weight meets V of up to MOST vs, where vs is within 2^8 of
    the leading position's (``Twin.fill``), whose weight is 2^-8 of the sum at least (of
    150 positions): 2^-110 of ``peak`` for each position, times MOST."""
    rng = np.random.default_rng(dim)
    flushed = 2.0 ** -110
    decode, varlen = ({t: (bits, lost + flushed) for t, (bits, lost) in weights.items()}
                      for weights in (DECODE, VARLEN))
    contexts, lengths = [150, 70, 30], [90, 1, 30]
    cu_q = [0, 90, 91, 121]
    cu_k = ints(np.cumsum([0] + contexts).tolist())
    for dtype in DTYPES:
        twin, tables, query = case(rng, contexts, (6, 2), dim, kind, dtype, 121, block)
        got = hip_quantized_prefill(query, *twin.tensors, ints(cu_q), cu_k, ints(tables),
                                    max_seqlen_q=90, scale=scale)
        check_attention(got, query, twin, tables, contexts, cu_q, scale, varlen[dtype])
        got = hip_quantized_prefill(query[:4], *twin.tensors, ints([0, 2, 3, 4]), cu_k,
                                    ints(tables), max_seqlen_q=2, scale=scale)
        check_attention(got, query[:4], twin, tables, contexts, [0, 2, 3, 4], scale,
                        decode[dtype])
        got = hip_quantized_decode(query[:3], *twin.tensors, ints(tables), ints(contexts),
                                   scale=scale)
        check_attention(got, query[:3], twin, tables, contexts, [0, 1, 2, 3], scale,
                        decode[dtype])


@pytest.mark.parametrize("dim,block", [(128, 16), (64, 64), (256, 16), (32, 16), (128, 8)])
def test_contexts_longer_than_their_tables(dim, block):
    """Positions behind a table's last block are not there; rows of few positions
    see what is."""
    rng = np.random.default_rng(block)
    contexts, lengths = [150, 70, 30], [90, 8, 30]
    cu_q = np.cumsum([0] + lengths).tolist()
    cu_k = ints(np.cumsum([0] + contexts).tolist())
    twin, tables, query = case(rng, contexts, (4, 2), dim, "fp8", "bf16", sum(lengths), block)
    width = 64 // block
    short = [row[:width] for row in tables]
    got = hip_quantized_prefill(query, *twin.tensors, ints(cu_q), cu_k, ints(short),
                                max_seqlen_q=90)
    check_attention(got, query, twin, short, contexts, cu_q, dim ** -0.5, VARLEN["bf16"])
    got = hip_quantized_prefill(query[:6], *twin.tensors, ints([0, 2, 5, 6]), cu_k, ints(short),
                                max_seqlen_q=3)
    check_attention(got, query[:6], twin, short, contexts, [0, 2, 5, 6], dim ** -0.5,
                    DECODE["bf16"])
    got = hip_quantized_decode(query[:3], *twin.tensors, ints(short), ints(contexts))
    check_attention(got, query[:3], twin, short, contexts, [0, 1, 2, 3], dim ** -0.5,
                    DECODE["bf16"])
