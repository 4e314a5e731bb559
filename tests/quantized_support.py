"""Caches in 8 bits for the tests: a pool on the device and its float64 twin."""

from __future__ import annotations

import numpy as np
import torch

from microinfer_amd.worker.kv_cache import KVCache
from oracle import quantized as oracle

CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Twin:
    """One layer of a cache on ``device`` and what it should hold."""

    def __init__(self, blocks, block, heads, dim, kind, layout="paired", device="cuda"):
        self.kind = kind
        self.cache = KVCache(1, blocks, block, heads, dim, dtype=CODES[kind], device=device,
                             layout=layout)
        self.layer = self.cache.layer(0)
        self.k, self.v = np.zeros((2, blocks, block, heads, dim))
        self.ks, self.vs = np.zeros((2, blocks, heads))

    @property
    def tensors(self):
        return (self.layer.keys, self.layer.values, self.layer.key_scales,
                self.layer.value_scales)

    def expect(self, slots, keys, values):
        """The write of these rows, in the twin."""
        for codes, scales, rows in ((self.k, self.ks, keys), (self.v, self.vs, values)):
            oracle.append(codes, scales, [int(s) for s in slots],
                          rows.double().cpu().numpy(), self.kind)

    def check(self):
        """The cache's codes and scales are the twin's, bit for bit."""
        for got, want in zip(self.tensors, (self.k, self.v, self.ks, self.vs)):
            got = got.cpu().double().numpy()
            np.testing.assert_array_equal(got, want)

    def fill(self, rng, sizes=None):
        """Random codes everywhere; scales of a power of two for each block and
        head, within 2^-4 .. 2^4 (or ``sizes``)."""
        blocks, block, heads, dim = self.k.shape
        for codes, scales, pool, s in ((self.k, self.ks, self.layer.keys, self.layer.key_scales),
                                       (self.v, self.vs, self.layer.values,
                                        self.layer.value_scales)):
            most = oracle.MOST[self.kind]
            x = rng.standard_normal(codes.shape) * most / 5
            codes[:] = oracle.nearest(np.clip(x, -most, most), self.kind)
            low, high = sizes or (-4, 4)
            exponents = rng.integers(low, high + 1, scales.shape)
            scales[:] = np.exp2(exponents - np.floor(np.log2(most)))
            values = torch.from_numpy(codes).float().to(pool.device)
            pool.view(torch.uint8).copy_(values.to(pool.dtype).view(torch.uint8))
            s.copy_(torch.from_numpy(scales).float())


def tables_of(rng, contexts, block, blocks, width=None):
    """-1 padded tables of distinct blocks."""
    need = [-(-c // block) for c in contexts]
    width = max(need + [1]) if width is None else width
    ids = iter(rng.permutation(blocks).tolist())
    return [[next(ids) for _ in range(n)] + [-1] * (width - n) for n in need]


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def check_attention(got, query, twin, tables, contexts, cu_q, scale, weights):
    """``got`` against float64, with the bounds of the arithmetic.

    A score is a sum of D products in float32, then a few factors: off by at
    most (D + 8) 2^-24 of scale * sum |q k| (``reach``), and the weight exp(s) of
    it by that plus the rounding of its argument (2^-24 |s|) and of exp2 (2^-22).
    Weights and their sum both carry it: twice. A sum of n weighted values in
    float32 adds n 2^-24 of sum p |v| at most, partitions and waves merge in a
    few more. ``weights``: (bits, lost): a weight times its V scale is rounded to
    2^-bits of it for the product with V, and f16 rounds it to 2^-25 at most
    where the row's largest is 2^10 or more, lost = 2^-35 of that (``peak``) for
    each of n, times a code of up to MOST. The result rounds to the output's type
    by half a step.
    """
    out, around, reach, peak = oracle.attention(
        query.double().cpu().numpy(), twin.k, twin.v, twin.ks, twin.vs, tables, contexts, cu_q,
        scale)
    bits, lost = weights
    dim = query.shape[-1]
    n = max([1] + [int(c) for c in contexts])
    weight = 2 * ((dim + 8) * 2.0 ** -24 + 2.0 ** -24) * reach + 2 * 2.0 ** -22
    bound = (weight[..., None] + n * 2.0 ** -24 + 16 * 2.0 ** -24 + 2 * 2.0 ** -bits) * around
    bound += n * lost * oracle.MOST[twin.kind] * peak[..., None]
    half = torch.finfo(got.dtype).eps / 2
    bound += half * (np.abs(out) + bound) + torch.finfo(got.dtype).smallest_normal * half * 2
    err = np.abs(got.double().cpu().numpy() - out)
    worst = np.unravel_index(np.argmax(np.nan_to_num(err - bound, nan=np.inf)), err.shape)
    assert np.all(err <= bound), (worst, err[worst], bound[worst], out[worst])
