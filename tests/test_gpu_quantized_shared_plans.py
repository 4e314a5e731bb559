"""Calls over an 8-bit cache that share a plan, from two threads and out of two
graphs at once, give the bits of the same call alone: partials are joined in the order of
their parts, so one that came from another call's workspace shows, however small."""

import threading

import numpy as np
import pytest
import torch

from microinfer_amd.layer.hip_quantized_attention import (hip_quantized_decode,
                                                          hip_quantized_prefill,
                                                          quantized_decode_plan,
                                                          quantized_prefill_plan)
from tests.quantized_support import DTYPES, Twin, ints, tables_of

pytestmark = pytest.mark.gpu

CONTEXTS = [1900, 700, 1300]
NEWS = [None, [5, 1, 3], [150, 40, 90]]  # decode, few rows a request, many


class Calls:
    def __init__(self, dtype, dim, seed):
        rng = np.random.default_rng(seed)
        self.twin = Twin(sum(-(-c // 16) for c in CONTEXTS) + 2, 16, 2, dim, "fp8")
        self.twin.fill(rng)
        self.tables = ints(tables_of(rng, CONTEXTS, 16, self.twin.k.shape[0]))
        self.lens = ints(CONTEXTS)
        self.cu_k = ints(np.cumsum([0] + CONTEXTS).tolist())
        self.cu_q = [None if new is None else ints(np.cumsum([0] + new).tolist())
                     for new in NEWS]
        self.sizes = dict(num_q_heads=8, num_kv_heads=2, head_dim=dim, dtype=DTYPES[dtype],
                          block_size=16, block_table_width=self.tables.shape[1])
        self.queries = [[torch.from_numpy(rng.standard_normal((sum(new or [1] * 3), 8, dim)))
                         .to(DTYPES[dtype]).cuda() for new in NEWS] for _ in range(2)]

    def plan(self, i):
        if NEWS[i] is None:
            return quantized_decode_plan(self.lens, **self.sizes)
        return quantized_prefill_plan(self.cu_q[i], self.cu_k, num_tokens=sum(NEWS[i]),
                                      max_seqlen_q=max(NEWS[i]), **self.sizes)

    def run(self, i, query, plan=None):
        if NEWS[i] is None:
            return hip_quantized_decode(query, *self.twin.tensors, self.tables, self.lens,
                                        plan=plan)
        return hip_quantized_prefill(query, *self.twin.tensors, self.cu_q[i], self.cu_k,
                                     self.tables, max_seqlen_q=max(NEWS[i]), plan=plan)

    def alone(self):
        outs = [[self.run(i, q) for i, q in enumerate(queries)] for queries in self.queries]
        torch.cuda.synchronize()
        return outs


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 64), ("f16", 128), ("bf16", 256)])
def test_two_threads(dtype, dim):
    calls = Calls(dtype, dim, 1)
    want = calls.alone()
    plans = [calls.plan(i) for i in range(len(NEWS))]
    torch.cuda.synchronize()
    results, errors = [None, None], []

    def work(who):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = [[calls.run(i, q, plans[i]) for i, q in enumerate(calls.queries[who])]
                        for _ in range(10)]
                torch.cuda.current_stream().synchronize()
            results[who] = outs
        except Exception as error:  # reported by the test's own thread
            errors.append(error)

    threads = [threading.Thread(target=work, args=(who,)) for who in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors
    for who in range(2):
        for outs in results[who]:
            for got, expected in zip(outs, want[who]):
                assert torch.equal(got, expected)


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 64), ("f16", 128), ("bf16", 256)])
def test_two_graphs(dtype, dim):
    """The plan is made in the first graph's capture and called in the second's."""
    calls = Calls(dtype, dim, 2)
    want = calls.alone()
    side = torch.cuda.Stream()
    for i in range(len(NEWS)):
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            plan = calls.plan(i)
            mine = calls.run(i, calls.queries[0][i], plan)
        first.replay()
        torch.cuda.synchronize()
        with torch.cuda.graph(second):
            theirs = calls.run(i, calls.queries[1][i], plan)
        for _ in range(5):
            mine.zero_()
            theirs.zero_()
            torch.cuda.synchronize()
            for _ in range(3):
                first.replay()
                with torch.cuda.stream(side):
                    second.replay()
            torch.cuda.synchronize()
            assert torch.equal(mine, want[0][i]) and torch.equal(theirs, want[1][i])
