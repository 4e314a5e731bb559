"""NaN in an 8-bit cache under varlen attention of long requests: which rows it
reaches (more than 32 query rows a KV head, so that the kernel of long requests
runs; the other kernels are tested with decode steps).

A NaN in K or V makes NaN of the rows that see it. One in V may do so to earlier
rows of its request too; one in K does not, and none reaches another request. What
lies behind a context, in unused blocks or outside the pool reaches no row. Rows
that no NaN reaches are checked against float64 with the bounds of
``check_attention``.
"""

import numpy as np
import pytest
import torch

from microinfer_amd.layer.hip_quantized_attention import hip_quantized_prefill
from microinfer_amd.worker.hip_quantized_kv import quantized_append
from tests.quantized_support import DTYPES, Twin, check_attention, ints, tables_of

pytestmark = pytest.mark.gpu

VARLEN = {"bf16": (11, 2.0 ** -35), "f16": (11, 2.0 ** -35), "f32": (24, 0)}
HQ, HKV, BLOCK = 8, 2, 16
CONTEXTS, NEW = [150, 90, 40], [100, 90, 12]  # the last rows see most of it


class Case:
    def __init__(self, kind, dtype, dim, seed, width=None):
        rng = np.random.default_rng(seed)
        self.dim, self.dtype = dim, dtype
        self.twin = Twin(sum(-(-c // BLOCK) for c in CONTEXTS) + 3, BLOCK, HKV, dim, kind)
        self.twin.fill(rng)
        self.tables = tables_of(rng, CONTEXTS, BLOCK, self.twin.k.shape[0], width)
        self.cu_q = np.cumsum([0] + NEW).tolist()
        self.cu_k = np.cumsum([0] + CONTEXTS).tolist()
        query = rng.standard_normal((sum(NEW), HQ, dim))
        self.query = torch.from_numpy(query).to(DTYPES[dtype]).cuda()

    def __call__(self):
        return hip_quantized_prefill(self.query, *self.twin.tensors, ints(self.cu_q),
                                     ints(self.cu_k), ints(self.tables), max_seqlen_q=max(NEW))

    def check(self, got):
        check_attention(got, self.query, self.twin, self.tables, CONTEXTS, self.cu_q,
                        self.dim ** -0.5, VARLEN[self.dtype])

    def seeing(self, request, position, head):
        """Rows and query heads that see a position at a KV head."""
        seen = torch.zeros(self.query.shape[:2], dtype=torch.bool, device="cuda")
        first = max(0, position - (CONTEXTS[request] - NEW[request]))
        share = HQ // HKV
        seen[self.cu_q[request] + first:self.cu_q[request + 1],
             head * share:(head + 1) * share] = True
        return seen


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("request_,position", [(0, 70), (0, 33), (1, 64), (1, 15), (1, 88),
                                               (2, 39)])
def test_nan_in_k_reaches_the_rows_that_see_it(kind, dtype, dim, request_, position):
    case = Case(kind, dtype, dim, position)
    clean = case()
    case.check(clean)
    page = case.tables[request_][position // BLOCK]
    held = [t.clone() for t in case.twin.tensors]
    for what in ("scale", "code"):
        if what == "code" and kind == "int8":
            continue
        if what == "scale":  # of the position's whole block
            case.twin.layer.key_scales[page, 1] = float("nan")
            seen = case.seeing(request_, position // BLOCK * BLOCK, 1)
        else:
            case.twin.layer.keys[page, position % BLOCK, 1, 3:4].view(torch.uint8).fill_(0x7f)
            seen = case.seeing(request_, position, 1)
        got = case()
        assert got[seen].isnan().all()
        case.check(torch.where(seen[..., None], clean, got))
        for t, was in zip(case.twin.tensors, held):
            if t.dtype != torch.float32:
                t, was = t.view(torch.uint8), was.view(torch.uint8)
            t.copy_(was)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("request_,position", [(0, 70), (1, 20), (2, 39)])
def test_nan_in_v_stays_in_its_request(kind, dtype, dim, request_, position):
    case = Case(kind, dtype, dim, position)
    clean = case()
    page = case.tables[request_][position // BLOCK]
    mine = torch.zeros(case.query.shape[0], dtype=torch.bool, device="cuda")
    mine[case.cu_q[request_]:case.cu_q[request_ + 1]] = True
    if kind == "int8":
        case.twin.layer.value_scales[page, 0] = float("nan")
        got = case()
        assert got[case.seeing(request_, position // BLOCK * BLOCK, 0)].isnan().all()
    else:
        case.twin.layer.values[page, position % BLOCK, 0, 5:6].view(torch.uint8).fill_(0xff)
        got = case()
        assert got[case.seeing(request_, position, 0)][:, 5].isnan().all()
        assert not got[..., :5].isnan().any() and not got[..., 6:].isnan().any()
    assert not got[~mine].isnan().any() and not got[:, HQ // HKV:].isnan().any()
    case.check(torch.where(got.isnan(), clean, got))


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_no_row_sees_may_be_nan(kind, dtype, dim):
    """Behind the contexts, in their tables' further blocks, in unused ones and
    in those of ids outside the pool."""
    case = Case(kind, dtype, dim, 7, width=14)
    twin = case.twin
    used = {table[j] for table, c in zip(case.tables, CONTEXTS) for j in range(-(-c // BLOCK))}
    spare = [page for page in range(twin.k.shape[0]) if page not in used]
    for pool, scales in ((twin.layer.keys, twin.layer.key_scales),
                         (twin.layer.values, twin.layer.value_scales)):
        for page in spare:
            scales[page] = float("nan")
            pool[page].view(torch.uint8).fill_(0x7f)
        if kind == "fp8":
            for table, c in zip(case.tables, CONTEXTS):
                if c % BLOCK:
                    pool[table[c // BLOCK], c % BLOCK:].view(torch.uint8).fill_(0xff)
    for table, c in zip(case.tables, CONTEXTS):
        table[-(-c // BLOCK)] = spare[0]
    case.tables[1][2] = twin.k.shape[0] + 5
    case.tables[0][0] = -7
    case.check(case())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_written_values_that_are_not_finite(dtype, dim):
    """As appends write them: an infinite K value in an int8 cache makes its
    block's scale NaN, and the rows ahead of the block do not see it."""
    rng = np.random.default_rng(dim)
    rows = 96
    twin = Twin(rows // BLOCK, BLOCK, HKV, dim, "int8")
    keys, values = (torch.from_numpy(rng.standard_normal((rows, HKV, dim))).bfloat16().cuda()
                    for _ in range(2))
    table = rng.permutation(rows // BLOCK).tolist()
    slots = [table[p // BLOCK] * BLOCK + p % BLOCK for p in range(rows)]
    query = torch.from_numpy(rng.standard_normal((rows, HQ, dim))).to(DTYPES[dtype]).cuda()

    def run():
        return hip_quantized_prefill(query, *twin.tensors, ints([0, rows]), ints([0, rows]),
                                     ints([table]), max_seqlen_q=rows)

    quantized_append(*twin.tensors, ints(slots), keys, values)
    twin.expect(slots, keys, values)
    clean = run()
    keys[70, 0, 4] = float("inf")
    quantized_append(*twin.tensors, ints(slots), keys, values)
    got = run()
    assert got[64:, :4].isnan().all()
    assert not got[:64].isnan().any() and not got[:, 4:].isnan().any()
    got[64:, :4] = clean[64:, :4]
    check_attention(got, query, twin, [table], [rows], [0, rows], dim ** -0.5, VARLEN[dtype])
