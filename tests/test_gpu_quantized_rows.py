"""Rows of varlen calls over an 8-bit cache that belong to no request: behind the
last one and ahead of the first. Every kernel leaves them as they were."""

import numpy as np
import pytest
import torch

from microinfer_amd import _lib
from tests.quantized_support import DTYPES, Twin, check_attention, ints, tables_of

pytestmark = pytest.mark.gpu

CONTEXTS = [300, 70, 95]
WEIGHTS = {"bf16": (11, 2.0 ** -35), "f32": (24, 0)}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,block", [(128, 16), (64, 16), (256, 16), (32, 16), (128, 8)])
@pytest.mark.parametrize("lengths", [[3, 0, 2], [60, 1, 90]])
def test_rows_of_no_request_stay(dtype, dim, block, lengths):
    rng = np.random.default_rng(dim + block)
    hq, hkv, ahead, behind = 8, 2, 5, 40
    blocks = sum(-(-c // block) for c in CONTEXTS)
    twin = Twin(blocks, block, hkv, dim, "fp8")
    twin.fill(rng)
    tables = tables_of(rng, CONTEXTS, block, blocks)
    rows = sum(lengths)
    total = ahead + rows + behind
    query = torch.from_numpy(rng.standard_normal((total, hq, dim))).to(DTYPES[dtype]).cuda()
    out = torch.full_like(query, 7.0)
    offsets = np.cumsum([0] + lengths)
    cu_q, cu_k = ints((offsets + ahead).tolist()), ints(np.cumsum([0] + CONTEXTS).tolist())
    at = ints(tables)
    lib, stream = _lib.load(), _lib.stream_handle(query.device)
    sizes = total, 3, max(lengths), hq, hkv, dim, block
    nbytes = lib.mi_quant_prefill_workspace_bytes(*sizes)
    assert (nbytes == 0) == (dim == 32 or block == 8 or (dim == 256 and max(lengths) > 64))
    workspace = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
    if nbytes:
        _lib.check(lib.mi_quant_prefill_plan(cu_q.data_ptr(), cu_k.data_ptr(), *sizes,
                                             at.shape[1], workspace.data_ptr(), nbytes, stream),
                   "mi_quant_prefill_plan")
    keys, values, ks, vs = twin.tensors
    _lib.check(lib.mi_quant_prefill(
        query.data_ptr(), hq * dim, dim, keys.data_ptr(), values.data_ptr(), *keys.stride()[:3],
        ks.data_ptr(), vs.data_ptr(), *ks.stride(), cu_q.data_ptr(), cu_k.data_ptr(),
        at.data_ptr(), at.shape[1], at.shape[1], out.data_ptr(), hq * dim, dim,
        workspace.data_ptr(), nbytes, total, 3, max(lengths), hq, hkv, dim, block, blocks, 0.1,
        _lib.DTYPE_CODES[query.dtype], 0, stream), "mi_quant_prefill")
    check_attention(out[ahead:ahead + rows], query[ahead:ahead + rows], twin, tables, CONTEXTS,
                    offsets.tolist(), 0.1, WEIGHTS[dtype])
    assert bool((out[:ahead] == 7).all()) and bool((out[ahead + rows:] == 7).all())
