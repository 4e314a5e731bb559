"""Host side of token log probabilities (no GPU): CPU tensors raise
RuntimeError; the C entry rejects bad sizes, pointers and workspaces before
launching anything.
"""

import pytest
import torch

from microinfer_amd import _lib
from microinfer_amd.layer.hip_logprobs import token_logprobs


def test_cpu_tensors_raise_runtime_error():
    with pytest.raises(RuntimeError, match="HIP device only"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


def _call(lib, **over):
    args = dict(logits=4096, stride=1000, rows=4, vocab=1000, dtype=2, temperatures=4096,
                tokens=4096, token_stride=2, given=2, logprobs=4096, entropy=4096,
                top_tokens=4096, top_logprobs=4096, top=5, workspace=4096,
                workspace_bytes=1 << 20, counters=4096)
    args.update(over)
    return lib.mi_token_logprobs(*args.values(), None)


def test_c_entry_validates_before_launch():
    lib = _lib.load()
    assert _call(lib, dtype=4) == 1 and "dtype" in _lib.last_error()
    for bad in (dict(rows=-1), dict(vocab=0), dict(given=-1), dict(top=-1)):
        assert _call(lib, **bad) == 1 and "sizes" in _lib.last_error()
    assert _call(lib, top=33) == 1 and "num_top" in _lib.last_error()
    assert _call(lib, vocab=4, stride=4, top=5) == 1
    assert _call(lib, vocab=(1 << 30) + 1, stride=1 << 31) == 2
    assert _call(lib, given=65537, token_stride=65537) == 2
    for name in ("logits", "tokens", "logprobs", "top_tokens", "top_logprobs"):
        assert _call(lib, **{name: None}) == 1 and "null" in _lib.last_error()
    assert _call(lib, stride=999) == 1 and "row_stride" in _lib.last_error()
    assert _call(lib, token_stride=1) == 1
    for name in ("logits", "temperatures", "tokens", "logprobs", "entropy", "top_tokens",
                 "top_logprobs"):
        assert _call(lib, **{name: 4097}) == 1 and "misaligned" in _lib.last_error()
    assert _call(lib, rows=(1 << 31) - 1, workspace=None, counters=None) == 2
    assert "too many rows" in _lib.last_error()
    assert _call(lib, rows=0) == 0 and _lib.last_error() == ""


def test_workspace_is_checked():
    lib = _lib.load()
    size = lib.mi_token_logprobs_workspace_bytes
    assert size(0, 1000, 5, 2) == 0 and size(4, 1000, 5, 9) == 0
    assert size(4096, 151936, 20, 2) == 0  # rows enough to fill the chip stay whole
    need = size(2, 151936, 5, 2)
    assert need > 0 and need % (2 * (16 + 5 * 8)) == 0
    big = dict(rows=2, vocab=151936, stride=151936)
    assert _call(lib, **big, workspace=None) == 3 and "workspace" in _lib.last_error()
    assert _call(lib, **big, workspace_bytes=need - 1) == 3
    assert _call(lib, **big, workspace=4104) == 3
    assert _call(lib, **big, counters=None) == 3 and "counters" in _lib.last_error()


def test_parts_of_any_number_of_rows():
    # A whole number of records per row, none where the rows fill the chip, up
    # to the last int32.
    size = _lib.load().mi_token_logprobs_workspace_bytes
    for rows in (1, 2, 19, 64, 100, 333, 700, 1000, 1024, 1025, 1281, (1 << 31) - 1024,
                 (1 << 31) - 1):
        for vocab, dtype in ((4096, 2), (32003, 0), (151936, 1), (1 << 30, 2)):
            need = size(rows, vocab, 8, dtype)
            assert need >= 0 and need % (rows * (16 + 64)) == 0
            parts = need // (rows * (16 + 64))
            assert parts != 1 and parts <= 64 and (rows <= 1024 or parts == 0)
            assert rows * parts <= 1280 or parts == 0
