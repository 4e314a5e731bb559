"""Host side of page copies (no GPU): CPU tensors raise RuntimeError; the C
entry rejects bad ids, counts, sizes and pointers before launching anything.
"""

import ctypes

import pytest
import torch

from microinfer_amd import _lib
from microinfer_amd.worker.hip_kv_blocks import _host_ints, copy_blocks


def test_cpu_pools_raise_runtime_error():
    pool = torch.zeros(2, 8, 4, 2, 16)
    with pytest.raises(RuntimeError, match="HIP device only"):
        copy_blocks(pool, pool.clone(), [0], [1])


def test_lists_are_host_integers():
    assert list(_host_ints((1, 2), "src")) == [1, 2]
    assert list(_host_ints(torch.tensor([3, 4]), "src")) == [3, 4]
    for bad in ([1.5], [2 ** 40], ["a"], 3, [None]):
        with pytest.raises(ValueError, match="src"):
            _host_ints(bad, "src")


def _call(lib, src=(0, 1), dst=(2, 3), tokens=None, **over):
    def ints(values):
        return None if values is None else (ctypes.c_int32 * max(len(values), 1))(*values)

    args = dict(keys=4096, values=8192, ls=1 << 16, bs=4096, ts=128, hs=2048, src=ints(src),
                dst=ints(dst), tokens=ints(tokens), pairs=len(src or dst), layers=2, heads=2,
                dim=128, block=16, blocks=8, dtype=2)
    args.update(over)
    return lib.mi_kv_copy_blocks(*args.values(), None)


def test_c_entry_validates_before_launch():
    lib = _lib.load()
    assert _call(lib, dtype=5) == 1 and "dtype" in _lib.last_error()
    for name in ("layers", "heads", "dim", "block", "blocks"):
        assert _call(lib, **{name: 0}) == 1 and "sizes" in _lib.last_error()
    assert _call(lib, pairs=-1) == 1
    for name in ("ls", "bs", "ts", "hs"):
        assert _call(lib, **{name: -16}) == 1 and "stride" in _lib.last_error()
    assert _call(lib, heads=1 << 20, block=1 << 10) == 2
    assert _call(lib, dim=1 << 20) == 2 and _call(lib, layers=1 << 17) == 2
    assert _call(lib, keys=None) == 1 and "null" in _lib.last_error()
    assert _call(lib, values=None) == 1 and _call(lib, src=None) == 1
    assert _call(lib, dst=None) == 1
    assert _call(lib, keys=4097) == 1 and "misaligned" in _lib.last_error()
    assert _call(lib, src=(0, 8)) == 1 and "block id" in _lib.last_error()
    assert _call(lib, src=(0, -1)) == 1 and _call(lib, dst=(2, 8)) == 1
    assert _call(lib, dst=(2, -7)) == 1
    assert _call(lib, tokens=(0, 17)) == 1 and "tokens" in _lib.last_error()
    assert _call(lib, tokens=(-1, 3)) == 1
    assert _call(lib, dst=(2, 2)) == 1 and "twice" in _lib.last_error()
    assert _call(lib, dst=(2, 2), tokens=(0, 16)) == 1
    # The same in a pool of many more blocks than pairs.
    big = dict(blocks=1 << 20)
    assert _call(lib, src=(0, 1 << 20), **big) == 1 and "block id" in _lib.last_error()
    assert _call(lib, dst=(9, 9), **big) == 1 and "twice" in _lib.last_error()
    assert _call(lib, dst=(9, 9), tokens=(0, 16), **big) == 1
    assert _call(lib, tokens=(0, 17), **big) == 1 and "tokens" in _lib.last_error()
    ring = tuple(range(300))
    assert _call(lib, src=ring, dst=ring[1:] + ring[:1], **big) == 2
    assert _call(lib, src=ring, dst=ring[1:] + ring[:1], blocks=300) == 2
    assert "cycle" in _lib.last_error()


def test_nothing_to_copy_is_no_launch():
    lib = _lib.load()
    assert _call(lib, src=(), dst=()) == 0
    assert _call(lib, tokens=(0, 0)) == 0
    assert _call(lib, src=(4, 5), dst=(4, 5)) == 0
    assert _call(lib, src=(4, 5), dst=(4, 5), blocks=5000) == 0
    assert _call(lib, src=(4, 5), dst=(5, 6), tokens=(0, 0), blocks=5000) == 0
    assert _lib.last_error() == ""
