"""Host side of decode over shared pages (no GPU): CPU tensors raise
RuntimeError; the C entries reject bad sizes, pointers and buffers before
launching anything.
"""

import pytest
import torch

from microinfer_amd import _lib
from microinfer_amd.layer.hip_shared_decode import (SharedDecodePlan, shared_decode_plan,
                                                    supported_shared_decode)


def _plan(**over):
    args = dict(context_lens=torch.zeros(2, dtype=torch.int32),
                group_starts=torch.zeros(2, dtype=torch.int32),
                shared_blocks=torch.zeros(1, dtype=torch.int32), num_q_heads=16, num_kv_heads=8,
                head_dim=128, dtype=torch.bfloat16, block_size=16, block_table_width=4)
    args.update(over)
    return shared_decode_plan(**args)


def test_cpu_tensors_raise_runtime_error():
    with pytest.raises(RuntimeError, match="HIP device only"):
        _plan()


def test_shapes_with_a_kernel():
    shape = dict(num_q_heads=16, num_kv_heads=8, head_dim=128, dtype=torch.float16,
                 block_size=16, num_seqs=3)
    assert supported_shared_decode(**shape)
    for other in (dict(num_q_heads=136), dict(head_dim=64), dict(dtype=torch.float32),
                  dict(block_size=8), dict(num_seqs=0), dict(num_seqs=4097)):
        assert not supported_shared_decode(**{**shape, **other})


def _plan_call(lib, **over):
    args = dict(lens=4096, seqs=4, starts=4096, shared=4096, groups=2, hq=16, hkv=8, dim=128,
                block=16, width=64, dtype=2, plan=4096, plan_bytes=1 << 20)
    args.update(over)
    return lib.mi_shared_decode_plan(*args.values(), None)


def _call(lib, **over):
    args = dict(q=4096, q_ts=2048, q_hs=128, kc=4096, vc=4096, bs=16384, ts=128, hs=2048,
                tables=4096, t_stride=64, width=64, plan=4096, plan_bytes=1 << 20, out=4096,
                o_ts=2048, o_hs=128, workspace=4096, ws_bytes=1 << 30, seqs=4, hq=16, hkv=8,
                dim=128, block=16, blocks=100, scale=1.0, dtype=2)
    args.update(over)
    return lib.mi_shared_decode(*args.values(), None)


@pytest.mark.parametrize("call", [_plan_call, _call])
def test_shapes_are_checked_before_launch(call):
    lib = _lib.load()
    assert call(lib, dtype=7) == 1 and "dtype" in _lib.last_error()
    for bad in (dict(seqs=-1), dict(hq=0), dict(hkv=0), dict(dim=0), dict(width=-1)):
        assert call(lib, **bad) == 1 and "sizes" in _lib.last_error()
    assert call(lib, hq=12) == 1 and "multiple" in _lib.last_error()
    assert call(lib, block=24) == 1 and "block_size" in _lib.last_error()
    for none in (dict(dtype=0), dict(dim=64), dict(hq=136), dict(block=8), dict(seqs=4097),
                 dict(width=1 << 27), dict(seqs=4096, hkv=4096, hq=4096)):
        assert call(lib, **none) == 2
    assert call(lib, plan=None) == 3 and "plan" in _lib.last_error()
    assert call(lib, plan=4112) == 3 and call(lib, plan_bytes=100) == 3
    assert call(lib, seqs=0) == 0 and _lib.last_error() == ""


def test_plan_pointers_are_checked():
    lib = _lib.load()
    assert _plan_call(lib, groups=-1) == 1 and "num_groups" in _lib.last_error()
    assert _plan_call(lib, groups=4097) == 2 and "groups" in _lib.last_error()
    for name in ("lens", "starts", "shared"):
        assert _plan_call(lib, **{name: None}) == 1 and "null" in _lib.last_error()
        assert _plan_call(lib, **{name: 4098}) == 1 and "misaligned" in _lib.last_error()
    need = lib.mi_shared_decode_plan_bytes(4, 16, 8)
    assert need % 32 == 0 and _plan_call(lib, plan_bytes=need - 1) == 3
    assert lib.mi_shared_decode_plan_bytes(0, 16, 8) == 0
    assert lib.mi_shared_decode_workspace_bytes(0, 16, 8) == 0


def test_call_pointers_are_checked():
    lib = _lib.load()
    for name in ("q", "kc", "vc", "tables", "out"):
        assert _call(lib, **{name: None}) == 1 and "null" in _lib.last_error()
        assert _call(lib, **{name: 4097}) == 1 and "misaligned" in _lib.last_error()
    for name in ("q_ts", "q_hs", "bs", "ts", "hs", "o_ts", "o_hs"):
        assert _call(lib, **{name: 100}) == 1 and "misaligned" in _lib.last_error()
    assert _call(lib, blocks=0) == 1
    assert _call(lib, ts=1 << 27) == 2 and "stride" in _lib.last_error()
    assert _call(lib, workspace=None) == 3 and "workspace" in _lib.last_error()
    assert _call(lib, workspace=4104) == 3
    need = lib.mi_shared_decode_workspace_bytes(4, 16, 8)
    assert _call(lib, ws_bytes=need - 1) == 3


def test_threads_have_workspaces_of_their_own(monkeypatch):
    # A call is two launches: another thread's, on the same stream, may come between.
    import threading

    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    plan = SharedDecodePlan(torch.empty(0), True, (), 64)

    def take(stream):
        return plan.workspace(torch.device("cpu"), stream)

    mine, others = take(1), []
    thread = threading.Thread(target=lambda: others.append((take(1), take(1))))
    thread.start()
    thread.join()
    assert mine.numel() == 64 and take(1) is mine and take(2) is not mine
    assert others[0][0] is others[0][1] is not mine
    assert others[0][0].data_ptr() != mine.data_ptr()
    capturing[0] = True  # a graph keeps its own
    assert take(1) is not mine
    capturing[0] = False
    assert take(1) is mine
