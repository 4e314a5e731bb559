"""Paged decode of sequences that share their first pages, on the HIP library.

``hip_shared_decode`` is ``hip_paged_decode`` for continuations of common
prompts (forks of a request, a system prompt): the pages that a group of
sequences shares are read once for every 64 query rows of a KV head (64 / G
sequences of G query heads per KV head) instead of once for each sequence.
Groups are consecutive sequences of the batch;
``shared_decode_plan`` lays out a step's work on the device from the lengths
and groups, and every layer of the step uses that plan.

16-bit caches with head_dim 128, up to 16 query heads per KV head and blocks
of at least 16 have a kernel of their own; the other types, heads and block
sizes that ``hip_paged_decode`` takes run on it, with the same result. Block
tables of more than 2^30 positions are refused.
"""

from __future__ import annotations

import threading
from dataclasses import dataclass, field

import torch

from microinfer_amd import _lib
from microinfer_amd.layer.hip_paged_attention import (_check_caches, _index32,
                                                      _inner_contiguous, _is_pow2, decode_plan,
                                                      hip_paged_decode)

MAX_SEQS = 4096
MAX_ROWS = 64  # query rows of a KV head that meet a shared page at once


@dataclass(frozen=True)
class SharedDecodePlan:
    """One step's work (``shared_decode_plan``), for calls of its sizes."""

    buffer: torch.Tensor
    shared: bool  # False: a ``decode_plan`` for ``hip_paged_decode``
    sizes: tuple  # sequences, Hq, Hkv, head_dim, dtype, block size, table width
    workspace_bytes: int = 0  # of a call with it
    # By thread and stream: its calls run one after the other. A call is two
    # launches, between which another thread's may come.
    _workspaces: dict[tuple[int, int], torch.Tensor] = field(default_factory=dict, repr=False,
                                                             compare=False)

    def workspace(self, device: torch.device, stream: int) -> torch.Tensor:
        """Memory of a call on ``stream``, the current one; a captured call's own,
        as its graph keeps it."""
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(self.workspace_bytes, dtype=torch.uint8, device=device)
        key = threading.get_ident(), stream
        have = self._workspaces.get(key)
        if have is None:
            have = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=device)
            self._workspaces[key] = have
        return have


def shared_order(tables) -> list[int]:
    """An order of ``tables`` (host lists of block ids) that puts those with a
    common beginning next to each other, in the order of their first."""
    firsts: dict = {}
    for i, table in enumerate(tables):
        firsts.setdefault(table[0] if table else None, []).append(i)
    order = []
    for same in firsts.values():
        if len(same) > 2:
            first = tables[same[0]]
            rank = {}
            for i in same:  # by what they share with the first, then by what follows
                table = tables[i]
                n = _common_blocks(first, table, min(len(first), len(table)))
                rank[i] = (-n, table[n] if n < len(table) else -1)
            same.sort(key=rank.__getitem__)
        order += same
    return order


def shared_groups(tables, contexts, block_size: int) -> tuple[list[int], list[int]]:
    """Groups of neighbours in ``tables`` that share their first whole blocks,
    for ``shared_decode_plan``: group starts (one more than groups) and the
    shared blocks of each. A sequence joins the group before it unless that
    would halve what the group shares, or what the sequence shares with its
    other neighbour, so order the tables first (``shared_order``)."""
    n = len(tables)
    whole = [min(context // block_size, len(table)) for table, context in zip(tables, contexts)]
    common = [0] * (n + 1)  # of each sequence and the one before it
    for i in range(1, n):
        common[i] = _common_blocks(tables[i - 1], tables[i], min(whole[i - 1], whole[i]))
    starts: list[int] = []
    shared: list = []
    for i in range(n):
        if starts:
            alone = shared[-1] is None
            both = common[i] if alone else min(common[i], shared[-1])
            if both and 2 * both >= max(common[i + 1], 0 if alone else shared[-1]):
                shared[-1] = both
                continue
        starts.append(i)
        shared.append(None)
    return starts + [n], [blocks or 0 for blocks in shared]


def _common_blocks(a: list[int], b: list[int], most: int) -> int:
    """Length of the common beginning of two tables, at most ``most``."""
    low, high = 0, most
    if most and a[0] != b[0]:
        return 0
    while low < high:  # the slices halve, so at most 2 * most entries are compared
        mid = (low + high + 1) // 2
        if a[low:mid] == b[low:mid]:
            low = mid
        else:
            high = mid - 1
    return low


def least_shared_positions(num_seqs: int, num_kv_heads: int,
                           num_q_heads: int | None = None) -> int:
    """Positions that the groups of a decode step must share, counted as often
    as their reads become fewer (``prefer_shared_decode``), to be better read
    together. ``num_q_heads``: by default two for each KV head.

    What has to be gained is the launch that the fused QKV decode saves, the
    plan, the host's time and, with each sequence and query head, the join. Whole
    steps of a 28-layer model (head_dim 128, bf16, block 16, one group with 100
    tokens of each sequence's own, from graphs), us without and with the groups,
    and what finding them takes the host:

        heads  sequences  shared tokens on both sides of the rule
        16/8    4          5136: 1114, 1152 + 18    20496: 1679, 1537 + 31
        16/8    8          2064: 1087, 1134 + 22     8208: 1499, 1291 + 37
        16/8   16          1184: 1134, 1165 + 38     4688: 1579, 1302 + 57
        16/8   64           672: 1350, 1384 + 113    2656: 1962, 1547 + 166
        32/8   16          2352: 1337, 1315 + 45     4688: 1663, 1407 + 59
        32/8   64          1328: 1663, 1635 + 138    2656: 2082, 1714 + 173
        64/8   64          1328: 1909, 1944 + 136    5296: 3102, 2297 + 232
        64/4    4                                   20496: 1785, 1614 + 32
        64/4   64          5296: 2502, 2283 + 233   10576: 3523, 2781 + 327
        32/2   64          5296: 1971, 1775 + 236   10576: 2687, 2103 + 327
        16/16  16           592: 1102, 1206 + 32     2352: 1445, 1272 + 45
    """
    if num_q_heads is None:
        num_q_heads = 2 * num_kv_heads
    base = min(1 << 14, (1 << 17) // num_kv_heads)  # few KV heads leave a plain step less parallel
    return base + (5120 + 192 * num_q_heads) * num_seqs // num_kv_heads


def prefer_shared_decode(starts, shared, block_size: int, num_kv_heads: int,
                         num_q_heads: int | None = None) -> bool:
    """Whether a decode step with the groups of ``shared_groups`` is better
    done with them. ``num_q_heads``: as for ``least_shared_positions``.

    A group's shared blocks are read once for every 64 query rows of a KV head,
    instead of by every sequence, of which the second finds them in the caches
    (16 pairs with 8192 shared tokens: 3606 us a step without and 3760 with)."""
    if num_q_heads is None:
        num_q_heads = 2 * num_kv_heads
    per_tile = max(MAX_ROWS // (num_q_heads // num_kv_heads), 1)
    counted = 0
    for g, blocks in enumerate(shared):
        members = starts[g + 1] - starts[g]
        counted += max(members - 1 - -(-members // per_tile), 0) * blocks
    return counted > 0 and \
        counted * block_size >= least_shared_positions(starts[-1], num_kv_heads, num_q_heads)


def supported_shared_decode(num_q_heads: int, num_kv_heads: int, head_dim: int,
                            dtype: torch.dtype, block_size: int, num_seqs: int) -> bool:
    """Whether sequences of this shape read shared pages together."""
    return (dtype in (torch.float16, torch.bfloat16) and head_dim == 128
            and num_q_heads <= 16 * num_kv_heads and block_size >= 16
            and 0 < num_seqs <= MAX_SEQS)


def shared_decode_plan(context_lens: torch.Tensor, group_starts: torch.Tensor,
                       shared_blocks: torch.Tensor, *, num_q_heads: int, num_kv_heads: int,
                       head_dim: int, dtype: torch.dtype, block_size: int,
                       block_table_width: int) -> SharedDecodePlan:
    """The plan of one decode step, from device tensors alone (capture-safe).

    Group g is the sequences ``group_starts[g] : group_starts[g + 1]``; the
    first ``shared_blocks[g]`` columns of their block tables are equal. Shared
    blocks that are not whole in every context of the group are read by each
    sequence for itself, as are those of a group of one and of sequences
    outside every group.
    """
    _lib.require_device(context_lens, group_starts, shared_blocks, what="shared_decode_plan")
    if num_kv_heads <= 0 or num_q_heads <= 0 or num_q_heads % num_kv_heads:
        raise ValueError("Hq must be divisible by Hkv")
    if not _is_pow2(block_size):
        raise ValueError("paged kernels require a power-of-two block size")
    if context_lens.ndim != 1 or group_starts.ndim != 1 or shared_blocks.ndim != 1:
        raise ValueError("context_lens, group_starts and shared_blocks must be 1-D")
    groups = shared_blocks.numel()
    if group_starts.numel() != groups + 1 and (groups or group_starts.numel()):
        raise ValueError("group_starts must have one entry more than shared_blocks")
    if groups > MAX_SEQS:
        raise ValueError(f"at most {MAX_SEQS} groups")
    if any(t.device != context_lens.device for t in (group_starts, shared_blocks)):
        raise ValueError("context_lens, group_starts and shared_blocks must share a device")
    num_seqs = context_lens.numel()
    sizes = (num_seqs, num_q_heads, num_kv_heads, head_dim, dtype, block_size,
             block_table_width)
    if not supported_shared_decode(num_q_heads, num_kv_heads, head_dim, dtype, block_size,
                                   num_seqs):
        heads = None
        if num_q_heads > 16 * num_kv_heads or head_dim != 128 or dtype == torch.float32 \
                or block_size < 16:
            heads = (num_q_heads, head_dim, dtype)
        return SharedDecodePlan(
            decode_plan(context_lens, num_kv_heads=num_kv_heads, block_size=block_size,
                        block_table_width=block_table_width, heads=heads), False, sizes)
    context_lens, group_starts, shared_blocks = (
        _index32(t) for t in (context_lens, group_starts, shared_blocks))
    lib = _lib.load()
    with _lib.on_device(context_lens.device):
        nbytes = lib.mi_shared_decode_plan_bytes(num_seqs, num_q_heads, num_kv_heads)
        buffer = torch.empty(nbytes, dtype=torch.uint8, device=context_lens.device)
        status = lib.mi_shared_decode_plan(
            context_lens.data_ptr(), num_seqs, group_starts.data_ptr(), shared_blocks.data_ptr(),
            groups, num_q_heads, num_kv_heads, head_dim, block_size, block_table_width,
            _lib.dtype_code(dtype), buffer.data_ptr(), nbytes,
            _lib.stream_handle(context_lens.device))
    _lib.check(status, "mi_shared_decode_plan")
    return SharedDecodePlan(
        buffer, True, sizes,
        lib.mi_shared_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads))


def hip_shared_decode(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                      block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                      plan: SharedDecodePlan, scale: float | None = None) -> torch.Tensor:
    """Decode one query row per sequence; ``hip_paged_decode``'s arguments and
    result, with ``plan`` from ``shared_decode_plan`` for these lengths.

    The caches hold the step's K/V rows already. Without a plan there are no
    groups to share pages in: call ``hip_paged_decode``.
    """
    shape, dtype, device = query.shape, query.dtype, query.device
    if len(shape) != 3:
        raise ValueError("query must have shape [requests, Hq, D]")
    if key_cache.ndim != 4:
        raise ValueError("key_cache must have shape [blocks, B, Hkv, D]")
    num_seqs, num_q_heads, head_dim = shape
    num_blocks, block_size, num_kv_heads, kv_dim = key_cache.shape
    if kv_dim != head_dim:
        raise ValueError("query and cache head dimensions differ")
    if device != key_cache.device or dtype != key_cache.dtype:
        raise ValueError("query and cache must share device/dtype")
    if block_tables.ndim != 2 or block_tables.shape[0] != num_seqs:
        raise ValueError("block_tables must have one row per request")
    if context_lens.numel() != num_seqs:
        raise ValueError("context_lens must have one entry per request")
    width = block_tables.shape[1]
    sizes = (num_seqs, num_q_heads, num_kv_heads, head_dim, dtype, block_size, width)
    if not isinstance(plan, SharedDecodePlan) or plan.sizes != sizes:
        raise ValueError("plan must come from shared_decode_plan() for this call's sizes")
    _lib.require_device(query, block_tables, context_lens, what="hip_shared_decode")
    buffer = plan.buffer
    if buffer.device != device or block_tables.device != device:
        raise ValueError("plan and block_tables must be on the query's device")
    key_cache, value_cache = _check_caches(key_cache, value_cache)
    query = _inner_contiguous(query)
    if not plan.shared:
        return hip_paged_decode(query, key_cache, value_cache, block_tables, context_lens,
                                scale=scale, plan=buffer if num_seqs else None)
    block_tables = _index32(block_tables)
    if scale is None:
        scale = head_dim ** -0.5
    q_token_stride, q_head_stride, _ = query.stride()
    if (query.data_ptr() | 2 * q_token_stride | 2 * q_head_stride) & 15:
        query = query.clone(memory_format=torch.contiguous_format)  # rows of whole vectors
        q_token_stride, q_head_stride, _ = query.stride()
    lib = _lib.load()
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    with _lib.on_device(device):
        stream = _lib.stream_handle(device)
        workspace = plan.workspace(device, stream)
        block_stride, token_stride, head_stride, _ = key_cache.stride()
        status = lib.mi_shared_decode(
            query.data_ptr(), q_token_stride, q_head_stride, key_cache.data_ptr(),
            value_cache.data_ptr(), block_stride, token_stride, head_stride,
            block_tables.data_ptr(), width, width, buffer.data_ptr(), buffer.numel(),
            out.data_ptr(), num_q_heads * head_dim, head_dim, workspace.data_ptr(),
            plan.workspace_bytes, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
            num_blocks, float(scale), _lib.DTYPE_CODES[dtype], stream)
    _lib.check(status, "mi_shared_decode")
    return out
