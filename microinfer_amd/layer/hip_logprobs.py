"""Log probabilities of tokens through the HIP library.

``token_logprobs`` gives, for each row of logits, the log probabilities of
given tokens (those drawn, or a prompt's next tokens), the best alternatives
with theirs and the entropy, in one pass over the logits: what ranks the
continuations of a prompt, proposes a beam's next tokens and answers a
request for logprobs. The order among alternatives is ``greedy_argmax``'s.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from microinfer_amd import _lib

_FLOAT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
MAX_TOP = 32

# Scratch of a stream's launches: arrival counters (zero-filled once, left zero
# by every launch) and the parts' results. Captured launches get their own
# (_scratch). Memory outgrown by a larger call goes back to torch's allocator,
# which reuses it on that stream behind the launches that still use it.
_scratches: dict[tuple[int, int], tuple[torch.Tensor, torch.Tensor]] = {}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor | None  # float32, of the tokens' shape
    entropy: torch.Tensor | None  # float32 [rows]
    top_tokens: torch.Tensor | None  # int64 [rows, top], best first
    top_logprobs: torch.Tensor | None  # float32 [rows, top]


def _scratch(device: torch.device, stream: int, rows: int, nbytes: int):
    """Counters for ``rows`` rows and ``nbytes`` of workspace."""
    if torch.cuda.is_current_stream_capturing():
        # Part of the graph, so graphs replayed side by side do not share them.
        return (torch.zeros(rows, dtype=torch.int32, device=device),
                torch.empty(nbytes, dtype=torch.uint8, device=device))
    key = (device.index, stream)
    have = _scratches.get(key)
    if have is None or have[0].numel() < rows or have[1].numel() < nbytes:
        if have is not None:
            rows, nbytes = max(rows, have[0].numel()), max(nbytes, have[1].numel())
        have = (torch.zeros(max(rows, 1024), dtype=torch.int32, device=device),
                torch.empty(max(nbytes, 1 << 18), dtype=torch.uint8, device=device))
        _scratches[key] = have
    return have


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0,
                   temperatures: torch.Tensor | None = None,
                   entropy: bool = False) -> TokenLogprobs:
    """``log_softmax(logits / temperatures)`` at ``tokens``, its ``top`` largest
    entries and the entropy of each row, in float32.

    ``logits`` is float16, bfloat16 or float32 ``[rows, vocab]`` with
    contiguous rows (any row stride). ``tokens`` is int64 or int32 ``[rows]`` or
    ``[rows, n]``; one outside the vocabulary gives NaN. ``top`` is at most 32:
    the largest logits, NaN above every number and the lowest index first
    among equals. ``temperatures`` is float32 ``[rows]``. A masked logit
    (``-inf``) has probability 0 and log probability ``-inf``; a row that holds
    NaN, ``+inf`` or nothing above ``-inf``, or whose temperature is not finite
    and positive, has NaN log probabilities and entropy, its ``top_tokens``
    still in order. Results that were not asked for are ``None``.
    """
    _lib.require_device(logits, tokens, temperatures, what="token log probabilities")
    if logits.dtype not in _FLOAT_DTYPES:
        raise ValueError("logits must be float16, bfloat16 or float32")
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, vocab] with vocab > 0")
    rows, vocab = logits.shape
    device = logits.device
    if vocab > 2 ** 30:
        raise ValueError("vocab must be at most 2^30")
    if type(top) is not int or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be an integer between 0 and {MAX_TOP}, at most vocab")
    if any(t is not None and t.device != device for t in (tokens, temperatures)):
        raise ValueError("tokens and temperatures must be on the logits' device")
    given = 0
    if tokens is not None:
        if tokens.dtype not in (torch.int64, torch.int32) or tokens.ndim not in (1, 2) \
                or tokens.shape[0] != rows:
            raise ValueError("tokens must be int64 or int32 [rows] or [rows, n]")
        given = 1 if tokens.ndim == 1 else tokens.shape[1]
        if given > 65536:
            raise ValueError("at most 65536 tokens per row")
    if temperatures is not None and (temperatures.dtype != torch.float32
                                     or temperatures.shape != (rows,)):
        raise ValueError("temperatures must be float32 [rows]")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()

    result = TokenLogprobs(
        None if tokens is None else torch.empty(tokens.shape, dtype=torch.float32, device=device),
        torch.empty(rows, dtype=torch.float32, device=device) if entropy else None,
        torch.empty((rows, top), dtype=torch.int64, device=device) if top else None,
        torch.empty((rows, top), dtype=torch.float32, device=device) if top else None)
    if rows == 0 or not (given or top or entropy):
        return result
    if tokens is not None and (tokens.dtype != torch.int64 or not tokens.is_contiguous()):
        tokens = tokens.to(torch.int64).contiguous()
    if temperatures is not None:
        temperatures = temperatures.contiguous()
    lib, code = _lib.load(), _lib.DTYPE_CODES[logits.dtype]
    need = lib.mi_token_logprobs_workspace_bytes(rows, vocab, top, code)
    with _lib.on_device(device):
        stream = _lib.stream_handle(device)
        counters = workspace = None
        if need:
            counters, workspace = _scratch(device, stream, rows, need)
        status = lib.mi_token_logprobs(
            logits.data_ptr(), logits.stride(0), rows, vocab, code,
            *[None if t is None else t.data_ptr() for t in (temperatures, tokens)], given, given,
            *[None if t is None else t.data_ptr() for t in result], top,
            None if workspace is None else workspace.data_ptr(), need,
            None if counters is None else counters.data_ptr(), stream)
    _lib.check(status, "mi_token_logprobs")
    return result
