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
    or below the smallest normal float32 (2^-126), has NaN log probabilities and
    entropy, its ``top_tokens`` still in order. Results that were not asked for are ``None``.
    """
    _lib.require_device(logits, tokens, temperatures, what="token log probabilities")
    code = _lib.DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float16, bfloat16 or float32")
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, vocab] with vocab > 0")
    rows, vocab = logits.shape
    device = logits.device
    if vocab > 2 ** 30:
        raise ValueError("vocab must be at most 2^30")
    if type(top) is not int or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be an integer between 0 and {MAX_TOP}, at most vocab")
    if (tokens is not None and tokens.device != device) or \
            (temperatures is not None and temperatures.device != device):
        raise ValueError("tokens and temperatures must be on the logits' device")
    given = 0
    logprobs = ent = top_tokens = top_logprobs = None
    logprobs_at = ent_at = top_tokens_at = top_logprobs_at = temperatures_at = None
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

    if tokens is not None:
        logprobs = torch.empty(tokens.shape, dtype=torch.float32, device=device)
        logprobs_at = logprobs.data_ptr()
    if entropy:
        ent = torch.empty(rows, dtype=torch.float32, device=device)
        ent_at = ent.data_ptr()
    if top:
        top_tokens = torch.empty((rows, top), dtype=torch.int64, device=device)
        top_logprobs = torch.empty((rows, top), dtype=torch.float32, device=device)
        top_tokens_at, top_logprobs_at = top_tokens.data_ptr(), top_logprobs.data_ptr()
    result = TokenLogprobs(logprobs, ent, top_tokens, top_logprobs)
    if rows == 0 or not (given or top or entropy):
        return result
    tokens_at = counters_at = workspace_at = None
    if tokens is not None:
        if tokens.dtype != torch.int64 or not tokens.is_contiguous():
            tokens = tokens.to(torch.int64).contiguous()
        tokens_at = tokens.data_ptr()
    if temperatures is not None:
        temperatures = temperatures.contiguous()
        temperatures_at = temperatures.data_ptr()
    lib = _lib.load()
    need = lib.mi_token_logprobs_workspace_bytes(rows, vocab, top, code)
    with _lib.on_device(device):
        stream = _lib.stream_handle(device)
        if need:
            counters, workspace = _scratch(device, stream, rows, need)
            counters_at, workspace_at = counters.data_ptr(), workspace.data_ptr()
        status = lib.mi_token_logprobs(
            logits.data_ptr(), logits.stride(0), rows, vocab, code, temperatures_at, tokens_at,
            given, given, logprobs_at, ent_at, top_tokens_at, top_logprobs_at, top, workspace_at,
            need, counters_at, stream)
    _lib.check(status, "mi_token_logprobs")
    return result
