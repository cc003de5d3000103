"""Log probabilities of given tokens, entropy and top alternatives of rows of logits (include/hy_logprobs.h), on torch
CUDA tensors. Behind a runtime's own LM head: TextRuntime.lm_head_logprobs.

The calls run asynchronously on torch's current stream of the logits' device and can be captured into a CUDA graph.
They have no backward pass: logits that require a gradient are refused.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import HY_ERR_INVALID_ARGUMENT, HyError, _check, load_library

_I, _L, _P = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
_ROW_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_raw_stream = torch._C._cuda_getCurrentRawStream


class TokenLogprobs(NamedTuple):
    """logprob: as the tokens, float32; entropy [rows] float32; top_ids [rows, top] int32 and top_logprobs [rows, top]
    float32 (None where top is 0)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


def _library():
    lib = load_library()
    if lib.hy_token_logprobs.argtypes is None:
        lib.hy_token_logprobs.argtypes = [_P, _I, _I, _L, _I, _I, _P, _I, _I, _P, _P, _P, _P, _P]
    return lib


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """log softmax(logits) at the given tokens, the entropy of every row and its `top` (0 to 64) most likely tokens.

    logits [rows, vocab] float32 or bfloat16 (rows may be strided), tokens [rows] or [rows, n] int32. Equal logits are
    ordered by the lower token. Logits of -infinity (masked tokens) have probability 0 and are no alternatives (-1 and
    -infinity where too few are left). A token outside the vocabulary (padding) gives NaN, as does all of a row that
    holds a NaN, +infinity or nothing above -infinity (its top_ids are -1)."""
    dtype, index = _ROW_DTYPES.get(logits.dtype), logits.get_device()
    if dtype is None or index < 0 or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise HyError(HY_ERR_INVALID_ARGUMENT, "logits must be a float32 or bfloat16 CUDA tensor [rows, vocab] with contiguous rows")
    if logits.requires_grad and torch.is_grad_enabled():
        raise HyError(HY_ERR_INVALID_ARGUMENT, "logits require a gradient: this call has none")
    rows, vocab = logits.shape
    if (tokens.dtype != torch.int32 or tokens.get_device() != index or tokens.dim() not in (1, 2) or
            tokens.shape[0] != rows or not tokens.is_contiguous()):
        raise HyError(HY_ERR_INVALID_ARGUMENT, "tokens must be a contiguous int32 tensor [rows] or [rows, n] beside the logits")
    if not 0 <= top <= 64:
        raise HyError(HY_ERR_INVALID_ARGUMENT, "top must be in 0..64 and at most vocab")
    per_row = 1 if tokens.dim() == 1 else tokens.shape[1]
    # One allocation: log probabilities, entropies, top ids, their log probabilities.
    n = rows * per_row
    held = torch.empty(n + rows + 2 * rows * top, dtype=torch.float32, device=logits.device)
    lp, entropy = held[:n].view(tokens.shape), held[n:n + rows]
    at = held.data_ptr()
    ids = alternatives = None
    if top:
        ids = held[n + rows:n + rows + rows * top].view(torch.int32).view(rows, top)
        alternatives = held[n + rows + rows * top:].view(rows, top)
    rc = _library().hy_token_logprobs(logits.data_ptr(), rows, vocab, logits.stride(0), dtype, index, tokens.data_ptr(),
                                      per_row, top, at, at + 4 * n, at + 4 * (n + rows), at + 4 * (n + rows + rows * top),
                                      _raw_stream(index))
    if rc:
        _check(rc)
    return TokenLogprobs(lp, entropy, ids, alternatives)
