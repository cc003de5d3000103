"""Log probabilities of given tokens, entropy and top alternatives of rows of logits (include/hy_logprobs.h), on torch
CUDA tensors. Behind a runtime's own LM head: TextRuntime.lm_head_logprobs.

The calls run asynchronously on torch's current stream of the logits' device and can be captured into a CUDA graph.
They have no backward pass and no forward-mode derivative: logits that require a gradient or carry a tangent are refused.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import HY_ERR_INVALID_ARGUMENT, HyError, _check, load_library
from .rotary import refuse_tangents

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


_LIB = None


def _library():
    global _LIB
    if _LIB is None:
        lib = load_library()
        lib.hy_token_logprobs.argtypes = [_P, _I, _I, _L, _I, _I, _P, _I, _I, _P, _P, _P, _P, _P]
        _LIB = lib
    return _LIB


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """log softmax(logits) at the given tokens, the entropy of every row and its `top` (0 to 64) most likely tokens.

    logits [rows, vocab] float32 or bfloat16 (rows may be strided), tokens [rows] or [rows, n] int32. Equal logits are
    ordered by the lower token. Logits of -infinity (masked tokens) have probability 0 and are no alternatives (-1 and
    -infinity where too few are left). A token outside the vocabulary (padding) gives NaN, as does all of a row that
    holds a NaN, +infinity or nothing above -infinity (its top_ids are -1)."""
    dtype, index, shape = _ROW_DTYPES.get(logits.dtype), logits.get_device(), logits.shape
    if dtype is None or index < 0 or len(shape) != 2:
        raise HyError(HY_ERR_INVALID_ARGUMENT, "logits must be a float32 or bfloat16 CUDA tensor [rows, vocab]")
    rows, vocab = shape
    stride, one = logits.stride()
    if one != 1 and vocab > 1:
        raise HyError(HY_ERR_INVALID_ARGUMENT, "the rows of logits must be contiguous")
    if logits.requires_grad and torch.is_grad_enabled():
        raise HyError(HY_ERR_INVALID_ARGUMENT, "logits require a gradient: this call has none")
    if forward_ad._current_level >= 0:
        refuse_tangents(logits)
    tshape = tokens.shape
    if (tokens.dtype is not torch.int32 or tokens.get_device() != index or len(tshape) not in (1, 2) or tshape[0] != rows or
            not tokens.is_contiguous()):
        raise HyError(HY_ERR_INVALID_ARGUMENT, "tokens must be a contiguous int32 tensor [rows] or [rows, n] beside the logits")
    if not 0 <= top <= 64:
        raise HyError(HY_ERR_INVALID_ARGUMENT, "top must be in 0..64 and at most vocab")
    per_row = 1 if len(tshape) == 1 else tshape[1]
    if rows >= 2 ** 31 or vocab >= 2 ** 31 or per_row >= 2 ** 31:   # (a C int would wrap)
        raise HyError(HY_ERR_INVALID_ARGUMENT, "rows, vocab and the tokens of a row must be below 2^31")
    lp, entropy = logits.new_empty(tshape, dtype=torch.float32), logits.new_empty(rows, dtype=torch.float32)
    ids = alternatives = at = ids_at = None
    if top:
        ids, alternatives = tokens.new_empty((rows, top)), logits.new_empty((rows, top), dtype=torch.float32)
        ids_at, at = ids.data_ptr(), alternatives.data_ptr()
    rc = (_LIB or _library()).hy_token_logprobs(logits.data_ptr(), rows, vocab, stride, dtype, index, tokens.data_ptr(), per_row,
                                                top, lp.data_ptr(), entropy.data_ptr(), ids_at, at, _raw_stream(index))
    if rc:
        _check(rc)
    return TokenLogprobs(lp, entropy, ids, alternatives)
