"""RMS norms of the query and key heads with the position rotation in the same pass (include/hy_rotary.h), as the
decoder (rotation first) and the DFlash draft (norm first) have them, on torch CUDA tensors. On the way into the paged
cache: paged.PagedKVCache.write_rotated.

The calls run asynchronously on torch's current stream of the rows' device and can be captured into a CUDA graph. They
have no backward pass and no forward-mode derivative: rows that require a gradient or carry a tangent are refused.
"""

from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd import forward_ad

from . import HY_ERR_INVALID_ARGUMENT, HyError, _check, load_library

_I, _L, _P = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
_ROW_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_raw_stream = torch._C._cuda_getCurrentRawStream


class _Rotation(ctypes.Structure):
    _fields_ = [("q_weight_dev", _P), ("k_weight_dev", _P), ("cos_dev", _P), ("sin_dev", _P), ("table_rows", _I),
                ("table_stride", _L), ("positions_dev", _P), ("eps", ctypes.c_float), ("rotate_first", _I)]


_pack = struct.Struct("@PPPPiqPfi").pack   # a hy_rotation as bytes: a third of the time that a ctypes structure takes
_LIB = None


def _library():
    global _LIB
    if _LIB is None:
        lib = load_library()
        lib.hy_norm_rotate.argtypes = [_P, _I, _I, _I, _I, _I, _I] + [_P, _L, _L] * 4 + [_P, _P]
        _LIB = lib
    return _LIB


def _refuse(message: str):
    raise HyError(HY_ERR_INVALID_ARGUMENT, message)


def refuse_tangents(*tensors: torch.Tensor) -> None:
    """Dual tensors (forward mode): these calls would drop their tangents. For where forward_ad._current_level >= 0."""
    if torch._C._is_fwd_grad_enabled() and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _refuse("a tensor carries a forward-mode tangent: these calls have no derivative")


def rotation(rows: int, dim: int, index: int, q_weight, k_weight, cos, sin, positions, eps, rotate_first) -> bytes:
    """A call's norms and angles, checked, as the bytes of a hy_rotation: weights [head_dim], cos and sin [table rows,
    head_dim] of one layout, all float32, and positions [rows] int32 (or None: row r takes the table's row r)."""
    f32 = torch.float32
    shape = cos.shape
    if torch.is_grad_enabled() and (q_weight.requires_grad or k_weight.requires_grad or cos.requires_grad or sin.requires_grad):
        _refuse("weights or angles that require a gradient: these calls have none")
    if forward_ad._current_level >= 0:
        refuse_tangents(q_weight, k_weight, cos, sin)
    if not (q_weight.dtype is f32 and k_weight.dtype is f32 and cos.dtype is f32 and sin.dtype is f32 and
            q_weight.get_device() == k_weight.get_device() == cos.get_device() == sin.get_device() == index):
        _refuse("weights, cos and sin must be float32 tensors on the rows' device")
    if q_weight.shape != (dim,) or k_weight.shape != (dim,) or len(shape) != 2 or shape[1] != dim or sin.shape != shape:
        _refuse(f"weights must be [{dim}], cos and sin [table rows, {dim}]")
    stride, one = cos.stride()
    if shape[0] <= 1:
        stride = dim
    elif sin.stride(0) != stride:
        _refuse("cos and sin must have one layout")
    if one != 1 or sin.stride(1) != 1 or q_weight.stride(0) != 1 or k_weight.stride(0) != 1:
        _refuse("weights and the rows of cos and sin must be contiguous")
    where = 0
    if positions is None:
        if shape[0] < rows:
            _refuse("without positions cos and sin must have a row for every row")
    else:
        if (positions.dtype is not torch.int32 or positions.shape != (rows,) or positions.get_device() != index or
                not positions.is_contiguous()):
            _refuse("positions must be a contiguous int32 tensor [rows] on the rows' device")
        where = positions.data_ptr()
    return _pack(q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(), shape[0], stride, where, eps,
                 rotate_first)


def norm_rotate(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                sin: torch.Tensor, positions: torch.Tensor | None = None, *, eps: float = 1e-5,
                rotate_first: bool = True, out: tuple[torch.Tensor, torch.Tensor] | None = None,
                status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The normed and rotated heads of rows q [rows, q heads, head_dim] and k [rows, kv heads, head_dim] (fp32 or bf16,
    any strides but the last; `out` may be (q, k) themselves):

        rotate_first:  y = turn(x);  y * w / sqrt(mean(y^2) + eps)
        otherwise:     turn(x * w / sqrt(mean(x^2) + eps))

    with turn(x) = x * cos + [-x[h:], x[:h]] * sin, h = head_dim / 2, and the cos and sin of the table's row
    positions[r] (row r without positions). A row whose position lies outside the table becomes NaN and sets bit 16 of
    `status` (an int32 tensor of one element, for instance PagedKVCache.status)."""
    kind, index, shape, kshape = q.dtype, q.get_device(), q.shape, k.shape
    dtype = _ROW_DTYPES.get(kind)
    if (dtype is None or index < 0 or len(shape) != 3 or len(kshape) != 3 or kshape[0] != shape[0] or
            kshape[2] != shape[2] or k.dtype is not kind or k.get_device() != index):
        _refuse("q [rows, q heads, head_dim] and k [rows, kv heads, head_dim] must be float32 or bfloat16 tensors of one "
                "CUDA device")
    if (q.requires_grad or k.requires_grad) and torch.is_grad_enabled():
        _refuse("rows that require a gradient: this call has none")
    if forward_ad._current_level >= 0:
        refuse_tangents(q, k, *(out or ()))
    rows, heads, dim = shape
    if out is None:
        a, b = q.new_empty(shape), k.new_empty(kshape)
        a0, a1, b0, b1 = heads * dim, dim, kshape[1] * dim, dim
    else:
        a, b = out
        for t, like in ((a, shape), (b, kshape)):
            if (t.dtype is not kind or t.shape != like or t.get_device() != index or t.stride(2) != 1 or
                    t.requires_grad and torch.is_grad_enabled()):
                _refuse("the outputs must be like q and k, with contiguous heads and without a gradient")
        a0, a1, _ = a.stride()
        b0, b1, _ = b.stride()
    q0, q1, q2 = q.stride()
    k0, k1, k2 = k.stride()
    if q2 != 1 or k2 != 1:
        _refuse("heads must be contiguous")
    if status is not None and (status.dtype is not torch.int32 or status.numel() < 1 or status.get_device() != index):
        _refuse("status must be an int32 tensor on the rows' device")
    turn = rotation(rows, dim, index, q_weight, k_weight, cos, sin, positions, eps, rotate_first)
    rc = (_LIB or _library()).hy_norm_rotate(turn, rows, heads, kshape[1], dim, dtype, index, q.data_ptr(), q0, q1, k.data_ptr(),
                                             k0, k1, a.data_ptr(), a0, a1, b.data_ptr(), b0, b1,
                                             None if status is None else status.data_ptr(), _raw_stream(index))
    if rc:
        _check(rc)
    return a, b
