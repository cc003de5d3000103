"""RMS norms of the query and key heads with the position rotation in the same pass (include/hy_rotary.h), as the
decoder (rotation first) and the DFlash draft (norm first) have them, on torch CUDA tensors. On the way into the paged
cache: paged.PagedKVCache.write_rotated.

The calls run asynchronously on torch's current stream of the rows' device and can be captured into a CUDA graph. They
have no backward pass: rows that require a gradient are refused.
"""

from __future__ import annotations

import ctypes

import torch

from . import HY_ERR_INVALID_ARGUMENT, HyError, _check, load_library

_I, _L, _P = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
_ROW_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_raw_stream = torch._C._cuda_getCurrentRawStream


class _Rotation(ctypes.Structure):
    _fields_ = [("q_weight_dev", _P), ("k_weight_dev", _P), ("cos_dev", _P), ("sin_dev", _P), ("table_rows", _I),
                ("table_stride", _L), ("positions_dev", _P), ("eps", ctypes.c_float), ("rotate_first", _I)]


def _library():
    lib = load_library()
    if lib.hy_norm_rotate.argtypes is None:
        lib.hy_norm_rotate.argtypes = [ctypes.POINTER(_Rotation), _I, _I, _I, _I, _I, _I] + [_P, _L, _L] * 4 + [_P, _P]
    return lib


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise HyError(HY_ERR_INVALID_ARGUMENT, message)


class Rotation:
    """Checked norms and angles of a call: weights [head_dim], cos and sin [table rows, head_dim] of one layout, all
    float32, and positions [rows] int32 (or None: row r takes the table's row r)."""

    __slots__ = ("c", "ref")

    def __init__(self, rows: int, dim: int, index: int, q_weight, k_weight, cos, sin, positions, eps, rotate_first):
        for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight"), (cos, "cos"), (sin, "sin")):
            if t.dtype != torch.float32 or t.get_device() != index or t.shape[-1] != dim or t.stride(-1) != 1:
                raise HyError(HY_ERR_INVALID_ARGUMENT, f"{name} must be a float32 tensor [..., {dim}] with contiguous "
                              "rows on the rows' device")
        if (q_weight.dim() != 1 or k_weight.dim() != 1 or cos.dim() != 2 or cos.shape != sin.shape or
                (cos.shape[0] > 1 and cos.stride(0) != sin.stride(0))):
            raise HyError(HY_ERR_INVALID_ARGUMENT, "weights are [head_dim], cos and sin [table rows, head_dim] of one layout")
        where = None
        if positions is not None:
            if (positions.dtype != torch.int32 or positions.shape != (rows,) or positions.get_device() != index or
                    not positions.is_contiguous()):
                raise HyError(HY_ERR_INVALID_ARGUMENT, "positions must be a contiguous int32 tensor [rows] on the rows' device")
            where = positions.data_ptr()
        else:
            _need(cos.shape[0] >= rows, "without positions cos and sin must have a row for every row")
        self.c = _Rotation(q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                           cos.stride(0) if cos.shape[0] > 1 else dim, where, eps, rotate_first)
        self.ref = ctypes.byref(self.c)


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
    dtype, index = _ROW_DTYPES.get(q.dtype), q.get_device()
    outs = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)) if out is None else out
    if (dtype is None or index < 0 or q.dim() != 3 or k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or
            outs[0].shape != q.shape or outs[1].shape != k.shape):
        raise HyError(HY_ERR_INVALID_ARGUMENT, "q [rows, q heads, head_dim] and k [rows, kv heads, head_dim] must be "
                      "float32 or bfloat16 CUDA tensors, the outputs like them")
    for t in (q, k, *outs):
        if t.dtype != q.dtype or t.get_device() != index or t.stride(2) != 1:
            raise HyError(HY_ERR_INVALID_ARGUMENT, "q, k and the outputs must have one type and device and contiguous heads")
        if t.requires_grad and torch.is_grad_enabled():
            raise HyError(HY_ERR_INVALID_ARGUMENT, "rows that require a gradient: this call has none")
    if status is not None:
        _need(status.dtype == torch.int32 and status.numel() >= 1 and status.get_device() == index,
              "status must be an int32 tensor on the rows' device")
    rows, heads, dim = q.shape
    turn = Rotation(rows, dim, index, q_weight, k_weight, cos, sin, positions, eps, rotate_first)
    q0, q1, _ = q.stride()
    k0, k1, _ = k.stride()
    a0, a1, _ = outs[0].stride()
    b0, b1, _ = outs[1].stride()
    rc = _library().hy_norm_rotate(turn.ref, rows, heads, k.shape[1], dim, dtype, index, q.data_ptr(), q0, q1,
                                   k.data_ptr(), k0, k1, outs[0].data_ptr(), a0, a1, outs[1].data_ptr(), b0, b1,
                                   None if status is None else status.data_ptr(), _raw_stream(index))
    if rc:
        _check(rc)
    return outs
