"""Paged KV cache on the device: pages that hold K / V rows (quantised as they are written),
read back, and attended to by the new rows of several sequences at once (include/hy_paged.h).

The tensors are torch CUDA tensors. The calls run asynchronously on torch's current stream of the
cache's device and can be captured into a CUDA graph; a replay follows what the batch's arrays hold then.
A call that does not hold raises HyError; what only the device can see (page numbers, lengths, row
ranges) sets bits of ``PagedKVCache.status``, which ``check()`` reads.
"""

from __future__ import annotations

import ctypes

import torch

from . import HY_ERR_INVALID_ARGUMENT, HyError, _check, load_library

DTYPE_F32, DTYPE_BF16, DTYPE_E4M3, DTYPE_INT8 = range(4)
_CACHE_DTYPES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float8_e4m3fn: DTYPE_E4M3,
                 torch.int8: DTYPE_INT8}
_ROW_DTYPES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16}
_STATUS = {1: "a page number lies outside the cache", 2: "a kv_len does not fit its row of the block table",
           4: "q_start is not ascending or leaves the rows", 8: "a bounded wait inside a kernel gave up"}

_I, _L, _P = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
_INT_MAX = 2 ** 31 - 1
_raw_stream = torch._C._cuda_getCurrentRawStream   # the handle alone, without building a torch.cuda.Stream


class _Cache(ctypes.Structure):
    _fields_ = [(n, _I) for n in ("dtype", "num_pages", "num_kv_heads", "page_size", "head_dim", "device")] + [
        ("k_dev", _P), ("v_dev", _P), ("page_stride", _L), ("head_stride", _L), ("row_stride", _L),
        ("k_scale_dev", _P), ("v_scale_dev", _P), ("scale_page_stride", _L), ("scale_head_stride", _L),
        ("scale_row_stride", _L), ("status_dev", _P)]


class _Batch(ctypes.Structure):
    _fields_ = [("num_seqs", _I), ("max_rows", _I), ("table_width", _I), ("table_stride", _L), ("q_start_dev", _P),
                ("kv_len_dev", _P), ("block_table_dev", _P)]


def _library():
    lib = load_library()
    if lib.hy_paged_kv_write.argtypes is None:
        rows = [ctypes.POINTER(_Cache), ctypes.POINTER(_Batch), _I, _I, _P, _L, _L, _P, _L, _L, _P]
        lib.hy_paged_kv_read.argtypes = rows
        lib.hy_paged_attention.argtypes = [ctypes.POINTER(_Cache), ctypes.POINTER(_Batch), _I, _I, _I, _P, _L, _L, _P,
                                           _L, _L, ctypes.c_float, _I, _I, _I, _P, ctypes.c_size_t, _P]
        lib.hy_paged_attention_workspace.argtypes = [ctypes.POINTER(_Cache), ctypes.POINTER(_Batch), _I, _I, _I,
                                                     ctypes.POINTER(ctypes.c_size_t)]
        lib.hy_paged_kv_write.argtypes = rows
    return lib


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise HyError(HY_ERR_INVALID_ARGUMENT, message)


class PagedBatch:
    """The sequences of a call: q_start [n + 1] and kv_len [n] int32, block_table [n, width] int32 (rows may be
    strided), on the cache's device. Sequence s has the rows q_start[s] .. q_start[s + 1] - 1 of the row tensors,
    standing at the last positions of its kv_len[s]. max_rows: about the most rows of a sequence (attention is laid
    out for it, all sequences alike: tokens beside long chunks are faster in a call of their own). The arrays may be changed in place between calls, and between replays of a captured call."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor, max_rows: int):
        for t, name in ((q_start, "q_start"), (kv_len, "kv_len"), (block_table, "block_table")):
            _need(t.dtype == torch.int32, f"{name} must be int32")
        n = kv_len.shape[0] if kv_len.dim() == 1 else -1
        _need(n >= 0 and q_start.shape == (n + 1,) and block_table.dim() == 2 and block_table.shape[0] == n,
              "q_start [n + 1], kv_len [n] and block_table [n, width] must agree")
        _need(q_start.is_contiguous() and kv_len.is_contiguous() and
              (block_table.shape[1] <= 1 or block_table.stride(1) == 1),
              "q_start, kv_len and the rows of block_table must be contiguous")
        _need(q_start.device == kv_len.device == block_table.device, "the batch's arrays must be on one device")
        self.q_start, self.kv_len, self.block_table, self.max_rows = q_start, kv_len, block_table, max_rows
        self.num_seqs, self.index = n, kv_len.get_device()
        self._c = _Batch(n, max_rows, block_table.shape[1], block_table.stride(0), q_start.data_ptr(),
                         kv_len.data_ptr(), block_table.data_ptr())
        self._ref = ctypes.byref(self._c)


class PagedKVCache:
    """K and V pages [pages, kv heads, page rows, head_dim] (any strides but the last, the same for both) in fp32,
    bf16, float8_e4m3fn or int8; the 8-bit types with fp32 scales [pages, kv heads, page rows], value = code * scale."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.dtype == v.dtype,
              "k and v must be [pages, kv heads, page rows, head_dim] tensors of one shape, layout and type")
        _need(k.dtype in _CACHE_DTYPES, "the cache must be float32, bfloat16, float8_e4m3fn or int8")
        _need(k.stride(3) == 1, "head_dim must be the contiguous dimension")
        _need(k.is_cuda and k.device == v.device, "k and v must be on one CUDA device")
        strides = (0, 0, 0)
        if k_scale is not None or v_scale is not None:
            _need(k_scale is not None and v_scale is not None and k_scale.shape == v_scale.shape == k.shape[:3] and
                  k_scale.stride() == v_scale.stride() and k_scale.dtype == v_scale.dtype == torch.float32 and
                  k_scale.device == v_scale.device == k.device,
                  "the scales must be float32 tensors [pages, kv heads, page rows] of one layout beside k and v")
            strides = k_scale.stride()
        self._lib = _library()
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, k.device
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        pages, heads, rows, dim = k.shape
        self._heads, self._dim, self._index, self._workspace = heads, dim, k.device.index, {}
        self._c = _Cache(_CACHE_DTYPES[k.dtype], pages, heads, rows, dim, k.device.index, k.data_ptr(), v.data_ptr(),
                         *k.stride()[:3], None if k_scale is None else k_scale.data_ptr(),
                         None if v_scale is None else v_scale.data_ptr(), *strides, self.status.data_ptr())
        self._ref = ctypes.byref(self._c)

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype,
                 device="cuda") -> "PagedKVCache":
        """A cache of zeros."""
        _need(dtype in _CACHE_DTYPES, "the cache must be float32, bfloat16, float8_e4m3fn or int8")
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8 if dtype.itemsize == 1 else dtype, device=device).view(dtype)
                for _ in range(2))
        scales = [torch.zeros(shape[:3], device=device) for _ in range(2)] if dtype.itemsize == 1 else [None, None]
        return cls(k, v, *scales)

    def _rows(self, t: torch.Tensor, heads: int, name: str) -> int:
        """Checks a row tensor [rows, heads, head_dim]; its type."""
        dtype = _ROW_DTYPES.get(t.dtype)
        shape = t.shape
        if (dtype is None or len(shape) != 3 or shape[2] != self._dim or (heads and shape[1] != heads) or
                t.get_device() != self._index or t.stride(2) != 1):
            raise HyError(HY_ERR_INVALID_ARGUMENT, f"{name} must be a float32 or bfloat16 tensor [rows, heads, "
                          f"{self._dim}] on {self.device} with contiguous heads")
        if t.requires_grad and torch.is_grad_enabled():
            raise HyError(HY_ERR_INVALID_ARGUMENT, f"{name} requires a gradient: these calls have none")
        return dtype

    def _call(self, fn, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, dtype: int) -> None:
        if batch.index != self._index:
            raise HyError(HY_ERR_INVALID_ARGUMENT, "the batch must be on the cache's device")
        k0, k1, _ = k.stride()
        v0, v1, _ = v.stride()
        rc = fn(self._ref, batch._ref, k.shape[0], dtype, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1,
                _raw_stream(self._index))
        if rc:
            _check(rc)

    def _pair(self, k: torch.Tensor, v: torch.Tensor) -> int:
        dtype = self._rows(k, self._heads, "k")
        if self._rows(v, self._heads, "v") != dtype or v.shape != k.shape:
            raise HyError(HY_ERR_INVALID_ARGUMENT, "k and v must have one shape and type")
        return dtype

    def write(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor) -> None:
        """Writes rows k, v [rows, kv heads, head_dim] at their positions (hy_paged_kv_write)."""
        self._call(self._lib.hy_paged_kv_write, batch, k, v, self._pair(k, v))

    def read(self, batch: PagedBatch, rows: int, dtype: torch.dtype = torch.float32,
             out: tuple[torch.Tensor, torch.Tensor] | None = None):
        """The batch's positions as rows k, v [rows, kv heads, head_dim] (hy_paged_kv_read). Rows of `out` that
        belong to no sequence are left as they were; without `out` they hold anything."""
        if out is None:
            code = _ROW_DTYPES.get(dtype)
            _need(code is not None, "rows are read as float32 or bfloat16")
            k = torch.empty((rows, self._heads, self._dim), dtype=dtype, device=self.device)
            out = (k, torch.empty_like(k))
        else:
            _need(out[0].shape[0] == rows and out[0].dtype == dtype, "out must hold `rows` rows of `dtype`")
            code = self._pair(*out)
        self._call(self._lib.hy_paged_kv_read, batch, *out, code)
        return out

    def attention(self, batch: PagedBatch, q: torch.Tensor, scale: float, *, causal: bool = True, window: int = 0,
                  sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of rows q [rows, q heads, head_dim] over the cache (hy_paged_attention): the row at position p
        sees the positions j <= p, with a window those with p - j < window or j < sinks; all of them where causal is
        false. Rows of `out` that belong to no sequence are left as they were; without `out` they hold anything. The
        workspace comes from torch's allocator, one for each call."""
        dtype = self._rows(q, 0, "q")
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
        elif self._rows(out, q.shape[1], "out") != dtype or out.shape != q.shape:
            raise HyError(HY_ERR_INVALID_ARGUMENT, "q and out must have one shape and type")
        if batch.index != self._index:
            raise HyError(HY_ERR_INVALID_ARGUMENT, "the batch must be on the cache's device")
        rows, heads, _ = q.shape
        key = (rows, heads, dtype, batch.num_seqs, batch.max_rows)
        need = self._workspace.get(key)   # bytes; they depend on nothing else
        if need is None:
            size = ctypes.c_size_t()
            _check(self._lib.hy_paged_attention_workspace(self._ref, batch._ref, rows, heads, dtype,
                                                          ctypes.byref(size)))
            if len(self._workspace) > 256:
                self._workspace.clear()
            need = self._workspace[key] = size.value
        work = torch.empty(need, dtype=torch.uint8, device=self.device)
        q0, q1, _ = q.stride()
        o0, o1, _ = out.stride()
        window, sinks = max(min(window, _INT_MAX), -1), max(min(sinks, _INT_MAX), -1)   # (a C int would wrap)
        rc = self._lib.hy_paged_attention(self._ref, batch._ref, rows, heads, dtype, q.data_ptr(), q0, q1,
                                          out.data_ptr(), o0, o1, scale, causal, window, sinks, work.data_ptr(), need,
                                          _raw_stream(self._index))
        if rc:
            _check(rc)
        return out

    def with_runtime(self, runtime, layer: int, batch: PagedBatch, rows: int, write: bool) -> None:
        """Moves rows [0, rows) of a TextRuntime's layer into (write) or out of the batch's positions, on the
        runtime's stream, ordered after and before torch's current stream."""
        k, v, dtype, rs, hs = runtime.kv_device_rows(layer)
        _need(runtime.cfg.device == self._index and batch.index == self._index,
              "the runtime, the cache and the batch must be on one device")
        _need(self._heads == 8 and self._dim == 128, "the runtime has 8 KV heads of 128")
        _need(0 <= rows <= runtime.cfg.max_context, "rows exceed the runtime's KV capacity")
        ours, theirs = torch.cuda.current_stream(self.device), torch.cuda.ExternalStream(runtime.stream, self.device)
        theirs.wait_stream(ours)
        fn = self._lib.hy_paged_kv_write if write else self._lib.hy_paged_kv_read
        _check(fn(self._ref, batch._ref, rows, dtype, k, rs, hs, v, rs, hs, runtime.stream))
        ours.wait_stream(theirs)

    def check(self) -> None:
        """Raises what the calls since the last check met on the device (waits for them), and clears it."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise HyError(HY_ERR_INVALID_ARGUMENT, "; ".join(m for b, m in _STATUS.items() if bits & b))
