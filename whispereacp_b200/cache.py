"""The paged key/value cache's host interface, over the C ABI of include/wsp_cache.h.

  appendLinear's cache write, attention over a Cache
                 Lib/WhisperEACP/Net/Net.h:110-171

``PagedCache`` holds two pools [pages, heads, page_rows, head_width] of torch
tensors on one device (and, for 8-bit storage, their scale bytes), and a
``CacheBatch`` says which rows of which pages a call's sequences hold.  What
the tensors of a batch contain is read when the work runs, so one batch serves
every step whose tensors are updated in place, in a captured CUDA graph too.

Calls queue on torch's current stream of the cache's device, or on ``stream``,
and return without waiting.  They have no gradients: in grad mode tensors that
require one are refused.
"""
from __future__ import annotations

import ctypes
import math
import threading

from ._native import (CCacheBatch, CCacheMemory, CCacheRows, CCacheShape, WSP_BFLOAT16, WSP_CACHE_BFLOAT16,
                      WSP_CACHE_E4M3, WSP_CACHE_FLOAT16, WSP_CACHE_INT8, WSP_FLOAT16, WSP_FLOAT32, ModelError, check,
                      library)

__all__ = ["PagedCache", "CacheBatch", "CACHE_STORAGE"]

CACHE_STORAGE = {"float16": WSP_CACHE_FLOAT16, "bfloat16": WSP_CACHE_BFLOAT16, "float8_e4m3fn": WSP_CACHE_E4M3,
                 "int8": WSP_CACHE_INT8}
_ROW_TYPES = {"float32": WSP_FLOAT32, "float16": WSP_FLOAT16, "bfloat16": WSP_BFLOAT16}
_codes: dict = {}  # torch dtype -> its code, filled as dtypes are met
_workspaces = threading.local()  # (device, stream) -> this thread's workspace there


def _torch():
    import torch
    return torch


def _name(dtype) -> str:
    return str(dtype).replace("torch.", "")


def _row_type(dtype) -> int:
    code = _ROW_TYPES.get(_name(dtype))
    if code is None:
        raise ValueError(f"rows are float32, float16 or bfloat16, not {_name(dtype)}")
    _codes[dtype] = code
    return code


def _refuse_gradient(name: str) -> None:
    """In grad mode a tensor that requires a gradient would silently get none."""
    if _torch().is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and the cache's operators have none: detach it, or call them "
                         "under torch.no_grad()")


class CacheBatch:
    """The sequences of a call (wsp_cache_batch).

    page_table  int32 [sequences, columns]: the pages of each, in order
    lengths     int32 [sequences]: rows held, the new ones counted
    starts      int32 [sequences + 1]: sequence s's new rows are rows
                starts[s] .. starts[s + 1] - 1 of a call's arrays, and its
                last ones (row i of n at position lengths[s] - n + i)
    max_rows    a bound of a sequence's new rows (None: taken from starts,
                which waits for the device); it chooses kernels only
    """

    def __init__(self, page_table, lengths, starts, max_rows: int | None = None):
        torch = _torch()
        for name, t, dim in (("page_table", page_table, 2), ("lengths", lengths, 1), ("starts", starts, 1)):
            if not t.is_cuda or t.dtype != torch.int32 or t.dim() != dim:
                raise ValueError(f"{name} must be a {dim}-dimensional int32 tensor on a CUDA device")
            if t.device != lengths.device:
                raise ValueError("a batch's tensors must be on one device")
            if t.shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError(f"{name} must be contiguous in its last dimension")
        sequences = lengths.shape[0]
        if page_table.shape[0] != sequences or starts.shape[0] != sequences + 1:
            raise ValueError(f"a batch of {sequences} sequences has {sequences} table rows and {sequences + 1} starts, "
                             f"not {page_table.shape[0]} and {starts.shape[0]}")
        if max_rows is None:
            max_rows = int((starts[1:] - starts[:-1]).max()) if sequences else 0
        self.page_table, self.lengths, self.starts, self.max_rows = page_table, lengths, starts, max_rows
        self.device, self.index = lengths.device, lengths.get_device()
        self._c = CCacheBatch(page_table.data_ptr(), lengths.data_ptr(), starts.data_ptr(),
                              page_table.stride(0) if sequences > 1 else page_table.shape[1], page_table.shape[1],
                              sequences, max_rows)
        self._ref = ctypes.byref(self._c)
        self.columns = page_table.shape[1]

    def rows(self) -> int:
        """The rows of the calls' arrays, starts[-1] as it stands: waits for the
        device."""
        return int(self.starts[-1])


class PagedCache:
    """A paged key/value cache over torch tensors (wsp_cache).

    keys, values              [pages, heads, page_rows, head_width], float16,
                              bfloat16, float8_e4m3fn or int8, contiguous in
                              the last dimension
    key_scales, value_scales  uint8 [pages, heads, page_rows], contiguous
                              (8-bit storage): byte b stands for 2^(b - 127)
    """

    def __init__(self, keys, values, key_scales=None, value_scales=None):
        self._handle = None
        if not keys.is_cuda or keys.dim() != 4:
            raise ValueError("keys must be a 4-dimensional tensor on a CUDA device")
        if values.shape != keys.shape or values.dtype != keys.dtype or values.device != keys.device or \
                values.stride() != keys.stride():
            raise ValueError("keys and values must be alike")
        for name, t in (("keys", keys), ("values", values)):
            if t.requires_grad:
                _refuse_gradient(name)
        storage = CACHE_STORAGE.get(_name(keys.dtype))
        if storage is None:
            raise ValueError(f"a cache holds one of {sorted(CACHE_STORAGE)}, not {_name(keys.dtype)}")
        pages, heads, page_rows, width = keys.shape
        if keys.stride(3) != 1:
            raise ValueError("keys and values must be contiguous in the last dimension")
        self.eight = storage in (WSP_CACHE_E4M3, WSP_CACHE_INT8)
        if self.eight:
            for t in (key_scales, value_scales):
                if t is None or _name(t.dtype) != "uint8" or tuple(t.shape) != (pages, heads, page_rows) or \
                        t.device != keys.device or not t.is_contiguous():
                    raise ValueError(f"an 8-bit cache has scale bytes, contiguous uint8 tensors "
                                     f"[{pages}, {heads}, {page_rows}] on its device")
        elif key_scales is not None or value_scales is not None:
            raise ValueError("a 16-bit cache has no scales")
        self._lib = library()
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.heads, self.head_width, self.page_rows, self.pages = heads, width, page_rows, pages
        self.device, self.dtype = keys.device, keys.dtype
        shape = CCacheShape(heads, width, page_rows, pages, storage)
        # A dimension of one element may have any stride; the pools' rows are where this says.
        strides = [keys.stride(i) if keys.shape[i] > 1 else width for i in range(3)]
        memory = CCacheMemory(keys.data_ptr(), values.data_ptr(),
                              key_scales.data_ptr() if self.eight else None,
                              value_scales.data_ptr() if self.eight else None, *strides)
        handle = ctypes.c_void_p()
        check(self._lib.wsp_cache_create(ctypes.byref(shape), keys.device.index, ctypes.byref(memory),
                                         ctypes.byref(handle)))
        self._handle = handle
        self._index = keys.device.index
        self._scale = 1.0 / math.sqrt(width)
        self._workspace_bytes: dict = {}
        self._raw_stream = getattr(_torch()._C, "_cuda_getCurrentRawStream", None) or \
            (lambda index: _torch().cuda.current_stream(index).cuda_stream)

    @classmethod
    def allocate(cls, pages: int, heads: int, page_rows: int, head_width: int, storage: str = "float16",
                 device="cuda") -> "PagedCache":
        """A cache over zeroed tensors; storage is a key of CACHE_STORAGE."""
        if storage not in CACHE_STORAGE:
            raise ValueError(f"storage must be one of {sorted(CACHE_STORAGE)}")
        torch = _torch()
        dtype = getattr(torch, storage)
        pools = [torch.zeros(pages, heads, page_rows, head_width, dtype=torch.int8 if dtype.itemsize == 1 else dtype,
                             device=device).view(dtype) for _ in range(2)]
        if dtype.itemsize > 1:
            return cls(*pools)
        return cls(*pools, *[torch.zeros(pages, heads, page_rows, dtype=torch.uint8, device=device) for _ in range(2)])

    def close(self) -> None:
        if getattr(self, "_handle", None):
            self._lib.wsp_cache_destroy(self._handle)
            self._handle = None

    def __del__(self):
        self.close()

    # ------------------------------------------------------------ operators

    def append(self, batch: CacheBatch, keys, values, stream=None) -> None:
        """Writes keys and values [rows, heads, head_width] (float32, float16 or
        bfloat16) into the pages: the sequences' new rows, rounded once to the
        storage."""
        rows = keys.shape[0]
        k, v = self._rows(keys, "keys", rows, self.heads), self._rows(values, "values", rows, self.heads)
        check(self._lib.wsp_cache_append(self._usable(batch), batch._ref, rows, ctypes.byref(k), ctypes.byref(v),
                                         self._stream(stream)))

    def read(self, batch: CacheBatch, keys=None, values=None, dtype=None, rows: int | None = None, stream=None):
        """(keys, values) [rows, heads, head_width]: the sequences' last rows as
        the values they stand for.  Without `keys` and `values` to fill, new
        tensors of `dtype` (None: the cache's; float32 for 8-bit storage);
        `rows`, then, is how many there are (None: taken from the batch's
        starts as they stand, which waits for the device, and so cannot be
        captured).  Rows of no sequence are left alone: in new tensors they
        hold anything."""
        if (keys is None) != (values is None):
            raise ValueError("keys and values to fill are given together")
        handle = self._usable(batch)
        if keys is None:
            torch = _torch()
            if rows is None:
                rows = batch.rows()
            if dtype is None:
                dtype = torch.float32 if self.eight else self.dtype
            code = _codes.get(dtype)
            if code is None:
                code = _row_type(dtype)
            with self._allocating(stream):
                keys = torch.empty(rows, self.heads, self.head_width, dtype=dtype, device=self.device)
                values = torch.empty_like(keys)
            k, v = self._plain(keys, self.heads, code), self._plain(values, self.heads, code)
        else:
            rows = keys.shape[0]
            k, v = self._rows(keys, "keys", rows, self.heads), self._rows(values, "values", rows, self.heads)
        check(self._lib.wsp_cache_read(handle, batch._ref, rows, ctypes.byref(k), ctypes.byref(v), self._stream(stream)))
        return keys, values

    def attend(self, batch: CacheBatch, queries, out=None, lse=None, scale: float | None = None, causal: bool = True,
               return_lse: bool = False, stream=None):
        """softmax(scale q . k) v of the new rows over what their sequences hold
        (append first): the positions up to a row's own, or all (causal=False).

        queries [rows, query_heads, head_width], float16 or bfloat16 (a 16-bit
        cache's own type); query_heads a multiple of the cache's heads.  scale
        None is 1 / sqrt(head_width).  Returns out (new, or the one given), or
        (out, lse) with return_lse or an `lse` to fill: float32 [rows,
        query_heads], the log of the sum of exponentials.  A row without a key
        gets zeros and -inf; rows of no sequence are left alone (in a new out
        they hold anything).
        """
        shape = queries.shape
        if len(shape) != 3:
            raise ModelError(f"queries must be [rows, query_heads, {self.head_width}], not {list(shape)}")
        rows, heads, _ = shape
        q = self._rows(queries, "queries", rows, heads)
        handle = self._usable(batch)
        key = (heads, batch.max_rows, batch.columns)
        needed = self._workspace_bytes.get(key)
        if needed is None:
            size = ctypes.c_size_t()
            check(self._lib.wsp_cache_attend_workspace(handle, batch._ref, rows, heads, ctypes.byref(size)))
            needed = self._workspace_bytes[key] = size.value
        torch = _torch()
        with self._allocating(stream):
            if out is None:
                out = torch.empty_like(queries, memory_format=torch.contiguous_format)
                o = self._plain(out, heads, q.dtype)
            else:
                o = self._rows(out, "out", rows, heads)
            if lse is None:
                if return_lse:
                    lse = torch.empty(rows, heads, dtype=torch.float32, device=self.device)
            elif lse.shape != (rows, heads) or lse.dtype != torch.float32 or not lse.is_contiguous() or \
                    lse.get_device() != self._index:
                raise ValueError(f"lse must be a contiguous float32 tensor [{rows}, {heads}] on the cache's device")
            elif lse.requires_grad:
                _refuse_gradient("lse")
            workspace = self._workspace(needed, stream) if needed else None
        check(self._lib.wsp_cache_attend(handle, batch._ref, rows, heads, ctypes.byref(q), ctypes.byref(o),
                                         lse.data_ptr() if lse is not None else None,
                                         self._scale if scale is None else scale, causal,
                                         workspace.data_ptr() if needed else None, needed, self._stream(stream)))
        return out if lse is None else (out, lse)

    def check(self) -> None:
        """Waits for the device and raises if a kernel gave up (wsp_cache_check)."""
        check(self._lib.wsp_cache_check(self._handle))

    # -------------------------------------------------------------- helpers

    def _usable(self, batch: CacheBatch):
        if self._handle is None:
            raise ValueError("the cache is closed")
        if batch.index != self._index:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        return self._handle

    def _rows(self, t, name: str, rows: int, heads: int) -> CCacheRows:
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on {self.device}, not {t.device}")
        if t.requires_grad:
            _refuse_gradient(name)
        if t.shape != (rows, heads, self.head_width):
            raise ModelError(f"{name} must be [{rows}, {heads}, {self.head_width}], not {list(t.shape)}")
        row_stride, head_stride, step = t.stride()
        if step != 1:
            raise ValueError(f"{name} must be contiguous in the last dimension")
        code = _codes.get(t.dtype)
        return CCacheRows(t.data_ptr(), row_stride, head_stride, _row_type(t.dtype) if code is None else code)

    def _plain(self, t, heads: int, code: int) -> CCacheRows:
        """A new, contiguous row array."""
        return CCacheRows(t.data_ptr(), heads * self.head_width, self.head_width, code)

    def _stream(self, stream):
        if stream is None:
            return self._raw_stream(self._index)
        return getattr(stream, "cuda_stream", stream)

    def _workspace(self, needed: int, stream):
        """A call's workspace.  Calls of one host thread on one of torch's
        streams follow one another, whichever cache they are of, so they share
        it, and it ends with the thread; a captured call, whose graph may run
        next to others, and a call on a given stream get their own, which
        torch's allocator keeps for that stream's later work."""
        torch = _torch()
        if stream is not None or self._capturing():
            return torch.empty(needed, dtype=torch.uint8, device=self.device)
        key = (self._index, self._raw_stream(self._index))
        held = _workspaces.__dict__.get(key)
        if held is None or held.numel() < needed:
            held = _workspaces.__dict__[key] = torch.empty(needed, dtype=torch.uint8, device=self.device)
        return held

    def _capturing(self) -> bool:
        """Whether the current stream of the cache's device, which need not be
        the current device, is being captured."""
        torch = _torch()
        if torch.cuda.current_device() == self._index:
            return torch.cuda.is_current_stream_capturing()
        with torch.cuda.device(self._index):
            return torch.cuda.is_current_stream_capturing()

    def _allocating(self, stream):
        """The context in which a call's tensors are allocated: its own stream,
        so that memory freed after the call is not handed to another too early."""
        torch = _torch()
        if stream is None:
            return _NOTHING
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(stream, device=self.device)
        return torch.cuda.stream(stream)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NOTHING = _Nothing()
