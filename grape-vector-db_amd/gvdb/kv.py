"""Token cache over the MI355X C ABI (include/gvdb.h: gvdb_kv_*): the keys and
values of a model's context, paged and held in 4 bits, with the attention that
reads them.

It stands beside the index as the index's own two stages do: tokens are
quantised as they are written (as :class:`gvdb.BinaryQuantizer` quantises
rows), :meth:`KvCache.attend` reads everything a sequence holds (the flat
scan), :meth:`KvCache.attend_topk` scores pages by small codes first and reads
the best ones exactly (the two-stage search).  The cache's buffers are torch
tensors; pages are handed out by the caller.  Work is enqueued on torch's
current stream of the cache's device; nothing waits.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Tuple

from . import InvalidArgument, InvalidVectorDimension, _ffi, check
from ._ffi import lib

__all__ = ["KvCache"]

# struct gvdb_kv_rows and struct gvdb_kv_batch of include/gvdb.h
_ROWS = struct.Struct("@PqqII").pack
_BATCH = struct.Struct("@PQIIPPIIII").pack


class KvCache:
    """Pages of ``page_size`` tokens for every key/value head.

    ``pool`` (uint8 [n_pages, kv_heads, page_size / 32, 34 * head_dim]), ``bounds``
    (int8 [n_pages, kv_heads, 2, head_dim]) and ``bound_exps`` (uint8 [n_pages,
    kv_heads]) are laid out as include/gvdb.h says.  ``page_table`` is int32
    [sequences, width]: each sequence's pages in token order.  A row tensor is
    [rows, heads, head_dim] in bf16, f16 or f32 with neighbouring channels side by
    side; its rows belong to the sequences by ``cu`` (int32 [sequences + 1]), or
    evenly without it.  ``stream`` (a HIP stream's handle) runs a call there instead of
    on torch's current stream: the caller orders the two streams; tensors may be dropped as
    soon as the call returns.  ``max_new`` (most rows of one sequence) and ``max_len`` (the
    largest length) size the launch and change no result.  Nothing here has a gradient: rows
    that require one are refused where gradients are recorded.
    """

    def __init__(self, n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        import torch

        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if page_size <= 0 or page_size % 32 or page_size > 1024:
            raise InvalidArgument("page_size is a multiple of 32, at most 1024")
        pool = torch.empty(n_pages, kv_heads, page_size // 32, 34 * head_dim, dtype=torch.uint8, device=dev)
        bounds = torch.empty(n_pages, kv_heads, 2, head_dim, dtype=torch.int8, device=dev)
        self._take(pool, bounds, torch.empty(n_pages, kv_heads, dtype=torch.uint8, device=dev))

    @classmethod
    def from_buffers(cls, pool, bounds, bound_exps) -> "KvCache":
        """The cache in buffers that are there already; they are kept, not copied."""
        self = cls.__new__(cls)
        self._take(pool, bounds, bound_exps)
        return self

    def _take(self, pool, bounds, bound_exps) -> None:
        import torch

        if pool.dim() != 4 or bounds.dim() != 4 or bound_exps.dim() != 2:
            raise InvalidArgument("pool and bounds have four dimensions, bound_exps two")
        n, h, tiles, size = pool.shape
        if size % 34 or tuple(bounds.shape) != (n, h, 2, size // 34) or tuple(bound_exps.shape) != (n, h):
            raise InvalidArgument("pool, bounds and bound_exps are of one cache")
        if size // 34 not in (64, 128, 256):
            raise InvalidVectorDimension("head_dim is 64, 128 or 256")
        if not 0 < n <= 1 << 31 or not 0 < h <= 4096 or not 0 < tiles <= 32:
            raise InvalidArgument("a cache has 1 .. 2^31 pages of at most 1024 tokens and 1 .. 4096 heads")
        for t, want in ((pool, torch.uint8), (bounds, torch.int8), (bound_exps, torch.uint8)):
            if t.dtype != want or not t.is_contiguous() or t.device != pool.device:
                raise InvalidArgument("the cache's buffers are contiguous uint8, int8 and uint8 tensors of one device")
        if pool.device.type != "cuda":
            raise InvalidArgument("the cache's buffers are on the GPU")
        self.pool, self.bounds, self.bound_exps = pool, bounds, bound_exps
        self.n_pages, self.kv_heads, self.head_dim, self.page_size = n, h, size // 34, tiles * 32
        self.device = pool.device
        self._lib = lib()
        self._torch = torch
        self._codes = {torch.float32: _ffi.GVDB_F32, torch.float16: _ffi.GVDB_F16, torch.bfloat16: _ffi.GVDB_BF16}
        self._i32, self._index, self._raw_stream = torch.int32, pool.get_device(), torch._C._cuda_getCurrentRawStream
        self._scale, self._sizes = 1.0 / math.sqrt(self.head_dim), {}
        self._c = _ffi.gvdb_kv_cache(pool.data_ptr(), bounds.data_ptr(), bound_exps.data_ptr(), n, h, self.head_dim,
                                     self.page_size, self._index)
        self._ref = C.byref(self._c)

    # -- arguments ----------------------------------------------------------
    # A step's calls are shorter on the device than in Python: the C structs are packed as bytes (a third of a ctypes
    # Structure's time), and a size's scratch is asked for once.
    def _rows(self, t, what: str, heads: int, rows: int, flags: int = 0) -> bytes:
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[0] != rows or shape[1] != heads or shape[2] != self.head_dim:
            raise InvalidArgument(f"{what} is [{rows}, {heads}, {self.head_dim}]: got {tuple(shape)}")
        code = self._codes.get(t.dtype)
        if code is None:
            raise InvalidArgument(f"{what} is bf16, f16 or f32: got {t.dtype}")
        if t.get_device() != self._index:
            raise InvalidArgument(f"{what} is on {t.device}, the cache on {self.device}")
        if stride[2] != 1:
            raise InvalidArgument(f"{what}'s neighbouring channels lie side by side")
        if t.requires_grad and self._torch.is_grad_enabled():  # its result would silently have none
            raise InvalidArgument(f"{what} requires a gradient, which a cache in 4 bits does not have: detach it, or call under torch.no_grad()")
        return _ROWS(t.data_ptr(), stride[0], stride[1], code, flags)

    def _batch(self, page_table, lengths, cu, rows: int, max_new: int, max_len: int):
        """(struct, sizes): the sizes are all that a call's scratch goes by."""
        i32, dev = self._i32, self._index
        shape, stride = page_table.shape, page_table.stride()
        if len(shape) != 2 or lengths.shape != shape[:1]:
            raise InvalidArgument("page_table is [sequences, width], lengths [sequences]")
        n, width = shape
        if page_table.dtype != i32 or lengths.dtype != i32 or page_table.get_device() != dev or lengths.get_device() != dev:
            raise InvalidArgument("page_table and lengths are int32 tensors on the cache's device")
        if (width > 1 and stride[1] != 1) or (n > 1 and (lengths.stride(0) != 1 or stride[0] < width)):
            raise InvalidArgument("page_table's rows and lengths are contiguous")
        if cu is None:
            at = 0
        else:
            if cu.dim() != 1 or cu.shape[0] != n + 1 or cu.dtype != i32 or cu.get_device() != dev or cu.stride(0) != 1:
                raise InvalidArgument("cu is a contiguous int32 [sequences + 1] on the cache's device")
            at = cu.data_ptr()
        if max_new < 0 or max_len < 0 or max_new > 0xFFFFFFFF or max_len > 0xFFFFFFFF:
            raise InvalidArgument("max_new and max_len are not negative, and below 2^32")
        return (_BATCH(page_table.data_ptr(), stride[0], width, n, lengths.data_ptr(), at, rows, max_new, max_len, 0),
                (rows, n, width, at != 0, max_new, max_len))

    def _stream(self):
        return self._raw_stream(self._index) or None

    def _on(self, stream: int, tensors, call):
        """``call()`` with torch's current stream made the given one.  What it allocates belongs to that stream; what it is given, and
        the cache, are kept from other use until that stream is through with them, and its results until the caller's is."""
        cuda = self._torch.cuda
        here = cuda.current_stream(self.device)
        there = cuda.ExternalStream(stream, device=self.device) if stream else cuda.default_stream(self.device)
        with cuda.stream(there):
            result = call()
        for t in (*tensors, self.pool, self.bounds, self.bound_exps):
            if t is not None:
                t.record_stream(there)
        for t in () if result is None else result if isinstance(result, (tuple, list)) else (result,):
            t.record_stream(here)
        return result

    # -- operators ----------------------------------------------------------
    def append(self, k, v, page_table, lengths, cu=None, max_new: int = 0, stream: Optional[int] = None) -> None:
        """Writes rows ``k`` and ``v`` as tokens ``lengths[s]`` .. of each sequence (``lengths``: tokens before the call)."""
        if stream is not None:
            return self._on(stream, (k, v, page_table, lengths, cu), lambda: self.append(k, v, page_table, lengths, cu, max_new))
        rows = k.shape[0]
        kr = self._rows(k, "k", self.kv_heads, rows)
        vr = self._rows(v, "v", self.kv_heads, rows)
        bt, _ = self._batch(page_table, lengths, cu, rows, max_new, 0)
        status = self._lib.gvdb_kv_append_device(self._ref, bt, kr, vr, self._stream())
        if status:
            check(status)

    def read(self, page_table, lengths, rows: int, cu=None, max_new: int = 0, dtype=None, out=None,
             stream: Optional[int] = None) -> Tuple:
        """The stored keys and values of the tokens that an append of ``rows`` rows with the same arguments writes.
        Rows behind the last sequence are left as they were in ``out``, and are 0 without it."""
        if stream is not None:
            return self._on(stream, (page_table, lengths, cu, *(() if out is None else (out[0], out[1]))),
                            lambda: self.read(page_table, lengths, rows, cu, max_new, dtype, out))
        torch, flags = self._torch, 0
        if out is None:
            shape, flags = (rows, self.kv_heads, self.head_dim), _ffi.GVDB_KV_ZERO_REST
            dtype = dtype or torch.bfloat16
            out = (torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device))
        kr = self._rows(out[0], "out[0]", self.kv_heads, rows, flags)
        vr = self._rows(out[1], "out[1]", self.kv_heads, rows, flags)
        bt, _ = self._batch(page_table, lengths, cu, rows, max_new, 0)
        status = self._lib.gvdb_kv_read_device(self._ref, bt, kr, vr, self._stream())
        if status:
            check(status)
        return out

    def _attend_args(self, q, page_table, lengths, cu, max_new, max_len, scale, out, lse, top):
        torch = self._torch
        shape = q.shape
        if len(shape) != 3:
            raise InvalidArgument("q is [rows, heads, head_dim]")
        rows, heads = shape[0], shape[1]
        qr, flags = self._rows(q, "q", heads, rows), 0
        if out is None:  # rows behind the last sequence read 0; in a given `out` they stay what they were
            out, flags = torch.empty_like(q), _ffi.GVDB_KV_ZERO_REST
        orow = self._rows(out, "out", heads, rows, flags)
        if lse is not None and (tuple(lse.shape) != (rows, heads) or lse.dtype != torch.float32 or lse.get_device() != self._index
                                or not lse.is_contiguous()):
            raise InvalidArgument("lse is a contiguous float32 [rows, heads] on the cache's device")
        bt, sizes = self._batch(page_table, lengths, cu, rows, max_new, max_len)
        key = (sizes, heads, top)
        size = self._sizes.get(key)
        if size is None:
            n = C.c_uint64()
            check(self._lib.gvdb_kv_scratch_bytes(self._ref, bt, heads, top, C.byref(n)))
            if len(self._sizes) >= 4096:
                self._sizes.clear()
            size = self._sizes[key] = n.value
        # torch's allocator keeps it apart from other streams' and graphs' scratch
        scratch = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        return heads, qr, orow, bt, (self._scale if scale is None else scale), out, scratch, size

    def attend(self, q, page_table, lengths, cu=None, max_new: int = 0, max_len: int = 0, scale: Optional[float] = None,
               causal: bool = True, out=None, lse=None, stream: Optional[int] = None):
        """Attention of rows ``q`` over their sequences' tokens (``lengths``: with the call's own).  With ``causal``, row i of a
        sequence's n sees the first ``length - n + i + 1`` tokens.  ``scale``: 1 / sqrt(head_dim) by default; ``lse``
        [rows, heads] float32 takes the logarithm of the softmax's denominator.  A row that sees nothing is 0."""
        if stream is not None:
            return self._on(stream, (q, page_table, lengths, cu, out, lse),
                            lambda: self.attend(q, page_table, lengths, cu, max_new, max_len, scale, causal, out, lse))
        heads, qr, orow, bt, scale, out, scratch, size = self._attend_args(q, page_table, lengths, cu, max_new, max_len, scale, out,
                                                                           lse, 0)
        status = self._lib.gvdb_kv_attend_device(self._ref, bt, qr, heads, scale, 1 if causal else 0, orow, _ffi.ptr(lse),
                                                 _ffi.ptr(scratch), size, self._stream())
        if status:
            check(status)
        return out

    def attend_topk(self, q, page_table, lengths, top: int, first: int = 1, recent: int = 1, cu=None, max_new: int = 0,
                    max_len: int = 0, scale: Optional[float] = None, out=None, chosen=None, lse=None,
                    stream: Optional[int] = None) -> Tuple:
        """Causal attention over ``top`` pages of each row and key/value head: the ``first`` first, the ``recent`` last, and
        those whose key bounds promise the largest scores.  Returns ``(out, chosen)``; ``chosen`` is int32 [rows, kv_heads,
        top], positions in the page table in order, -1 behind the last."""
        if stream is not None:
            return self._on(stream, (q, page_table, lengths, cu, out, chosen, lse),
                            lambda: self.attend_topk(q, page_table, lengths, top, first, recent, cu, max_new, max_len, scale, out, chosen, lse))
        torch = self._torch
        if top < 1 or first < 0 or recent < 0 or first + recent > top:
            raise InvalidArgument("top is at least 1 and at least first + recent, which are not negative")
        shape = (q.shape[0], self.kv_heads, top)
        if out is not None and chosen is None and cu is not None:  # its rows behind the last sequence are left alone as out's are
            chosen = torch.full(shape, -1, dtype=torch.int32, device=self.device)
        heads, qr, orow, bt, scale, out, scratch, size = self._attend_args(q, page_table, lengths, cu, max_new, max_len, scale, out,
                                                                           lse, top)
        if chosen is None:
            chosen = torch.empty(shape, dtype=torch.int32, device=self.device)
        elif tuple(chosen.shape) != shape or chosen.dtype != torch.int32 or chosen.get_device() != self._index or not chosen.is_contiguous():
            raise InvalidArgument("chosen is a contiguous int32 [rows, kv_heads, top] on the cache's device")
        status = self._lib.gvdb_kv_attend_topk_device(self._ref, bt, qr, heads, scale, top, first, recent, orow, chosen.data_ptr(),
                                                      _ffi.ptr(lse), _ffi.ptr(scratch), size, self._stream())
        if status:
            check(status)
        return out, chosen
