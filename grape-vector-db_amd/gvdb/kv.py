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
from typing import Optional, Tuple

from . import InvalidArgument, InvalidVectorDimension, _ffi, check
from ._ffi import lib

__all__ = ["KvCache"]


class KvCache:
    """Pages of ``page_size`` tokens for every key/value head.

    ``pool`` (uint8 [n_pages, kv_heads, page_size / 32, 34 * head_dim]), ``bounds``
    (int8 [n_pages, kv_heads, 2, head_dim]) and ``bound_exps`` (uint8 [n_pages,
    kv_heads]) are laid out as include/gvdb.h says.  ``page_table`` is int32
    [sequences, width]: each sequence's pages in token order.  A row tensor is
    [rows, heads, head_dim] in bf16, f16 or f32 with neighbouring channels side by
    side; its rows belong to the sequences by ``cu`` (int32 [sequences + 1]), or
    evenly without it.  ``max_new`` (most rows of one sequence) and ``max_len`` (the
    largest length) size the launch and change no result.
    """

    def __init__(self, n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        import torch

        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if page_size <= 0 or page_size % 32:
            raise InvalidArgument("page_size is a multiple of 32")
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
        self._c = _ffi.gvdb_kv_cache(pool.data_ptr(), bounds.data_ptr(), bound_exps.data_ptr(), n, h, self.head_dim,
                                     self.page_size, self.device.index or 0)
        self._ref = C.byref(self._c)

    # -- arguments ----------------------------------------------------------
    def _rows(self, t, what: str, heads: int, rows: int):
        if t.dim() != 3 or t.shape[0] != rows or t.shape[1] != heads or t.shape[2] != self.head_dim:
            raise InvalidArgument(f"{what} is [{rows}, {heads}, {self.head_dim}]: got {tuple(t.shape)}")
        code = self._codes.get(t.dtype)
        if code is None:
            raise InvalidArgument(f"{what} is bf16, f16 or f32: got {t.dtype}")
        if t.device != self.device:
            raise InvalidArgument(f"{what} is on {t.device}, the cache on {self.device}")
        s = t.stride()
        if s[2] != 1:
            raise InvalidArgument(f"{what}'s neighbouring channels lie side by side")
        return _ffi.gvdb_kv_rows(t.data_ptr(), s[0], s[1], code, 0)

    def _batch(self, page_table, lengths, cu, rows: int, max_new: int, max_len: int):
        i32, dev = self._torch.int32, self.device
        if page_table.dim() != 2 or lengths.dim() != 1 or lengths.shape[0] != page_table.shape[0]:
            raise InvalidArgument("page_table is [sequences, width], lengths [sequences]")
        n = page_table.shape[0]
        if page_table.dtype != i32 or lengths.dtype != i32 or page_table.device != dev or lengths.device != dev:
            raise InvalidArgument("page_table and lengths are int32 tensors on the cache's device")
        if page_table.stride(1) != 1 or (n > 1 and lengths.stride(0) != 1):
            raise InvalidArgument("page_table's rows and lengths are contiguous")
        if cu is not None and (cu.dim() != 1 or cu.shape[0] != n + 1 or cu.dtype != i32 or cu.device != dev or cu.stride(0) != 1):
            raise InvalidArgument("cu is a contiguous int32 [sequences + 1] on the cache's device")
        if max_new < 0 or max_len < 0:
            raise InvalidArgument("max_new and max_len are not negative")
        return _ffi.gvdb_kv_batch(page_table.data_ptr(), page_table.stride(0), page_table.shape[1], n, lengths.data_ptr(),
                                  None if cu is None else cu.data_ptr(), rows, max_new, max_len, 0)

    def _stream(self, stream: Optional[int]):
        if stream is not None:
            return stream or None
        return self._torch.cuda.current_stream(self.device).cuda_stream or None

    # -- operators ----------------------------------------------------------
    def append(self, k, v, page_table, lengths, cu=None, max_new: int = 0, stream: Optional[int] = None) -> None:
        """Writes rows ``k`` and ``v`` as tokens ``lengths[s]`` .. of each sequence (``lengths``: tokens before the call)."""
        kr = self._rows(k, "k", self.kv_heads, k.shape[0])
        vr = self._rows(v, "v", self.kv_heads, k.shape[0])
        bt = self._batch(page_table, lengths, cu, k.shape[0], max_new, 0)
        check(self._lib.gvdb_kv_append_device(self._ref, C.byref(bt), C.byref(kr), C.byref(vr), self._stream(stream)))

    def read(self, page_table, lengths, rows: int, cu=None, max_new: int = 0, dtype=None, out=None,
             stream: Optional[int] = None) -> Tuple:
        """The stored keys and values of the tokens that an append of ``rows`` rows with the same arguments writes.
        Rows behind the last sequence are left as they were in ``out``, and are 0 without it."""
        torch = self._torch
        if out is None:
            make = torch.empty if cu is None else torch.zeros
            shape = (rows, self.kv_heads, self.head_dim)
            dtype = dtype or torch.bfloat16
            out = (make(shape, dtype=dtype, device=self.device), make(shape, dtype=dtype, device=self.device))
        kr = self._rows(out[0], "out[0]", self.kv_heads, rows)
        vr = self._rows(out[1], "out[1]", self.kv_heads, rows)
        bt = self._batch(page_table, lengths, cu, rows, max_new, 0)
        check(self._lib.gvdb_kv_read_device(self._ref, C.byref(bt), C.byref(kr), C.byref(vr), self._stream(stream)))
        return out

    def _attend_args(self, q, page_table, lengths, cu, max_new, max_len, scale, out, lse):
        torch = self._torch
        if q.dim() != 3:
            raise InvalidArgument("q is [rows, heads, head_dim]")
        rows, heads = q.shape[0], q.shape[1]
        qr = self._rows(q, "q", heads, rows)
        if out is None:
            # rows behind the last sequence are not written: without `out` they read 0
            out = (torch.empty if cu is None else torch.zeros)(q.shape, dtype=q.dtype, device=self.device)
        orow = self._rows(out, "out", heads, rows)
        if lse is not None and (tuple(lse.shape) != (rows, heads) or lse.dtype != torch.float32 or lse.device != self.device
                                or not lse.is_contiguous()):
            raise InvalidArgument("lse is a contiguous float32 [rows, heads] on the cache's device")
        bt = self._batch(page_table, lengths, cu, rows, max_new, max_len)
        return heads, qr, orow, bt, (1.0 / math.sqrt(self.head_dim) if scale is None else scale), out

    def _scratch(self, bt, heads: int, top: int):
        n = C.c_uint64()
        check(self._lib.gvdb_kv_scratch_bytes(self._ref, C.byref(bt), heads, top, C.byref(n)))
        # torch's allocator keeps it apart from other streams' and graphs' scratch
        return self._torch.empty(n.value, dtype=self._torch.uint8, device=self.device) if n.value else None, n.value

    def attend(self, q, page_table, lengths, cu=None, max_new: int = 0, max_len: int = 0, scale: Optional[float] = None,
               causal: bool = True, out=None, lse=None, stream: Optional[int] = None):
        """Attention of rows ``q`` over their sequences' tokens (``lengths``: with the call's own).  With ``causal``, row i of a
        sequence's n sees the first ``length - n + i + 1`` tokens.  ``scale``: 1 / sqrt(head_dim) by default; ``lse``
        [rows, heads] float32 takes the logarithm of the softmax's denominator.  A row that sees nothing is 0."""
        heads, qr, orow, bt, scale, out = self._attend_args(q, page_table, lengths, cu, max_new, max_len, scale, out, lse)
        scratch, size = self._scratch(bt, heads, 0)
        check(self._lib.gvdb_kv_attend_device(self._ref, C.byref(bt), C.byref(qr), heads, scale, int(causal), C.byref(orow),
                                              _ffi.ptr(lse), _ffi.ptr(scratch), size, self._stream(stream)))
        return out

    def attend_topk(self, q, page_table, lengths, top: int, first: int = 1, recent: int = 1, cu=None, max_new: int = 0,
                    max_len: int = 0, scale: Optional[float] = None, out=None, chosen=None, lse=None,
                    stream: Optional[int] = None) -> Tuple:
        """Causal attention over ``top`` pages of each row and key/value head: the ``first`` first, the ``recent`` last, and
        those whose key bounds promise the largest scores.  Returns ``(out, chosen)``; ``chosen`` is int32 [rows, kv_heads,
        top], positions in the page table in order, -1 behind the last."""
        torch = self._torch
        heads, qr, orow, bt, scale, out = self._attend_args(q, page_table, lengths, cu, max_new, max_len, scale, out, lse)
        if top < 1 or first < 0 or recent < 0:
            raise InvalidArgument("top is at least 1, first and recent are not negative")
        shape = (q.shape[0], self.kv_heads, top)
        if chosen is None:
            chosen = torch.empty(shape, dtype=torch.int32, device=self.device) if cu is None else torch.full(
                shape, -1, dtype=torch.int32, device=self.device)
        elif tuple(chosen.shape) != shape or chosen.dtype != torch.int32 or chosen.device != self.device or not chosen.is_contiguous():
            raise InvalidArgument("chosen is a contiguous int32 [rows, kv_heads, top] on the cache's device")
        scratch, size = self._scratch(bt, heads, top)
        check(self._lib.gvdb_kv_attend_topk_device(self._ref, C.byref(bt), C.byref(qr), heads, scale, top, first, recent,
                                                   C.byref(orow), chosen.data_ptr(), _ffi.ptr(lse), _ffi.ptr(scratch), size,
                                                   self._stream(stream)))
        return out, chosen
