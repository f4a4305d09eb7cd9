"""Paged key/value cache: append, attention of one new token, eviction.

`PagedKV` wraps the gawee_kv entry points of include/gawee_cuda.h, which state
what each call computes, what it leaves alone and which calls may overlap.
The caller owns every array; the handle holds the shapes and the scratch
memory.  Arrays are device tensors of the handle's device, of any library
whose tensors have `data_ptr()`, `shape`, `stride()`, `is_contiguous()`,
`dtype` and `get_device()` as PyTorch's do.

    pages:    k_pages, v_pages [num_pages, kv_heads, page_size, head_dim]
    table:    block_table int32 [batch, columns], a sequence's pages in order
    lengths:  int32 [batch], cached rows of each sequence

A decode step of one layer, in one captured graph for every length:

    kv = PagedKV("bf16", heads, kv_heads, head_dim, page_size, num_pages, max_batch, max_pages)
    kv.attend(k_pages, v_pages, q, table, lengths, out, k=k_new, v=v_new, stream=stream)

Calls are asynchronous on `stream` (a stream object or a cudaStream_t value;
None: the device's default stream).  Errors that only the device can see
(a table entry that names no page) are raised by `synchronize`.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

from .runtime import GaweeError, _stream_ptr, load_library

DTYPES = {"f32": 0, "f16": 2, "bf16": 7}
_NAMES = {"float32": 0, "float16": 2, "bfloat16": 7, "int32": 4}
_dtype_codes: dict = {}

# The argument structures of include/gawee_cuda.h, packed with C alignment.
_DESC = struct.Struct("@iiiiiqqiii0q")  # 0q: the padding behind the last member
_APPEND = struct.Struct("@PPPPiqqqPPPqii")
_ATTEND = struct.Struct("@PPPPiqqifPqiPPPqqPqqPqqPqqq")
_EVICT = struct.Struct("@PPPqqPqqqiPqiPqiPPiiP")


def _code(t) -> int:
    """The GAWEE_ code of a tensor's dtype, -1 for one that the cache does not take."""
    d = t.dtype
    c = _dtype_codes.get(d)
    if c is None:
        c = _dtype_codes[d] = _NAMES.get(str(d).rsplit(".", 1)[-1], -1)
    return c


def _invalid(msg: str) -> GaweeError:
    return GaweeError(1, msg)


class PagedKV:
    """Shapes and scratch memory of a paged key/value cache on one B200.

    dtype, kv_heads, head_dim, page_size, num_pages: of the pages.
    page_stride: elements between pages (0: they are dense), where one buffer
        holds more than this cache, e.g. [num_pages, 2, kv_heads, ...] for K and V.
    heads: query heads, a multiple of kv_heads.
    max_batch, max_pages: rows and columns of a block table at most.
    weights: whether `attend` may return attention weights.
    device: -1 for a handle whose calls only check their arguments.
    """

    def __init__(self, dtype: str, heads: int, kv_heads: int, head_dim: int, page_size: int, num_pages: int,
                 max_batch: int, max_pages: int, weights: bool = False, page_stride: int = 0, device: int = 0):
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be one of {sorted(DTYPES)}, not {dtype!r}")
        self._h = None
        for name, n in (("heads", heads), ("kv_heads", kv_heads), ("head_dim", head_dim), ("page_size", page_size),
                        ("max_batch", max_batch), ("max_pages", max_pages)):
            if not 0 < n < 1 << 31:  # a C int would take it modulo 2^32
                raise _invalid(f"{name} is {n}")
        self._lib = load_library()
        h = ctypes.c_void_p()
        try:
            desc = _DESC.pack(DTYPES[dtype], heads, kv_heads, head_dim, page_size, num_pages, page_stride, max_batch,
                              max_pages, 1 if weights else 0)
        except struct.error as e:
            raise _invalid(str(e)) from None
        self._check(self._lib.gawee_kv_create(desc, device, ctypes.byref(h)))
        self._h = h
        self.device = device
        self._dt = DTYPES[dtype]
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self._page_shape = (num_pages, kv_heads, page_size, head_dim)
        self._page_stride = page_stride or kv_heads * page_size * head_dim
        self._dense_pages = self._page_stride == kv_heads * page_size * head_dim
        self._page_strides = (self._page_stride, page_size * head_dim, head_dim, 1)

    def close(self):
        if getattr(self, "_h", None):
            self._lib.gawee_kv_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st: int):
        if st:
            buf = ctypes.create_string_buffer(4096)
            self._lib.gawee_last_error(None, buf, len(buf))
            raise GaweeError(st, buf.value.decode())

    # -- argument checks ---------------------------------------------------------
    def _on_device(self, t, name: str, code: Optional[int]) -> int:
        """The address of `t`, of dtype `code` (None: f32, f16 or bf16) on the handle's device."""
        if t.get_device() != self.device:
            raise _invalid(f"{name} is on device {t.get_device()}, the handle on {self.device}")
        c = _dtype_codes.get(t.dtype)
        if c is None:
            c = _code(t)
        if c != code if code is not None else c not in (0, 2, 7):
            raise _invalid(f"{name} has dtype {t.dtype}")
        return t.data_ptr()

    def _pages(self, t, name: str) -> int:
        if t.shape != self._page_shape:
            raise _invalid(f"{name} has shape {tuple(t.shape)}, expected {self._page_shape}")
        if self._dense_pages and t.is_contiguous():
            return self._on_device(t, name, self._dt)
        s = t.stride()
        n, kvh, page, dim = self._page_shape
        if s != self._page_strides and (s[3] != 1 or (page > 1 and s[2] != dim) or (kvh > 1 and s[1] != page * dim)
                or (n > 1 and s[0] != self._page_stride)):
            raise _invalid(f"{name} has strides {tuple(s)}: pages are dense, {self._page_stride} elements apart")
        return self._on_device(t, name, self._dt)

    def _rows(self, t, name: str, n: int, heads: int, code: Optional[int]):
        """(address, stride between rows) of [n, heads, head_dim] with dense rows."""
        if t.shape != (n, heads, self.head_dim):
            raise _invalid(f"{name} has shape {tuple(t.shape)}, expected {(n, heads, self.head_dim)}")
        if t.is_contiguous():
            return self._on_device(t, name, code), heads * self.head_dim
        s = t.stride()
        if s[2] != 1 or (heads > 1 and s[1] != self.head_dim):
            raise _invalid(f"{name} has strides {tuple(s)}: each row [heads, head_dim] is dense")
        return self._on_device(t, name, code), s[0]

    def _ints(self, t, name: str, n: int) -> int:
        if t.shape != (n,) or not t.is_contiguous():
            raise _invalid(f"{name} must be a dense array of {n} int32 values, got shape {tuple(t.shape)}")
        return self._on_device(t, name, 4)

    def _table(self, t, name: str):
        """(address, stride, rows, columns)"""
        shape = t.shape
        if len(shape) == 2 and t.is_contiguous():
            return self._on_device(t, name, 4), shape[1], shape[0], shape[1]
        s = t.stride()
        if len(shape) != 2 or (shape[1] > 1 and s[1] != 1):
            raise _invalid(f"{name} must be int32 [batch, columns] with dense rows")
        return self._on_device(t, name, 4), s[0], shape[0], shape[1]

    def _weights(self, t, name: str, batch: int):
        """(address, stride between heads, between sequences, columns)"""
        if len(t.shape) != 3 or t.shape[:2] != (batch, self.kv_heads) or t.shape[2] < 1 or t.stride()[2] != 1:
            raise _invalid(f"{name} must be f32 [{batch}, {self.kv_heads}, columns] with dense rows, "
                           f"got shape {tuple(t.shape)}")
        s = t.stride()
        return self._on_device(t, name, 0), s[1], s[0], t.shape[2]

    # -- operators ---------------------------------------------------------------
    def append(self, k_pages, v_pages, k, v, block_table, positions, sequences=None, stream=None):
        """Write new rows k, v [tokens, kv_heads, head_dim] to the pages: token t
        becomes row positions[t] of sequence sequences[t] (None: of sequence t).
        Tokens with a negative position or sequence are left out."""
        n = k.shape[0]
        kp, ks = self._rows(k, "k", n, self.kv_heads, None)
        vp, vs = self._rows(v, "v", n, self.kv_heads, _code(k))
        tp, ts, batch, cols = self._table(block_table, "block_table")
        a = _APPEND.pack(self._pages(k_pages, "k_pages"), self._pages(v_pages, "v_pages"), kp, vp, _code(k), ks, vs, n,
                         0 if sequences is None else self._ints(sequences, "sequences", n),
                         self._ints(positions, "positions", n), tp, ts, cols, batch)
        self._check(self._lib.gawee_kv_append(self._h, a, _stream_ptr(stream)))

    def attend(self, k_pages, v_pages, q, block_table, lengths, out, scale: Optional[float] = None, k=None, v=None,
               mask=None, weights=None, weights_out=None, stream=None):
        """Attention of one new token per sequence, q [batch, heads, head_dim],
        over its cached rows, into `out`; returns `out`.

        scale: of the scores (None: 1 / sqrt(head_dim)).
        k, v [batch, kv_heads, head_dim]: the new token's rows, first stored as row length - 1.
        mask f32 [batch or 1, columns]: added to the scaled scores; -inf takes a row out.
        weights, weights_out f32 [batch, kv_heads, columns]: weights_out = weights
            (None: 0) + the attention weights of this token; may be one array."""
        batch = q.shape[0]
        code = _code(q)
        qp, qs = self._rows(q, "q", batch, self.heads, None)
        op, os_ = self._rows(out, "out", batch, self.heads, code)
        tp, ts, rows, cols = self._table(block_table, "block_table")
        if rows != batch:
            raise _invalid(f"block_table has {rows} rows, q has {batch}")
        kp = vp = mp = wp = wop = 0
        ks = vs = ms = mc = ws = wb = wos = wob = wc = 0
        if k is not None:
            kp, ks = self._rows(k, "k", batch, self.kv_heads, code)
        if v is not None:
            vp, vs = self._rows(v, "v", batch, self.kv_heads, code)
        if mask is not None:
            if len(mask.shape) != 2 or mask.shape[0] not in (1, batch) or mask.shape[1] < 1 or (mask.shape[1] > 1 and mask.stride()[1] != 1):
                raise _invalid(f"mask must be f32 [{batch} or 1, columns] with dense rows, got shape {tuple(mask.shape)}")
            mp, mc = self._on_device(mask, "mask", 0), mask.shape[1]
            ms = mask.stride()[0] if mask.shape[0] > 1 else 0
        if weights_out is not None:
            wop, wos, wob, wc = self._weights(weights_out, "weights_out", batch)
        if weights is not None:
            wp, ws, wb, c = self._weights(weights, "weights", batch)
            if weights_out is not None and c != wc:
                raise _invalid(f"weights has {c} columns, weights_out {wc}")
        try:
            a = _ATTEND.pack(self._pages(k_pages, "k_pages"), self._pages(v_pages, "v_pages"), qp, op, code, qs, os_,
                             batch, self.head_dim ** -0.5 if scale is None else scale, tp, ts, cols,
                             self._ints(lengths, "lengths", batch), kp, vp, ks, vs, mp, ms, mc, wp, ws, wb, wop, wos,
                             wob, wc)
        except (struct.error, OverflowError) as e:  # a value that its C type cannot hold
            raise _invalid(f"scale is {scale!r}: {e}") from None
        self._check(self._lib.gawee_kv_attend(self._h, a, _stream_ptr(stream)))
        return out

    def evict(self, k_pages, v_pages, weights, block_table, lengths, budget: int, recent: int, kept, weights_out,
              lengths_out, to_table=None, stream=None):
        """Cut sequences longer than `budget` to it: per key/value head the last
        `recent` rows and those of the greatest weight stay and are packed, in
        order, into the first rows of the sequence's pages, or of the pages of
        `to_table`.  kept int32 [batch, kv_heads, budget] receives their earlier
        positions; weights_out may be `weights` and lengths_out `lengths`."""
        tp, ts, batch, cols = self._table(block_table, "block_table")
        wp, ws, wb, wc = self._weights(weights, "weights", batch)
        wop, wos, wob, c = self._weights(weights_out, "weights_out", batch)
        if c != wc:
            raise _invalid(f"weights has {wc} columns, weights_out {c}")
        if kept.shape != (batch, self.kv_heads, budget) or not kept.is_contiguous():
            raise _invalid(f"kept must be dense int32 {(batch, self.kv_heads, budget)}, got shape {tuple(kept.shape)}")
        if not 0 <= recent <= budget:
            raise _invalid(f"recent is {recent}, outside 0 .. {budget}")
        top = tos = toc = 0
        if to_table is not None:
            top, tos, rows, toc = self._table(to_table, "to_table")
            if rows != batch:
                raise _invalid(f"to_table has {rows} rows, block_table {batch}")
        try:
            a = _EVICT.pack(self._pages(k_pages, "k_pages"), self._pages(v_pages, "v_pages"), wp, ws, wb, wop, wos, wob,
                            wc, batch, tp, ts, cols, top, tos, toc, self._ints(lengths, "lengths", batch),
                            self._ints(lengths_out, "lengths_out", batch), budget, recent,
                            self._on_device(kept, "kept", 4))
        except struct.error as e:
            raise _invalid(f"budget is {budget!r}, recent {recent!r}: {e}") from None
        self._check(self._lib.gawee_kv_evict(self._h, a, _stream_ptr(stream)))

    def synchronize(self, stream=None):
        """Wait for `stream` and raise what a call found wrong on the device since the last check."""
        self._check(self._lib.gawee_kv_synchronize(self._h, _stream_ptr(stream)))
