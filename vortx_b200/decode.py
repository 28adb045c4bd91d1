"""What a decode step does besides its projections, on block-quantised data: a cache of keys and values that is
quantised as it is written (vx_kv_*), attention of new or drafted tokens over it (vx_kv_attention), and a
mixture-of-experts layer (vx_moe).  vortx has no counterpart; the calls take the shape of Gemv.dispatch
(backend, pass, outputs, inputs).  Tensors, views, buffers and plain device pointers are accepted alike; a view with
gaps between its rows needs the call's stride argument, where it has one.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from . import _lib
from .backend import Backend, GpuBuffer, GpuPass
from .linalg import QuantizedMatrix, _ptr_len


_F32, _I32, _U32 = (np.dtype(t) for t in (np.float32, np.int32, np.uint32))
_WORDS = (_I32, _U32)


def _check_len(what: str, length: Optional[int], rows: int, stride: int, width: int) -> None:
    if stride < 0:
        raise ValueError(f"the stride of {what} must not be negative")
    if length is not None and rows and (rows - 1) * stride + width > length:
        raise IndexError(f"{what} is shorter than {rows} rows")


def _dense(view, width: Optional[int]) -> bool:
    """Whether a view's elements are next to each other: all of them, or those of each row of `width` elements."""
    below = 1
    for i in range(view.rank() - 1, -1, -1):
        if width is not None and below >= width:
            break
        if view.size(i) > 1 and view.stride(i) != below:
            return False
        below *= view.size(i)
    return True


def _typed(what: str, t, dtypes, width: Optional[int] = None) -> tuple:
    """Device pointer and length of t.  Where the element type is known it must be one of dtypes.  A view must be dense; if the
    call says how far apart its rows of `width` elements are, only these.  A buffer must not have been freed: its
    address is zero then, which would mean an argument that is not given, and a view's is one near it."""
    if type(t) is GpuBuffer:                                # these calls cost as much on the host as on the device
        if t.dtype in dtypes and t.ptr:
            return t.ptr, t._len
        buf = t
    elif hasattr(t, "as_tensor_ref"):
        view = t.as_tensor_ref()
        buf = view.raw_buffer()
        if not _dense(view, width):
            raise ValueError(f"{what}: the {'rows' if width else 'elements'} of the view must be dense")
    else:
        return _ptr_len(t)
    if buf.dtype not in dtypes:
        raise TypeError(f"{what} must hold {dtypes[0].name} elements, not {buf.dtype.name}")
    if not buf.ptr and buf._len:
        raise ValueError(f"{what} has been freed")
    return _ptr_len(t)


class _Pointer:
    """In place of a buffer where a plain pointer was given: nobody knows whether it is still good."""

    ptr = 1


def _buffer_of(t):
    buf = t if type(t) is GpuBuffer else t.as_tensor_ref().raw_buffer() if hasattr(t, "as_tensor_ref") else _Pointer
    return buf if buf.ptr else _Pointer                     # of no elements


class CacheRows:
    """Which tokens the rows of a call are (vx_kv_rows): row begin[s] + i is token start[s] + i of sequence s, whose token
    p lies in page table[s, p // page_tokens].  The arrays are int32 on the device (table [seqs, max_pages], begin
    [seqs + 1], start [seqs]) and are read when the call runs; `rows` is how many rows the call's tensors have.
    `seqs` and `max_pages` follow from the lengths unless plain pointers are given.  Pointers are captured at
    construction; calls after one of the buffers has been freed are refused."""

    def __init__(self, table, begin, start, rows: int, seqs: Optional[int] = None, max_pages: Optional[int] = None):
        (tp, tl), (bp, bl), (sp, sl) = (_typed(n, t, _WORDS) for n, t in (("table", table), ("begin", begin), ("start", start)))
        if seqs is None:
            if sl is None:
                raise ValueError("seqs is needed with a plain pointer")
            seqs = sl
        given = max_pages is not None
        if max_pages is None:
            if tl is None:
                raise ValueError("max_pages is needed with a plain pointer")
            max_pages = tl // seqs if seqs else 0
        if (tl is not None and tl < seqs * max_pages) or (bl is not None and seqs and bl < seqs + 1) or (sl is not None and sl < seqs):
            raise IndexError("table, begin or start is shorter than the sequences need")
        if not given and seqs > 0 and tl % seqs:
            raise ValueError("the table does not have the same number of pages for every sequence")
        if rows < 0 or seqs < 0 or max_pages < 0:
            raise ValueError("rows, seqs and max_pages must not be negative")
        self.rows, self.seqs, self.max_pages = rows, seqs, max_pages
        self._keep = (table, begin, start)
        self._buffers = _buffer_of(table), _buffer_of(begin), _buffer_of(start)
        self._c = _lib.VxKvRows(tp or None, max_pages, bp or None, sp or None, seqs, rows)
        self._pointer = C.byref(self._c)

    @property
    def _ref(self):
        table, begin, start = self._buffers
        if not (table.ptr and begin.ptr and start.ptr):
            raise ValueError("the rows' table, begin or start has been freed")
        return self._pointer


class QuantizedCache:
    """Keys and values in Q8_0 / Q4_0 blocks on the device (vx_kv_cache): `pages` pages of `page_tokens` tokens."""

    def __init__(self, backend: Backend, k_type: int, v_type: int, heads: int, head_dim: int, pages: int, page_tokens: int = 64):
        for name, v in (("heads", heads), ("head_dim", head_dim), ("pages", pages), ("page_tokens", page_tokens)):
            if v < 0:
                raise ValueError(f"{name} must not be negative")
        self._h = None
        h = C.c_void_p()
        _lib.check(_lib.load().vx_kv_cache_create(backend._ctx, k_type, v_type, heads, head_dim, pages, page_tokens, C.byref(h)))
        self.backend, self._h = backend, h
        self.k_type, self.v_type, self.heads, self.head_dim = k_type, v_type, heads, head_dim
        self.pages, self.page_tokens, self.width = pages, page_tokens, heads * head_dim

    def device_bytes(self) -> int:
        n = C.c_size_t()
        _lib.check(_lib.load().vx_kv_cache_info(self._h, None, None, None, None, None, None, C.byref(n)))
        return int(n.value)

    def _rows_of(self, what: str, t, rows: CacheRows, stride: Optional[int]):
        apart, stride = stride is not None, self.width if stride is None else stride
        if t is None:
            return None, stride
        p, n = _typed(what, t, (_F32,), self.width if apart else None)
        _check_len(what, n, rows.rows, stride, self.width)
        return p, stride

    def append(self, pass_: Optional[GpuPass], k, v, rows: CacheRows, k_stride: Optional[int] = None,
               v_stride: Optional[int] = None, backend: Optional[Backend] = None) -> None:
        """Quantises the rows of k and v (heads * head_dim f32 each) into their places."""
        kp, ks = self._rows_of("k", k, rows, k_stride)
        vp, vs = self._rows_of("v", v, rows, v_stride)
        _lib.check(_lib.load().vx_kv_append((backend or self.backend)._ctx, self._h, rows._ref, kp, ks, vp, vs))

    def read(self, pass_: Optional[GpuPass], k, v, rows: CacheRows, k_stride: Optional[int] = None,
             v_stride: Optional[int] = None, backend: Optional[Backend] = None) -> None:
        """The reverse: k and / or v (None: not wanted) receive the values that the codes stand for."""
        kp, ks = self._rows_of("k", k, rows, k_stride)
        vp, vs = self._rows_of("v", v, rows, v_stride)
        _lib.check(_lib.load().vx_kv_read((backend or self.backend)._ctx, self._h, rows._ref, kp, ks, vp, vs))

    def free(self) -> None:
        if self._h and self.backend._ctx:
            _lib.check(_lib.load().vx_kv_cache_free(self.backend._ctx, self._h))
        self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def tree_mask(parents: Sequence[int]) -> np.ndarray:
    """The mask of a tree of drafted tokens: parents[i] < i is the token that i continues, or -1; row i of the result
    (uint32 [n, ceil(n / 32)]) has the bits of i and its ancestors."""
    n = len(parents)
    may = np.zeros((n, -(-n // 32) * 32), np.uint8)
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"token {i} cannot continue token {p}")
        if p >= 0:
            may[i] = may[p]
        may[i, i] = 1
    return np.packbits(may, axis=1, bitorder="little").view("<u4").astype(np.uint32)


class CacheAttention:
    """Attention over a QuantizedCache (vx_kv_attention); holds the workspace of its calls, of up to `max_seqs` sequences each.
    `heads` query heads share the cache's heads evenly."""

    def __init__(self, backend: Backend, cache: QuantizedCache, heads: int, max_seqs: int):
        if heads < 0 or max_seqs < 0:
            raise ValueError("heads and max_seqs must not be negative")
        self._h = None
        if not cache._h:
            raise ValueError("the cache has been freed")
        h = C.c_void_p()
        _lib.check(_lib.load().vx_kv_attention_create(backend._ctx, cache._h, heads, max_seqs, C.byref(h)))
        self.backend, self.cache, self.heads, self.max_seqs, self._h = backend, cache, heads, max_seqs, h
        self.width = heads * cache.head_dim

    def dispatch(self, backend: Backend, pass_: Optional[GpuPass], out, q, rows: CacheRows, scale: Optional[float] = None, mask=None,
                 mask_words: Optional[int] = None, q_stride: Optional[int] = None, out_stride: Optional[int] = None) -> None:
        """out[r, h] = attention of q[r, h] over the tokens before the call's and, among the call's own (already appended),
        those whose bits its row of `mask` (32-bit words, mask_words a row) has set; mask None: those up to itself.
        scale defaults to 1 / sqrt(head_dim).  out may be q, with q's stride."""
        qs = self.width if q_stride is None else q_stride
        os = self.width if out_stride is None else out_stride
        qp, ql = _typed("q", q, (_F32,), None if q_stride is None else self.width)
        op, ol = _typed("out", out, (_F32,), None if out_stride is None else self.width)
        _check_len("q", ql, rows.rows, qs, self.width)
        _check_len("out", ol, rows.rows, os, self.width)
        mp, words = None, 0
        if mask is not None:
            mp, ml = _typed("mask", mask, _WORDS)
            if mask_words is None:
                if ml is None:
                    raise ValueError("mask_words is needed with a plain pointer")
                mask_words = ml // rows.rows if rows.rows else 1
                if mask_words and rows.rows and ml % rows.rows:
                    raise ValueError("the mask does not have the same number of words for every row")
            words = mask_words
            _check_len("mask", ml, rows.rows, words, words)
        if not self.cache._h:
            raise ValueError("the cache has been freed")
        s = self.cache.head_dim ** -0.5 if scale is None else scale
        _lib.check(_lib.load().vx_kv_attention_run(backend._ctx, self._h, rows._ref, qp, qs, op, os, s, mp, words))

    def free(self) -> None:
        if self._h and self.backend._ctx:
            _lib.check(_lib.load().vx_kv_attention_free(self.backend._ctx, self._h))
        self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class MoeLayer:
    """A routed layer of gated experts on block-quantised weights (vx_moe).  router: f32 [experts, hidden] on the device;
    gate, up: the experts' matrices one below the other (experts * inner rows, hidden columns); down: experts * hidden
    rows, inner columns."""

    def __init__(self, backend: Backend, router, gate: QuantizedMatrix, up: QuantizedMatrix, down: QuantizedMatrix, experts: int,
                 top_k: int, normalise: bool = True, max_tokens: int = 32):
        if experts < 0 or top_k < 0 or max_tokens < 0:
            raise ValueError("experts, top_k and max_tokens must not be negative")
        self._h = None
        rp, rl = _typed("router", router, (_F32,))
        if rl is not None and rl < experts * gate.cols:
            raise IndexError("router is shorter than experts * hidden")
        h = C.c_void_p()
        _lib.check(_lib.load().vx_moe_create(backend._ctx, rp, experts, gate._h, up._h, down._h, top_k, int(bool(normalise)), max_tokens,
                                             C.byref(h)))
        self.backend, self._h = backend, h
        self._router_buffer = router if type(router) is GpuBuffer else router.as_tensor_ref().raw_buffer() if hasattr(router, "as_tensor_ref") else None
        self._router, self._gate, self._up, self._down = router, gate, up, down  # read by every call
        self.experts, self.top_k, self.hidden, self.inner, self.max_tokens = experts, top_k, gate.cols, down.cols, max_tokens

    def dispatch(self, backend: Backend, pass_: Optional[GpuPass], y, x, tokens: int = 1, x_stride: Optional[int] = None,
                 y_stride: Optional[int] = None, ids=None, weights=None) -> None:
        """y[t] = the layer's output for x[t], t < tokens; ids (int32) and weights (f32), both [tokens, top_k] and optional, receive
        the chosen experts, best first, and what their outputs were weighted with.  y may be x or overlap it."""
        if tokens < 0:
            raise ValueError("tokens must not be negative")
        if not (self._gate._h and self._up._h and self._down._h) or (self._router_buffer is not None and not self._router_buffer.ptr):
            raise ValueError("the layer's weights have been freed")
        xs = self.hidden if x_stride is None else x_stride
        ys = self.hidden if y_stride is None else y_stride
        xp, xl = _typed("x", x, (_F32,), None if x_stride is None else self.hidden)
        yp, yl = _typed("y", y, (_F32,), None if y_stride is None else self.hidden)
        _check_len("x", xl, tokens, xs, self.hidden)
        _check_len("y", yl, tokens, ys, self.hidden)
        ip = wp = None
        if ids is not None:
            ip, n = _typed("ids", ids, _WORDS)
            _check_len("ids", n, tokens, self.top_k, self.top_k)
        if weights is not None:
            wp, n = _typed("weights", weights, (_F32,))
            _check_len("weights", n, tokens, self.top_k, self.top_k)
        _lib.check(_lib.load().vx_moe_run(backend._ctx, self._h, xp, xs, yp, ys, tokens, ip, wp))

    def free(self) -> None:
        if self._h and self.backend._ctx:
            _lib.check(_lib.load().vx_moe_free(self.backend._ctx, self._h))
        self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
