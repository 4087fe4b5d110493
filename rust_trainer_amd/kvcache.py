"""A paged cache of keys and values and the operators on it (no counterpart in the reference, which trains and scores
whole sequences): appending new tokens with the rotation of their positions, attention of runs and of drafted
trees of new tokens over what is cached, and keeping a tree's accepted tokens.

``KvCache`` owns the pages of every layer on the device (or wraps the caller's).  A call names its sequences with
``Seqs``: the tokens that each holds, its pages, and how many of the call's rows are its own.  The host methods take numpy
rows of float32, float16 or (their bits as uint16, with ``type=TYPE_BF16``) bfloat16; the ``_d`` methods take device
addresses and a stream and only enqueue.  ``GpuModel.extend`` runs a whole model over a cache.
"""
from __future__ import annotations

import ctypes
import dataclasses

import numpy as np

from . import _ffi
from .distill import _addr, _rows
from .frozen import Context, default_context


@dataclasses.dataclass
class Seqs:
    """The sequences of a call: ``lens`` [b] tokens held, ``table`` [b x pages] page ids, ``starts`` [b + 1] the rows of
    each one's new tokens (None: as many for each)."""
    lens: np.ndarray
    table: np.ndarray
    starts: np.ndarray | None = None

    def _view(self) -> _ffi.RtqKvSeqs:
        self.lens = np.ascontiguousarray(self.lens, dtype=np.int32).reshape(-1)
        self.table = np.ascontiguousarray(self.table, dtype=np.int32)
        b = self.lens.size
        assert self.table.ndim == 2 and self.table.shape[0] == b, "one table row per sequence"
        if self.starts is not None:
            self.starts = np.ascontiguousarray(self.starts, dtype=np.int32).reshape(-1)
            assert self.starts.size == b + 1, "starts: one per sequence, and the end"
        return _ffi.RtqKvSeqs(b, self.lens.ctypes.data, _addr(self.starts), self.table.ctypes.data, self.table.shape[1])


@dataclasses.dataclass
class Rope:
    """The rotation of the heads' first ``dim`` elements, after an optional RMS norm of each head (``q_norm``, ``k_norm``)."""
    dim: int
    base: float = 10000.0
    neox: bool = True
    freq_scale: float = 1.0
    factors: np.ndarray | None = None
    q_norm: np.ndarray | None = None
    k_norm: np.ndarray | None = None
    eps: float = 1e-6
    offset: float = 0.0

    def _view(self, head_dim: int) -> _ffi.RtqRope:
        for n in ("factors", "q_norm", "k_norm"):
            a = getattr(self, n)
            if a is not None:
                setattr(self, n, np.ascontiguousarray(a, dtype=np.float32).reshape(-1))
        for w in (self.q_norm, self.k_norm):
            assert w is None or w.size == head_dim, "one norm weight per element of a head"
        return _ffi.RtqRope(self.dim, self.base, self.freq_scale, int(self.neox), _addr(self.factors),
                            0 if self.factors is None else self.factors.size, _addr(self.q_norm), _addr(self.k_norm), self.eps, self.offset)


def seqs_d(b: int, lens_ptr: int, table_ptr: int, ld: int, starts_ptr: int = 0) -> _ffi.RtqKvSeqs:
    """Sequences whose lists are in device memory, for the ``_d`` methods (the memory stays the caller's)."""
    return _ffi.RtqKvSeqs(b, lens_ptr, starts_ptr or None, table_ptr, ld)


def rope_d(dim: int, base: float = 10000.0, neox: bool = True, freq_scale: float = 1.0, factors=None, q_norm_ptr: int = 0, k_norm_ptr: int = 0,
           eps: float = 1e-6, offset: float = 0.0) -> _ffi.RtqRope:
    """A rotation for the ``_d`` methods: the norms' weights in device memory, the frequency factors on the host."""
    f = None if factors is None else np.ascontiguousarray(factors, dtype=np.float32).reshape(-1)
    r = _ffi.RtqRope(dim, base, freq_scale, int(neox), _addr(f), 0 if f is None else f.size, q_norm_ptr or None, k_norm_ptr or None, eps, offset)
    r._keep = f
    return r


class KvCache:
    """``n_pages`` pages of ``page_size`` slots for each of ``n_layer`` layers, ``type`` TYPE_F16 or TYPE_BF16.  ``pages_d``: the device
    addresses of the caller's keys [layer, page, head, slot, head_dim] and values [layer, page, head, head_dim, slot]."""

    def __init__(self, n_layer: int, n_pages: int, page_size: int, n_head_kv: int, head_dim: int, type: int = _ffi.TYPE_F16,
                 ctx: Context | None = None, pages_d: tuple[int, int] | None = None):
        self.ctx = ctx or default_context()
        self._h = None
        self.n_layer, self.n_pages, self.page_size, self.n_head_kv, self.head_dim, self.type = n_layer, n_pages, page_size, n_head_kv, head_dim, type
        k, v = pages_d or (None, None)
        h = ctypes.c_void_p()
        _ffi.check(_ffi.lib().rtq_kv_cache_create(self.ctx.handle, type, n_layer, n_pages, page_size, n_head_kv, head_dim, k, v, ctypes.byref(h)),
                   "rtq_kv_cache_create")
        self._h = h
        self.ctx._owned.add(self)

    @property
    def handle(self) -> ctypes.c_void_p:
        if self._h is None:
            raise RuntimeError("cache destroyed")
        return self._h

    def close(self) -> None:
        if getattr(self, "_h", None) is not None:
            _ffi.lib().rtq_kv_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def pages(self, layer: int = 0) -> tuple[int, int]:
        """Device addresses of a layer's keys and values."""
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        _ffi.check(_ffi.lib().rtq_kv_cache_pages(self.handle, layer, ctypes.byref(k), ctypes.byref(v)), "rtq_kv_cache_pages")
        return int(k.value), int(v.value)

    # ---- host arrays
    def append(self, layer: int, seqs: Seqs, k, v, rope: Rope, q=None, positions=None, type: int | None = None) -> np.ndarray | None:
        """The new tokens' keys (normed, rotated) and values enter the layer; returns the queries ``q`` normed and rotated."""
        ka, ty, ldk = _rows(k, type, "append")
        va, tv, ldv = _rows(v, type, "append")
        n, width = ka.shape[0], self.n_head_kv * self.head_dim
        assert ka.shape == va.shape == (n, width) and ty == tv, "k and v: one row of heads per new token, of one type"
        qa, ldq, nh, out = None, 0, 0, None
        if q is not None:
            qa, tq, ldq = _rows(q, type, "append")
            assert tq == ty and qa.shape[0] == n and qa.shape[1] % self.head_dim == 0, "q: a row of heads per new token, of the keys' type"
            nh = qa.shape[1] // self.head_dim
            out = np.zeros(qa.shape, qa.dtype)
        pos = None if positions is None else np.ascontiguousarray(positions, dtype=np.int32).reshape(-1)
        assert pos is None or pos.size == n, "one position per new token"
        sv, rv = seqs._view(), rope._view(self.head_dim)
        _ffi.check(_ffi.lib().rtq_kv_append(self.handle, layer, ctypes.byref(sv), n, ty, ctypes.byref(rv), _addr(pos), ka.ctypes.data, ldk,
                                            va.ctypes.data, ldv, nh, _addr(qa), ldq, _addr(out), 0 if out is None else out.shape[1]),
                   "rtq_kv_append")
        return out

    def attend(self, layer: int, seqs: Seqs, q, parents=None, scale: float = 0.0, type: int | None = None) -> np.ndarray:
        """Attention of the new tokens' queries (rotated) over the layer, which holds their keys and values already: over
        what is cached and, of the new tokens, those before (or, with ``parents``, a token's chain of parents) and itself."""
        qa, ty, ldq = _rows(q, type, "attend")
        n = qa.shape[0]
        assert qa.shape[1] % self.head_dim == 0, "q: whole heads"
        par = None if parents is None else np.ascontiguousarray(parents, dtype=np.int32).reshape(-1)
        assert par is None or par.size == n, "one parent per new token"
        out = np.zeros(qa.shape, qa.dtype)
        sv = seqs._view()
        _ffi.check(_ffi.lib().rtq_kv_attend(self.handle, layer, ctypes.byref(sv), n, ty, qa.shape[1] // self.head_dim, scale, _addr(par),
                                            qa.ctypes.data, ldq, out.ctypes.data, out.shape[1]), "rtq_kv_attend")
        return out

    def keep(self, seqs: Seqs, kept) -> np.ndarray:
        """Keeps the listed new tokens of each sequence (``kept``: lists of ascending indices) in every layer, right after the
        held ones; returns the lengths after it."""
        most = max([len(r) for r in kept] + [1])
        a = np.full((len(kept), most), -1, np.int32)
        for i, r in enumerate(kept):
            a[i, :len(r)] = r
        sv = seqs._view()
        assert len(kept) == sv.b, "one list per sequence"
        after = np.empty(sv.b, np.int32)
        _ffi.check(_ffi.lib().rtq_kv_keep(self.handle, ctypes.byref(sv), a.ctypes.data, most, after.ctypes.data), "rtq_kv_keep")
        return after

    # ---- device-pointer variants (ints are device addresses, 0: none; stream 0 = the HIP null stream)
    def append_d(self, layer: int, seqs: _ffi.RtqKvSeqs, n: int, type: int, rope: _ffi.RtqRope, k_ptr: int, ldk: int, v_ptr: int, ldv: int,
                 n_head: int = 0, q_ptr: int = 0, ldq: int = 0, q_out_ptr: int = 0, ldo: int = 0, positions_ptr: int = 0,
                 stream: int = 0) -> None:
        _ffi.check(_ffi.lib().rtq_kv_append_d(self.handle, layer, ctypes.byref(seqs), n, type, ctypes.byref(rope), positions_ptr or None, k_ptr, ldk,
                                              v_ptr, ldv, n_head, q_ptr or None, ldq, q_out_ptr or None, ldo, stream or None),
                   "rtq_kv_append_d")

    def attend_d(self, layer: int, seqs: _ffi.RtqKvSeqs, n: int, type: int, n_head: int, q_ptr: int, ldq: int, out_ptr: int, ldo: int,
                 parents_ptr: int = 0, scale: float = 0.0, stream: int = 0) -> None:
        _ffi.check(_ffi.lib().rtq_kv_attend_d(self.handle, layer, ctypes.byref(seqs), n, type, n_head, scale, parents_ptr or None, q_ptr, ldq,
                                              out_ptr, ldo, stream or None), "rtq_kv_attend_d")

    def keep_d(self, seqs: _ffi.RtqKvSeqs, kept_ptr: int, ldk: int, lens_out_ptr: int = 0, stream: int = 0) -> None:
        _ffi.check(_ffi.lib().rtq_kv_keep_d(self.handle, ctypes.byref(seqs), kept_ptr, ldk, lens_out_ptr or None, stream or None),
                   "rtq_kv_keep_d")
