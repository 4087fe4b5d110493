"""Operators on rows of vocabulary logits: a teacher's top logits, distillation from them, and the verification of
drafted tokens (no counterpart in the reference, whose loss is the labels' cross-entropy).

``top_logits(logits, k)`` keeps of each row what a teacher's answer needs: the ``k`` largest logits and the
log-sum-exp of the others, a ``Teacher``.  ``distill(logits, teacher, ...)`` is the student's side: the divergence
from the teacher, mixed with the labels' cross-entropy, and its gradient.  ``verify_draft(...)`` accepts or rejects
tokens that a draft model (a distilled student, say) proposed, such that what comes out is distributed as the
target's samples.

Rows are numpy arrays of float32 or float16 (bfloat16: its bits in uint16 arrays, with ``type=TYPE_BF16``); a row may be longer
apart than it is long (a view ``a[:, :vocab]``).  ``head_top_logits`` and ``head_distill`` take the rows from an LM head
(``GpuModel.top_logits``, ``forward_backward_distill`` and ``verify_draft`` from a whole model).  The ``_d`` variants take device addresses and a stream and only enqueue.
"""
from __future__ import annotations

import ctypes
import dataclasses

import numpy as np

from . import _ffi
from .frozen import Context, HipFrozen, default_context


@dataclasses.dataclass
class Teacher:
    """A teacher's top logits: ``ids`` and ``vals`` [n x k] (ids below 0: empty slots), ``rest`` [n] the log of
    the sum of exp(logit / temperature) over its other tokens, or None."""
    ids: np.ndarray
    vals: np.ndarray
    rest: np.ndarray | None = None
    temperature: float = 1.0

    def _view(self, n: int) -> _ffi.RtqTeacher:
        self.ids = np.ascontiguousarray(self.ids, dtype=np.int32)
        self.vals = np.ascontiguousarray(self.vals, dtype=np.float32)
        assert self.ids.ndim == 2 and self.ids.shape[0] == n, "one list of teacher tokens per row"
        assert self.vals.shape == self.ids.shape, "one logit per teacher token"
        if self.rest is not None:
            self.rest = np.ascontiguousarray(self.rest, dtype=np.float32).reshape(-1)
            assert self.rest.size == n, "one rest per row"
        return _ffi.RtqTeacher(self.ids.shape[1], self.ids.ctypes.data, self.vals.ctypes.data,
                               None if self.rest is None else self.rest.ctypes.data, self.temperature)


def _rows(a, type: int | None, what: str) -> tuple[np.ndarray, int, int]:
    """(array, type id, row stride in elements) of [n x vocab] logits."""
    a = np.asarray(a)
    assert a.ndim == 2, f"{what}: expected rows of logits"
    if type is None:
        type = {np.dtype(np.float32): _ffi.TYPE_F32, np.dtype(np.float16): _ffi.TYPE_F16}.get(a.dtype)
        assert type is not None, f"{what}: {a.dtype} logits"
    own = {_ffi.TYPE_F32: np.float32, _ffi.TYPE_F16: np.float16}.get(type)
    bits = type != _ffi.TYPE_F32 and a.dtype.itemsize == 2 and a.dtype.kind != "f"  # 16-bit types as integers
    assert a.dtype.isnative and (a.dtype.type is own or bits), f"{what}: {a.dtype} is not of the given type"
    if a.size and (a.strides[1] != a.itemsize or (a.shape[0] > 1 and (a.strides[0] % a.itemsize or a.strides[0] < a.shape[1] * a.itemsize))):
        a = np.ascontiguousarray(a)
    return a, type, a.strides[0] // a.itemsize if a.shape[0] > 1 else a.shape[1]


def _per_row(a, dtype, n: int, what: str) -> np.ndarray | None:
    a = None if a is None else np.ascontiguousarray(a, dtype=dtype).reshape(-1)
    assert a is None or a.size == n, f"one {what} per row"
    return a


def _addr(a) -> int | None:
    return None if a is None else a.ctypes.data


def top_logits(logits, k: int, temperature: float = 1.0, type: int | None = None, ctx: Context | None = None) -> Teacher:
    """The ``k`` largest logits of each row, largest first (equal ones by the lower id), and the rest's log-sum-exp."""
    a, ty, ld = _rows(logits, type, "top_logits")
    n = a.shape[0]
    vals, ids, rest = np.empty((n, k), np.float32), np.empty((n, k), np.int32), np.empty(n, np.float32)
    _ffi.check(_ffi.lib().rtq_top_logits((ctx or default_context()).handle, a.ctypes.data, ty, n, a.shape[1], ld, k, temperature,
                                         vals.ctypes.data, ids.ctypes.data, rest.ctypes.data), "rtq_top_logits")
    return Teacher(ids, vals, rest, temperature)


def distill(logits, teacher: Teacher, labels=None, weights=None, hard: float = 0.0, type: int | None = None,
            ctx: Context | None = None) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """``(kl, logp, dlogits)`` of student rows: the divergence from the teacher at its temperature, the labels'
    log-probabilities (empty without ``labels``) and, with ``weights``, the gradient of
    ``sum w ((1 - hard) T^2 kl - hard logp)`` in the logits' type (empty without)."""
    a, ty, ld = _rows(logits, type, "distill")
    n, vocab = a.shape
    view = teacher._view(n)
    tok, w = _per_row(labels, np.int32, n, "label"), _per_row(weights, np.float32, n, "weight")
    kl = np.empty(n, np.float32)
    logp = None if tok is None else np.empty(n, np.float32)
    dz = None if w is None else np.empty((n, vocab), a.dtype)
    _ffi.check(_ffi.lib().rtq_distill((ctx or default_context()).handle, a.ctypes.data, ty, n, vocab, ld, ctypes.byref(view), _addr(tok),
                                      _addr(w), hard, kl.ctypes.data, _addr(logp), _addr(dz), vocab), "rtq_distill")
    return kl, np.empty(0, np.float32) if logp is None else logp, np.empty((0, vocab), a.dtype) if dz is None else dz


def verify_draft(logits, drafted, uniforms=None, draft=None, lens=None, temperature: float = 1.0, type: int | None = None,
                 ctx: Context | None = None) -> tuple[np.ndarray, np.ndarray]:
    """``(accepted, tokens)`` for ``drafted`` [b x d]: how many of each sequence's drafted tokens the target
    accepts, and [b x (d + 1)] the accepted ones, the token drawn after them, -1 beyond.  ``logits`` are the
    target's [b (d + 1) x vocab], ``draft`` the rows the tokens were drawn from ([b d x vocab]; None: all
    probability on the drafted token), ``uniforms`` [b x (d + 1)] in [0, 1) (not needed at temperature 0)."""
    x = np.ascontiguousarray(drafted, dtype=np.int32)
    assert x.ndim == 2, "drafted: [b x d]"
    b, d = x.shape
    a, ty, ld = _rows(logits, type, "verify_draft")
    assert a.shape[0] == b * (d + 1), "d + 1 target rows per sequence"
    q, ldq = None, 0
    if draft is not None:
        q, tq, ldq = _rows(draft, type, "verify_draft")
        assert tq == ty, "target and draft logits are of one type"
        assert q.shape == (b * d, a.shape[1]), "d draft rows per sequence, of the target's vocabulary"
    u = None if uniforms is None else np.ascontiguousarray(uniforms, dtype=np.float32)
    assert u is None or u.shape == (b, d + 1), "uniforms: [b x (d + 1)]"
    n = None if lens is None else np.ascontiguousarray(lens, dtype=np.int32).reshape(-1)
    assert n is None or n.size == b, "one length per sequence"
    accepted, tokens = np.empty(b, np.int32), np.empty((b, d + 1), np.int32)
    _ffi.check(_ffi.lib().rtq_verify_draft((ctx or default_context()).handle, a.ctypes.data, ty, ld, _addr(q), ldq, b, d, a.shape[1],
                                           x.ctypes.data, _addr(n), _addr(u), temperature, accepted.ctypes.data,
                                           tokens.ctypes.data), "rtq_verify_draft")
    return accepted, tokens


def _head(lm_head: HipFrozen, final_norm, x, positions) -> tuple[np.ndarray, np.ndarray, np.ndarray, int]:
    d = lm_head.in_dim()
    x = np.ascontiguousarray(x, dtype=np.float32).reshape(-1)
    assert x.size % d == 0, "x is not a whole number of rows"
    norm = np.ascontiguousarray(final_norm, dtype=np.float32)
    assert norm.size == d, "final_norm length != hidden size"
    return norm, x, np.ascontiguousarray(positions, dtype=np.int32).reshape(-1), x.size // d


def head_top_logits(lm_head: HipFrozen, final_norm, x, positions, k: int, temperature: float = 1.0, eps: float = 1e-6,
                    offset: float = 0.0) -> Teacher:
    """``top_logits`` of the LM head's logits at ``positions`` of the [t x d] hidden states ``x`` (as ``head`` forms them)."""
    norm, x, pos, t = _head(lm_head, final_norm, x, positions)
    n = pos.size
    vals, ids, rest = np.empty((n, k), np.float32), np.empty((n, k), np.int32), np.empty(n, np.float32)
    _ffi.check(_ffi.lib().rtq_lm_top_logits(lm_head.ctx.handle, lm_head.handle, norm.ctypes.data, eps, offset, x.ctypes.data, t,
                                            pos.ctypes.data, n, k, temperature, vals.ctypes.data, ids.ctypes.data,
                                            rest.ctypes.data), "rtq_lm_top_logits")
    return Teacher(ids, vals, rest, temperature)


def head_distill(lm_head: HipFrozen, final_norm, x, positions, teacher: Teacher, labels=None, weights=None, hard: float = 0.0,
                 eps: float = 1e-6, offset: float = 0.0) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """``(kl, logp, dx)``: ``distill`` of the LM head's logits at ``positions``, with ``weights`` the gradient to the
    hidden states ``x`` (zero rows outside ``positions``; empty without weights)."""
    norm, x, pos, t = _head(lm_head, final_norm, x, positions)
    n = pos.size
    view = teacher._view(n)
    tok, w = _per_row(labels, np.int32, n, "label"), _per_row(weights, np.float32, n, "weight")
    kl, logp = np.empty(n, np.float32), None if tok is None else np.empty(n, np.float32)
    dx = None if w is None else np.empty(x.size, np.float32)
    _ffi.check(_ffi.lib().rtq_lm_distill(lm_head.ctx.handle, lm_head.handle, norm.ctypes.data, eps, offset, x.ctypes.data, t,
                                         pos.ctypes.data, _addr(tok), _addr(w), n, ctypes.byref(view), hard, kl.ctypes.data,
                                         _addr(logp), _addr(dx)), "rtq_lm_distill")
    return kl, np.empty(0, np.float32) if logp is None else logp, np.empty(0, np.float32) if dx is None else dx


# ---- device-pointer variants (ints are device addresses, 0: none; stream 0 = the HIP null stream)
def top_logits_d(ctx: Context, logits_ptr: int, type: int, n: int, vocab: int, ld: int, k: int, vals_ptr: int, ids_ptr: int,
                 rest_ptr: int = 0, temperature: float = 1.0, stream: int = 0) -> None:
    _ffi.check(_ffi.lib().rtq_top_logits_d(ctx.handle, logits_ptr, type, n, vocab, ld, k, temperature, vals_ptr, ids_ptr,
                                           rest_ptr or None, stream or None), "rtq_top_logits_d")


def teacher_d(k: int, ids_ptr: int, vals_ptr: int, rest_ptr: int = 0, temperature: float = 1.0) -> _ffi.RtqTeacher:
    """A teacher's top logits in device memory, for ``distill_d`` (the memory stays the caller's)."""
    return _ffi.RtqTeacher(k, ids_ptr, vals_ptr, rest_ptr or None, temperature)


def distill_d(ctx: Context, logits_ptr: int, type: int, n: int, vocab: int, ld: int, teacher: _ffi.RtqTeacher, tok_ptr: int,
              weights_ptr: int, kl_ptr: int, logp_ptr: int, dlogits_ptr: int, ldd: int, hard: float = 0.0,
              stream: int = 0) -> None:
    _ffi.check(_ffi.lib().rtq_distill_d(ctx.handle, logits_ptr, type, n, vocab, ld, ctypes.byref(teacher), tok_ptr or None,
                                        weights_ptr or None, hard, kl_ptr, logp_ptr or None, dlogits_ptr or None, ldd,
                                        stream or None), "rtq_distill_d")


def verify_draft_d(ctx: Context, logits_ptr: int, type: int, ld: int, draft_ptr: int, ldq: int, b: int, d: int, vocab: int,
                   drafted_ptr: int, lens_ptr: int, uniforms_ptr: int, accepted_ptr: int, tokens_ptr: int,
                   temperature: float = 1.0, stream: int = 0) -> None:
    _ffi.check(_ffi.lib().rtq_verify_draft_d(ctx.handle, logits_ptr, type, ld, draft_ptr or None, ldq, b, d, vocab, drafted_ptr,
                                             lens_ptr or None, uniforms_ptr or None, temperature, accepted_ptr, tokens_ptr,
                                             stream or None), "rtq_verify_draft_d")
