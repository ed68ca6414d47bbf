"""Operators around a decoder's attention that the reference's graphs spell out in elementary ops, as single calls:

* ``QkNormRope``        RMS norm of every query and key head and their rotation (ApplyRope,
  transformers/src/ops/apply_rope.rs:169-176) in one pass
* ``SharedPrefixSdpa``  attention of sequences that share a prefix, which is read once for all of them;
  ``inplace_kv_sdpa_eval_shared`` is the same over caches, with the append of a step
* ``ScoredSdpa``        Sdpa (transformers/src/ops/sdpa.rs:83-89) whose scores are capped by a tanh, fall with the distance,
  stay inside documents or see a prefix

An object keeps its workspace from call to call: its calls follow each other on one stream.  A graph that recorded a call uses
that workspace: the object has to live as long as the graph, and later calls of other shapes leave it be.
"""
from __future__ import annotations

import ctypes as C
from array import array

import numpy as np

from ._lib import TractRocmError, call
from .ops import _as_device, _canon4, _check_norm_weights, _code, _cos_sin_batch, _same, _scale_arg, _strides4, _I64x3
from .runtime import DeviceTensor, Workspace, _sh

_PI64 = C.c_int64 * 1   # (where a row of lengths begins)
_I32 = np.dtype(np.int32)
_F32 = np.dtype(np.float32)


def _optr(t):
    return None if t is None else t.ptr


def _output(out, shape, dtype):
    if out is None:
        return DeviceTensor(shape, dtype)
    if out.shape != shape or not _same(out.dtype, dtype):
        raise TractRocmError("out must have Q's shape and datum type")
    return out


class _Scratch:
    """An operator's workspace.  It grows; what it outgrew is kept, since recorded graphs go on using it (at most as much again)."""

    def __init__(self):
        self._all = []

    def holding(self, need: int, stream) -> Workspace:
        ws = self._all[-1] if self._all else None
        if ws is None or ws.nbytes < need:
            ws = Workspace(0, 0, 0, 0, stream, nbytes=need if ws is None else max(need, 2 * ws.nbytes))
            self._all.append(ws)
        return ws


class QkNormRope:
    """y = x * rsqrt(mean(x^2) + eps) * weight, then y * cos + RotateHalf(y) * sin, for every head of Q and K."""

    def __init__(self, eps: float = 1e-6):
        self.eps = float(eps)
        self._last = (None, None)

    def name(self) -> str:
        return "QkNormRope"

    def is_stateless(self) -> bool:
        return True

    def output_facts(self, q_shape, k_shape, *_):
        return tuple(q_shape), tuple(k_shape)

    def eval(self, q, k, q_weight, k_weight, cos, sin, stream=None, q_strides=None, k_strides=None, q_out=None, k_out=None):
        """Q [batch, q_heads, n, head_dim], K [batch, kv_heads, n, head_dim], weights [head_dim] or None, Cos and Sin
        [1 or batch, 1, n, head_dim].  Strides: of views, in elements (None: dense).  Returns (q, k), dense."""
        if not isinstance(q, DeviceTensor):
            q, k, cos, sin = (_as_device(t, stream) for t in (q, k, cos, sin))
            q_weight, k_weight = (None if w is None else _as_device(w, stream) for w in (q_weight, k_weight))
        dtype, shape, k_shape = q.dtype, q.shape, k.shape
        # (A decode step's call takes the device 3.4 us: shapes and types are looked into where they are not the last call's.)
        key = (shape, k_shape, cos.shape, sin.shape, q_strides and tuple(q_strides), k_strides and tuple(k_strides), dtype, k.dtype, cos.dtype, sin.dtype,
               q_weight is None or (q_weight.shape, q_weight.dtype), k_weight is None or (k_weight.shape, k_weight.dtype))
        last_key, sizes = self._last   # (a pair, read once: another thread's call may put its own there)
        if key != last_key:
            for t in (k, q_weight, k_weight, cos, sin):
                if t is not None and not _same(t.dtype, dtype):
                    raise TractRocmError("Q, K, weights, cos and sin must share a datum type")
            if len(shape) != 4 or len(k_shape) != 4 or k_shape[0] != shape[0] or k_shape[2:] != shape[2:]:
                raise TractRocmError(f"Q {shape} and K {k_shape} must be [batch, heads, n, head_dim] and differ in heads only")
            b, hq, n, d = shape
            cb = _cos_sin_batch(cos, sin, b, n, d)
            _check_norm_weights(q_weight, k_weight, d)
            sizes = 0 if cb == 1 else n * d, _code(dtype), b, hq, k_shape[1], n, d, _strides4(q_strides), _strides4(k_strides)
            self._last = key, sizes
        if q_out is None or q_out.shape != shape or q_out.dtype is not dtype:
            q_out = _output(q_out, shape, dtype)
        if k_out is None or k_out.shape != k_shape or k_out.dtype is not dtype:
            k_out = _output(k_out, k_shape, dtype)
        call("trocm_qk_norm_rope", q.ptr, k.ptr, None if q_weight is None else q_weight.ptr, None if k_weight is None else k_weight.ptr, self.eps,
             cos.ptr, sin.ptr, *sizes, q_out.ptr, k_out.ptr, None if stream is None else _sh(stream))
        return q_out, k_out


class SharedPrefixSdpa:
    """Attention of n_seq sequences over one prefix and over their own keys behind it."""

    def __init__(self, scale=None, is_causal: bool = True):
        self.scale, self.is_causal = scale, bool(is_causal)
        self._scratch, self._last = _Scratch(), (None, None, None)

    def eval(self, q, prefix_k, prefix_v, k, v, lens, stream=None, out=None, prefix_len=None) -> DeviceTensor:
        """Q [n_seq, q_heads, q_len, head_dim]; prefix K and V [1, kv_heads, room, head_dim] of which `prefix_len` tokens (None:
        all) count; K and V [n_seq, kv_heads, room, head_dim] of which sequence i's first lens[i] tokens count."""
        if not isinstance(q, DeviceTensor):
            q, prefix_k, prefix_v, k, v = (_as_device(t, stream) for t in (q, prefix_k, prefix_v, k, v))
        dtype, shape = q.dtype, q.shape
        key = (shape, k.shape, v.shape, prefix_k.shape, prefix_v.shape, prefix_len, dtype, k.dtype, v.dtype, prefix_k.dtype, prefix_v.dtype)
        last_key, sizes, ws = self._last   # (read once: another thread's call may put its own there)
        if key != last_key:                # (the last call's need no second look)
            for t in (prefix_k, prefix_v, k, v):
                if not _same(t.dtype, dtype):
                    raise TractRocmError("Q, K and V must share a datum type")
            if len(shape) != 4 or len(k.shape) != 4 or len(prefix_k.shape) != 4 or k.shape != v.shape or prefix_k.shape != prefix_v.shape:
                raise TractRocmError("shared prefix: inputs must be of rank 4, K and V of one shape")
            n, hq, sq, d = shape
            _, hkv, room, _ = k.shape
            p_room = prefix_k.shape[2]
            p = p_room if prefix_len is None else int(prefix_len)
            if k.shape != (n, hkv, room, d) or prefix_k.shape != (1, hkv, p_room, d) or not 0 <= p <= p_room:
                raise TractRocmError(f"shared prefix: Q {shape}, prefix {prefix_k.shape} and K {k.shape} do not match")
            need = Workspace.shared_bytes_for(n, hq, sq, d)
            sizes, ws = ((_code(dtype), n, hq, hkv, sq, d), p, (C.c_int64 * 2)(p_room * d, d), _I64x3(hkv * room * d, room * d, d), need), self._scratch.holding(need, stream)
            self._last = key, sizes, ws
        sizes, p, prefix_strides, strides, need = sizes
        n, room = shape[0], k.shape[2]
        lens = array("q", lens)
        if len(lens) != n or (n and max(lens) > room):   # (negative ones are refused below)
            raise TractRocmError(f"shared prefix: lens must be {n} lengths of 0..={room}")
        if out is None or out.shape != shape or out.dtype is not dtype:
            out = _output(out, shape, dtype)
        call("trocm_sdpa_shared_prefix", q.ptr, *sizes, prefix_k.ptr, prefix_v.ptr, p, prefix_strides, k.ptr, v.ptr, strides,
             _PI64.from_buffer(lens) if n else _I64x3(0, 0, 0), out.ptr, _scale_arg(self.scale), int(self.is_causal), ws.buf.ptr, need,
             None if stream is None else _sh(stream))
        return out


def inplace_kv_sdpa_eval_shared(q: DeviceTensor, k_new, v_new, prefix_k, prefix_v, k_caches, v_caches, scale=None, causal: bool = True,
                                workspace: Workspace | None = None, stream=None, out: DeviceTensor | None = None) -> DeviceTensor:
    """One step of `n_seq` sequences that share a prefix: append k_new[i], v_new[i] ([n_seq, Hkv, n_new, D]) to sequence i's
    caches, then attend q[i] ([n_seq, Hq, n_new, D]) over the prefix caches and over its own.  With k_new and v_new None:
    attend to what is there.  A sequence's caches may be new; the prefix caches must have been pushed to."""
    if len(q.shape) != 4:
        raise TractRocmError("shared prefix: inputs must be of rank 4")
    n, hq, sq, d = q.shape
    if len(k_caches) != n or len(v_caches) != n:
        raise TractRocmError("shared prefix: one K and one V cache per sequence expected")
    if prefix_k.handle is None or prefix_v.handle is None:
        raise TractRocmError("empty kv-cache")
    _, hkv, _, cached_d = _canon4(prefix_k._shape)
    if d != cached_d:   # (all sizes of the call are taken from the caches)
        raise TractRocmError(f"shared prefix: Q {q.shape} is not of the prefix's head size {cached_d}")
    if k_new is not None or v_new is not None:
        if k_new is None or v_new is None or k_new.shape != (n, hkv, sq, d) or v_new.shape != k_new.shape:
            raise TractRocmError("shared prefix: k_new / v_new must be [n_seq, kv_heads, n_new, head_dim]")
        if not _same(k_new.dtype, q.dtype) or not _same(v_new.dtype, q.dtype):
            raise TractRocmError("Q, K_new and V_new must share a datum type")
    for c in (*k_caches, *v_caches):
        if c._h is None:
            c._create((1, hkv, 0, d), q.dtype)
    out = _output(out, q.shape, q.dtype)
    ws = workspace or Workspace(n, hq, sq, d, stream, nbytes=Workspace.shared_bytes_for(n, hq, sq, d))
    ks = (C.c_void_p * n)(*[c._h for c in k_caches])
    vs = (C.c_void_p * n)(*[c._h for c in v_caches])
    call("trocm_inplace_kv_sdpa_eval_shared", q.ptr, _optr(k_new), _optr(v_new), _code(q.dtype), hq, n, sq, prefix_k.handle, prefix_v.handle,
         ks, vs, out.ptr, _scale_arg(scale), int(causal), ws.ptr, ws.nbytes, _sh(stream))
    return out


class ScoredSdpa:
    """Sdpa whose scores are capped (softcap * tanh(s / softcap)), lose a slope per head times the distance, stay inside packed
    documents and, where causal, also see the first prefix_lens[b] keys."""

    def __init__(self, scale=None, softcap: float = 0.0, is_causal: bool = True):
        self.scale, self.softcap, self.is_causal = scale, float(softcap), bool(is_causal)
        self._scratch, self._last = _Scratch(), (None, None)

    def name(self) -> str:
        return "ScoredSdpa"

    @staticmethod
    def _rules(slopes, documents, prefix_lens, b, hq, sk, stream):
        slopes, documents, prefix_lens = (None if t is None else _as_device(t, stream) for t in (slopes, documents, prefix_lens))
        if slopes is not None and (slopes.shape != (hq,) or not _same(slopes.dtype, _F32)):
            raise TractRocmError(f"slopes must be f32 of shape [{hq}]")
        if documents is not None and (documents.shape != (b, sk) or not _same(documents.dtype, _I32)):
            raise TractRocmError(f"documents must be int32 of shape [{b}, {sk}]")
        if prefix_lens is not None and (prefix_lens.shape != (b,) or not _same(prefix_lens.dtype, _I32)):
            raise TractRocmError(f"prefix_lens must be int32 of shape [{b}]")
        return slopes, documents, prefix_lens

    def eval(self, q, k, v, slopes=None, documents=None, prefix_lens=None, stream=None, out=None) -> DeviceTensor:
        """Q, K, V of rank 3 or 4; slopes f32 [q_heads], documents int32 [batch, kv_len], prefix_lens int32 [batch]."""
        if not isinstance(q, DeviceTensor):
            q, k, v = (_as_device(t, stream) for t in (q, k, v))
        dtype, shape = q.dtype, q.shape
        key = (shape, k.shape, v.shape, dtype, k.dtype, v.dtype)
        last_key, sizes = self._last   # (read once: another thread's call may put its own there)
        if key != last_key:            # (the last call's need no second look)
            if not (_same(k.dtype, dtype) and _same(v.dtype, dtype)):
                raise TractRocmError("Q, K and V must share a datum type")
            b, hq, sq, d = _canon4(shape)
            _, hkv, sk, _ = _canon4(k.shape)
            if _canon4(k.shape) != (b, hkv, sk, d) or k.shape != v.shape:
                raise TractRocmError("K/V shape mismatch")
            sizes = _code(dtype), b, hq, hkv, sq, sk, d
            self._last = key, sizes
        _, b, hq, _, sq, sk, d = sizes
        if slopes is not None or documents is not None or prefix_lens is not None:
            slopes, documents, prefix_lens = self._rules(slopes, documents, prefix_lens, b, hq, sk, stream)
        if out is None or out.shape != shape or out.dtype is not dtype:
            out = _output(out, shape, dtype)
        need = Workspace.bytes_for(b, hq, sq, d)
        ws = self._scratch.holding(need, stream)
        call("trocm_sdpa_scored", q.ptr, k.ptr, v.ptr, out.ptr, *sizes, None, _scale_arg(self.scale), self.softcap, _optr(slopes), _optr(documents),
             _optr(prefix_lens), int(self.is_causal), ws.buf.ptr, need, None if stream is None else _sh(stream))
        return out

    def eval_cached(self, q: DeviceTensor, k_cache, v_cache, slopes=None, documents=None, prefix_lens=None, stream=None, out=None) -> DeviceTensor:
        """Q over the valid region of two InPlaceKvCaches (kv_len is their length)."""
        if k_cache.handle is None or v_cache.handle is None:
            raise TractRocmError("empty kv-cache")
        b, hq, sq, d = _canon4(q.shape)
        cb, _, _, cd = _canon4(k_cache._shape)
        if (b, d) != (cb, cd):
            raise TractRocmError(f"Q {q.shape} does not match the cache's {k_cache._shape}")
        slopes, documents, prefix_lens = self._rules(slopes, documents, prefix_lens, b, hq, k_cache.len(), stream)
        out = _output(out, q.shape, q.dtype)
        need = Workspace.bytes_for(b, hq, sq, d)
        ws = self._scratch.holding(need, stream)
        call("trocm_sdpa_cached_scored", q.ptr, _code(q.dtype), hq, sq, k_cache.handle, v_cache.handle, out.ptr, _scale_arg(self.scale), self.softcap,
             _optr(slopes), _optr(documents), _optr(prefix_lens), int(self.is_causal), ws.ptr, need, _sh(stream))
        return out
