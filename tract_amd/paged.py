"""Serving over pages of keys and values, and beam search over them.  No counterpart in the reference, whose caches are a tensor per
sequence (gpu/src/ops/dyn_kv_cache.rs:58-113): here sequences hold pages of one pool through a table, and tables, lengths and the stack of
free pages live on the device.

* ``PagedPlan``     pages for the tokens that a step adds, and where each token goes
* ``PagedAppend``   new rows of keys and values into their pages
* ``PagedSdpa``     attention of one or a few new tokens per sequence over its pages
* ``PagedReorder``  sequences that go on from other sequences, sharing pages; ``PagedCopy`` copies those that they cannot share
* ``BeamSelect``    the best continuations of a request's beams
* ``PagedKvCache``  the pools of a model's layers with their tables: a step is ``plan``, ``append`` and ``attend`` per layer

``PagedSdpa`` and ``BeamSelect`` keep their workspaces from call to call: their calls follow each other on one stream.  A graph that
recorded a call uses that workspace: the object has to live as long as the graph, and later calls of other shapes leave it be.
"""
from __future__ import annotations

import ctypes as C
import functools

import numpy as np

from ._lib import TractRocmError, call
from .ops import _as_device, _code, _same, _scale_arg, _I64x3
from .runtime import DeviceTensor, _sh
from .scored import _optr, _output, _Scratch

_I32, _F32 = np.dtype(np.int32), np.dtype(np.float32)
_I64x2 = C.c_int64 * 2


def _ints(what, t, shape):
    if t.shape != tuple(shape) or not _same(t.dtype, _I32):
        raise TractRocmError(f"{what} must be int32 of shape {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t


def _outputs(out, shapes):
    """The named int32 outputs: those of `out`, which must be of the shapes, and new ones for the others."""
    out = {} if out is None else dict(out)
    for name, shape in shapes.items():
        t = out.get(name)
        if t is None:
            out[name] = DeviceTensor(shape, _I32)
        else:
            _ints(name, t, shape)
    return out


def _holds(out, shapes) -> bool:
    """Whether `out` has all of the named int32 outputs (a loop: this runs with every call)."""
    if out is None:
        return False
    for name, shape in shapes.items():
        t = out.get(name)
        if t is None or t.shape != shape or t.dtype is not _I32:
            return False
    return True


def _strides(given, kind, n):
    if given is None:
        return None
    if len(given) < n:
        raise TractRocmError(f"expected {n} strides, got {list(given)}")
    return kind(*[int(s) for s in given[:n]])


def _pool(k_pages, v_pages):
    if len(k_pages.shape) != 4 or k_pages.shape != v_pages.shape or not _same(k_pages.dtype, v_pages.dtype):
        raise TractRocmError(f"K and V pages must be [n_pages, kv_heads, page_size, head_dim] of one shape and type, got {k_pages.shape} and {v_pages.shape}")
    return k_pages.shape


class PagedPlan:
    """Pages and slots for a step's tokens, from the sequences' lengths (trocm_paged_plan)."""

    def __init__(self, page_size: int):
        self.page_size = int(page_size)
        self._last = (None, None)

    def name(self) -> str:
        return "PagedPlan"

    def eval(self, lens, n_new, table, free_pages, free_count, tokens: int, refs=None, stream=None, out=None) -> dict:
        """lens, n_new [n_seq]; table [n_seq, width], whose new pages are written; free_pages [n_pages] of which the first
        free_count [1] are free; refs [n_pages] or None, 1 for new pages; `tokens` packed rows.  Returns (into `out`, where given)
        lens [n_seq], starts [n_seq + 1], slots and positions [tokens], free_count [1], refused [1]; none of them may be an input."""
        if not isinstance(lens, DeviceTensor) or not isinstance(n_new, DeviceTensor):
            lens, n_new = _as_device(lens, stream), _as_device(n_new, stream)
        key = (lens.shape, n_new.shape, table.shape, free_pages.shape, free_count.shape, tokens, refs is None or (refs.shape, refs.dtype),
               lens.dtype, n_new.dtype, table.dtype, free_pages.dtype, free_count.dtype)
        last_key, sizes = self._last   # (a pair, read once: another thread's call may put its own there)
        if key != last_key:
            if len(table.shape) != 2 or len(free_pages.shape) != 1 or tokens < 0:
                raise TractRocmError("paged_plan: table must be [n_seq, width], free_pages [n_pages], tokens not negative")
            n, width = table.shape
            for what, t, shape in (("lens", lens, (n,)), ("n_new", n_new, (n,)), ("table", table, (n, width)), ("free_pages", free_pages, free_pages.shape),
                                   ("free_count", free_count, (1,))):
                _ints(what, t, shape)
            if refs is not None:
                _ints("refs", refs, free_pages.shape)
            sizes = n, width, free_pages.shape[0], {"lens": (n,), "starts": (n + 1,), "slots": (tokens,), "positions": (tokens,), "free_count": (1,), "refused": (1,)}
            self._last = key, sizes
        n, width, n_pages, shapes = sizes
        if not _holds(out, shapes):
            out = _outputs(out, shapes)
        call("trocm_paged_plan", lens.ptr, n_new.ptr, n, self.page_size, table.ptr, width, free_pages.ptr, free_count.ptr, n_pages, None if refs is None else refs.ptr,
             tokens, out["lens"].ptr, out["starts"].ptr, out["slots"].ptr, out["positions"].ptr, out["free_count"].ptr, out["refused"].ptr, None if stream is None else _sh(stream))
        return out


class PagedAppend:
    """Rows of K and V into their pages (trocm_paged_append)."""

    def __init__(self):
        self._last = (None, None)

    def name(self) -> str:
        return "PagedAppend"

    def eval(self, k, v, slots, k_pages, v_pages, stream=None, k_strides=None, v_strides=None, page_strides=None) -> None:
        """K and V [tokens, kv_heads, head_dim], strides of views for token and head in elements (None: dense); slots [tokens];
        pages [n_pages, kv_heads, page_size, head_dim], strides for page, head and token (None: dense)."""
        if not isinstance(k, DeviceTensor) or not isinstance(v, DeviceTensor):
            k, v = _as_device(k, stream), _as_device(v, stream)
        key = (k.shape, v.shape, slots.shape, k_pages.shape, v_pages.shape, k.dtype, v.dtype, slots.dtype, k_pages.dtype, v_pages.dtype,
               k_strides and tuple(k_strides), v_strides and tuple(v_strides), page_strides and tuple(page_strides))
        last_key, sizes = self._last
        if key != last_key:
            n_pages, hkv, page, d = _pool(k_pages, v_pages)
            if len(k.shape) != 3 or k.shape[1:] != (hkv, d) or v.shape != k.shape or not _same(k.dtype, k_pages.dtype) or not _same(v.dtype, k_pages.dtype):
                raise TractRocmError(f"paged_append: K {k.shape} and V {v.shape} must be [tokens, {hkv}, {d}] of the pages' type")
            _ints("slots", slots, k.shape[:1])
            sizes = (_code(k.dtype), k.shape[0], hkv, d, _strides(k_strides, _I64x2, 2), _strides(v_strides, _I64x2, 2)), (n_pages, page, _strides(page_strides, _I64x3, 3))
            self._last = key, sizes
        call("trocm_paged_append", k.ptr, v.ptr, *sizes[0], slots.ptr, k_pages.ptr, v_pages.ptr, *sizes[1], None if stream is None else _sh(stream))


@functools.lru_cache(maxsize=1024)   # (a function of its arguments alone)
def _sdpa_bytes(n_seq, q_heads, kv_heads, q_len, head_dim) -> int:
    n = C.c_size_t()
    call("trocm_sdpa_paged_workspace_bytes", n_seq, q_heads, kv_heads, q_len, head_dim, C.byref(n))
    return n.value


class PagedSdpa:
    """softmax(scale Q K^T) V over the pages of every sequence (trocm_sdpa_paged)."""

    def __init__(self, scale=None, is_causal: bool = True):
        self.scale, self.is_causal = scale, bool(is_causal)
        self._scratch, self._last = _Scratch(), (None, None, None)

    def name(self) -> str:
        return "PagedSdpa"

    def eval(self, q, k_pages, v_pages, table, lens, stream=None, out=None, page_strides=None) -> DeviceTensor:
        """Q [n_seq, q_heads, q_len, head_dim]; pages [n_pages, kv_heads, page_size, head_dim], strides for page, head and token
        (None: dense); table [n_seq, width]; lens [n_seq], the new tokens counted."""
        if not isinstance(q, DeviceTensor):
            q = _as_device(q, stream)
        dtype, shape = q.dtype, q.shape
        key = (shape, k_pages.shape, v_pages.shape, table.shape, lens.shape, dtype, k_pages.dtype, v_pages.dtype, table.dtype, lens.dtype, page_strides and tuple(page_strides))
        last_key, sizes, ws = self._last
        if key != last_key:
            n_pages, hkv, page, d = _pool(k_pages, v_pages)
            if len(shape) != 4 or shape[3] != d or not _same(k_pages.dtype, dtype):
                raise TractRocmError(f"paged attention: Q {shape} must be [n_seq, q_heads, q_len, {d}] of the pages' type")
            n, hq, sq, _ = shape
            if len(table.shape) != 2:
                raise TractRocmError("paged attention: table must be [n_seq, width]")
            _ints("table", table, (n, table.shape[1])), _ints("lens", lens, (n,))
            if hkv == 0 or hq % hkv:
                raise TractRocmError(f"Q heads ({hq}) must be a multiple of K/V heads ({hkv})")
            need = _sdpa_bytes(n, hq, hkv, sq, d)
            sizes, ws = ((_code(dtype), n, hq, hkv, sq, d), (n_pages, page, _strides(page_strides, _I64x3, 3)), table.shape[1], need), self._scratch.holding(need, stream)
            self._last = key, sizes, ws
        sizes, pages, width, need = sizes
        if out is None or out.shape != shape or out.dtype is not dtype:
            out = _output(out, shape, dtype)
        call("trocm_sdpa_paged", q.ptr, *sizes, k_pages.ptr, v_pages.ptr, *pages, table.ptr, width, lens.ptr, out.ptr, _scale_arg(self.scale), int(self.is_causal),
             ws.buf.ptr, need, None if stream is None else _sh(stream))
        return out


class PagedReorder:
    """Sequences that go on from other sequences (trocm_paged_reorder)."""

    def __init__(self, page_size: int):
        self.page_size = int(page_size)
        self._last = (None, None)

    def name(self) -> str:
        return "PagedReorder"

    def eval(self, parents, table, lens, refs, free_pages, free_count, stream=None, out=None) -> dict:
        """Sequence j becomes parents[j] (-1: empty); the rest as PagedPlan has it.  Returns (into `out`, where given) table, lens, refs,
        free_pages, free_count, copies [n_seq, 3] for PagedCopy and missing [1] (not 0: nothing has changed); none of them may be an input."""
        if not isinstance(parents, DeviceTensor):
            parents = _as_device(parents, stream)
        key = (parents.shape, table.shape, lens.shape, refs.shape, free_pages.shape, free_count.shape,
               parents.dtype, table.dtype, lens.dtype, refs.dtype, free_pages.dtype, free_count.dtype)
        last_key, sizes = self._last
        if key != last_key:
            if len(table.shape) != 2 or len(refs.shape) != 1:
                raise TractRocmError("paged_reorder: table must be [n_seq, width], refs [n_pages]")
            (n, width), n_pages = table.shape, refs.shape[0]
            for what, t, shape in (("parents", parents, (n,)), ("table", table, (n, width)), ("lens", lens, (n,)), ("refs", refs, (n_pages,)), ("free_pages", free_pages, (n_pages,)),
                                   ("free_count", free_count, (1,))):
                _ints(what, t, shape)
            sizes = n, width, n_pages, {"table": (n, width), "lens": (n,), "refs": (n_pages,), "free_pages": (n_pages,), "free_count": (1,), "copies": (n, 3), "missing": (1,)}
            self._last = key, sizes
        n, width, n_pages, shapes = sizes
        if not _holds(out, shapes):
            out = _outputs(out, shapes)
        call("trocm_paged_reorder", parents.ptr, n, self.page_size, table.ptr, width, lens.ptr, refs.ptr, free_pages.ptr, free_count.ptr, n_pages, out["table"].ptr,
             out["lens"].ptr, out["refs"].ptr, out["free_pages"].ptr, out["free_count"].ptr, out["copies"].ptr, out["missing"].ptr, None if stream is None else _sh(stream))
        return out


class PagedCopy:
    """The rows of pages that sequences could not share, in all pools (trocm_paged_copy)."""

    def name(self) -> str:
        return "PagedCopy"

    def eval(self, copies, pools, stream=None, page_strides=None) -> None:
        """copies [n, 3] as PagedReorder returns them; pools: the K and V pages of all layers, of one shape and type."""
        if not pools:
            return
        first = pools[0]
        shape, dtype = first.shape, first.dtype
        if len(shape) != 4 or any(p.shape != shape or not _same(p.dtype, dtype) for p in pools):
            raise TractRocmError("paged_copy: pools must be [n_pages, kv_heads, page_size, head_dim] of one shape and type")
        if len(copies.shape) != 2:
            raise TractRocmError("paged_copy: copies must be [n, 3]")
        _ints("copies", copies, (copies.shape[0], 3))
        n_pages, hkv, page, d = shape
        at = (C.c_void_p * len(pools))(*[p.ptr.value for p in pools])
        call("trocm_paged_copy", copies.ptr, copies.shape[0], at, len(pools), _code(dtype), hkv, d, n_pages, page, _strides(page_strides, _I64x3, 3),
             None if stream is None else _sh(stream))


@functools.lru_cache(maxsize=1024)
def _beam_bytes(batch, beams, vocab, keep) -> int:
    n = C.c_size_t()
    call("trocm_beam_select_workspace_bytes", batch, beams, vocab, keep, C.byref(n))
    return n.value


class BeamSelect:
    """The `keep` best of score + log_softmax(logits) over a request's beams and the vocabulary (trocm_beam_select)."""

    def __init__(self, keep: int, eos: int = -1):
        self.keep, self.eos = int(keep), int(eos)
        self._scratch, self._last = _Scratch(), (None, None, None)

    def name(self) -> str:
        return "BeamSelect"

    def eval(self, logits, scores, ended=None, stream=None, out=None, row_stride: int = 0) -> dict:
        """logits [batch, beams, vocab], rows `row_stride` elements apart (0: dense); scores f32 [batch, beams]; ended int32
        [batch, beams] or None.  Returns (into `out`, where given) scores f32, parents (rows: request * beams + beam), tokens and ended
        int32, all [batch, keep], best first."""
        if not isinstance(logits, DeviceTensor) or not isinstance(scores, DeviceTensor):
            logits, scores = _as_device(logits, stream), _as_device(scores, stream)
        if ended is not None and not isinstance(ended, DeviceTensor):
            ended = _as_device(ended, stream)
        key = (self.keep, logits.shape, scores.shape, logits.dtype, scores.dtype, ended is None or (ended.shape, ended.dtype))
        last_key, sizes, ws = self._last
        if key != last_key:
            if len(logits.shape) != 3 or scores.shape != logits.shape[:2] or not _same(scores.dtype, _F32):
                raise TractRocmError(f"beam_select: logits {logits.shape} must be [batch, beams, vocab] and scores f32 of [batch, beams]")
            if ended is not None:
                _ints("ended", ended, scores.shape)
            batch, beams, vocab = logits.shape
            need = _beam_bytes(batch, beams, vocab, self.keep)
            shape = batch, self.keep
            sizes, ws = ((_code(logits.dtype), batch, beams, vocab), shape, {"parents": shape, "tokens": shape, "ended": shape}, need), self._scratch.holding(need, stream)
            self._last = key, sizes, ws
        sizes, shape, shapes, need = sizes
        scores_out = None if out is None else out.get("scores")
        if scores_out is None or scores_out.shape != shape or scores_out.dtype is not _F32 or not _holds(out, shapes):
            if scores_out is None:
                scores_out = DeviceTensor(shape, _F32)
            elif scores_out.shape != shape or not _same(scores_out.dtype, _F32):
                raise TractRocmError(f"scores must be f32 of shape {list(shape)}")
            out = _outputs(out, shapes)
            out["scores"] = scores_out
        call("trocm_beam_select", logits.ptr, *sizes, row_stride, scores.ptr, _optr(ended), self.eos, self.keep, scores_out.ptr, out["parents"].ptr, out["tokens"].ptr,
             out["ended"].ptr, ws.buf.ptr, need, None if stream is None else _sh(stream))
        return out


class PagedKvCache:
    """The pages of a model's layers, and their tables: `max_seqs` places for sequences of up to `max_tokens` tokens each.

    A step is ``plan`` (how many tokens each place gets), then ``append`` and ``attend`` for every layer.  ``reorder`` lets places go on
    from other places (beams) and empties those whose parent is -1, whose pages become free.  Nothing of this waits for the device, but
    ``lens``, ``free`` and ``refused``, which read it back.  Tables change hands between two sets of buffers with every ``plan`` and
    ``reorder``: a recorded graph holds an even number of each, or is recorded twice."""

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int, max_tokens: int, dtype=np.float16, layers: int = 1, scale=None):
        self.page_size, self.max_seqs, self.n_pages = int(page_size), int(max_seqs), int(n_pages)
        if self.page_size < 1 or self.n_pages < 1 or layers < 1 or max_seqs < 1 or max_tokens < 1:
            raise TractRocmError("paged cache: sizes must be positive")
        width = -(-int(max_tokens) // self.page_size)
        dtype = np.dtype(dtype)
        self.k = [DeviceTensor((n_pages, kv_heads, page_size, head_dim), dtype) for _ in range(layers)]
        self.v = [DeviceTensor((n_pages, kv_heads, page_size, head_dim), dtype) for _ in range(layers)]
        up = DeviceTensor.from_numpy
        self._table = [up(np.full((max_seqs, width), -1, np.int32)) for _ in range(2)]
        self._lens = [up(np.zeros(max_seqs, np.int32)) for _ in range(2)]
        self._refs = [up(np.zeros(n_pages, np.int32)) for _ in range(2)]
        self._free = [up(np.arange(n_pages, dtype=np.int32)[::-1]) for _ in range(2)]   # (pages are taken from the end: 0 first)
        self._count = [up(np.array([n_pages], np.int32)) for _ in range(2)]
        self._at = {"table": 0, "lens": 0, "refs": 0, "free": 0, "count": 0}             # which of the two holds now
        self._refused, self._missing, self._copies = DeviceTensor((1,), _I32), DeviceTensor((1,), _I32), DeviceTensor((max_seqs, 3), _I32)
        self._plan, self._append, self._reorder, self._copy = PagedPlan(page_size), PagedAppend(), PagedReorder(page_size), PagedCopy()
        self._sdpa = PagedSdpa(scale)
        self.slots = self.positions = self.starts = None

    def _now(self, name):
        return getattr(self, "_" + name)[self._at[name]]

    def _next(self, name):
        return getattr(self, "_" + name)[1 - self._at[name]]

    @property
    def table(self) -> DeviceTensor:
        return self._now("table")

    @property
    def device_lens(self) -> DeviceTensor:
        return self._now("lens")

    def plan(self, n_new, tokens: int, stream=None, out=None) -> dict:
        """n_new [max_seqs] tokens for every place (0: none), which are `tokens` packed rows.  Afterwards `slots`, `positions` and
        `starts` are the step's, and the lengths count its tokens."""
        out = {} if out is None else dict(out)
        out.update(lens=self._next("lens"), free_count=self._next("count"), refused=self._refused)
        out = self._plan.eval(self._now("lens"), n_new, self._now("table"), self._now("free"), self._now("count"), tokens, refs=self._now("refs"), stream=stream, out=out)
        for name in ("lens", "count"):
            self._at[name] ^= 1
        self.slots, self.positions, self.starts = out["slots"], out["positions"], out["starts"]
        return out

    def append(self, layer: int, k, v, stream=None, k_strides=None, v_strides=None) -> None:
        """The step's packed rows of a layer, [tokens, kv_heads, head_dim]."""
        if self.slots is None:
            raise TractRocmError("paged cache: plan a step before its rows are appended")
        self._append.eval(k, v, self.slots, self.k[layer], self.v[layer], stream=stream, k_strides=k_strides, v_strides=v_strides)

    def attend(self, layer: int, q, stream=None, out=None) -> DeviceTensor:
        """Q [max_seqs, q_heads, q_len, head_dim] over the pages of every place, causal."""
        return self._sdpa.eval(q, self.k[layer], self.v[layer], self._now("table"), self._now("lens"), stream=stream, out=out)

    def reorder(self, parents, stream=None) -> None:
        """Place j goes on from place parents[j]; -1 empties it.  Copies what cannot be shared, in all layers."""
        out = {"table": self._next("table"), "lens": self._next("lens"), "refs": self._next("refs"), "free_pages": self._next("free"), "free_count": self._next("count"),
               "copies": self._copies, "missing": self._missing}
        self._reorder.eval(parents, self._now("table"), self._now("lens"), self._now("refs"), self._now("free"), self._now("count"), stream=stream, out=out)
        self._copy.eval(self._copies, self.k + self.v, stream=stream)
        for name in self._at:
            self._at[name] ^= 1

    def lens(self, stream=None) -> np.ndarray:
        return self._now("lens").to_numpy(stream)

    def free(self, stream=None) -> int:
        """How many pages are free."""
        return int(self._now("count").to_numpy(stream)[0])

    def refused(self, stream=None) -> int:
        """How many places the last plan refused."""
        return int(self._refused.to_numpy(stream)[0])

    def missing(self, stream=None) -> int:
        """How many free pages the last reorder lacked (0: it is done)."""
        return int(self._missing.to_numpy(stream)[0])
