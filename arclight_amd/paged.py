"""A paged f16 KV cache over include/arclight_paged.h: appending a batch's
keys and values to it, attention of the sequences' new tokens over it, and
cells moved in all layers.

    cache = PagedCache(k_pool, v_pool, table)          # (n_pages, P, Hkv, 128) f16 x 2, (n_seq, max_pages) i32
    append(cache, q, k, v, pos, seq, q_out, q_w=..., k_w=..., eps=1e-6, rope=abi.qwen3_rope())
    out = attention(cache, q_out_by_sequence, lens, scale=1 / 128 ** 0.5)

Cell c of sequence s is cell c % P of page table[s, c // P]. append takes one
row for each token, q (T, Hq, 128) and k, v (T, Hkv, 128) f32, with its
position and its sequence (negative: a padding row); attention takes q
(n_seq, T, Hq, 128) f32, the last T tokens (or counts[s] of them) of each
sequence's lens[s] cells. A decode step's rows are the same in both, one
token for each sequence. norm=False rotates the rows as they are, without q_w
and k_w.

A layer with a window: attention(..., window=4096, first=4) sees the last 4096
positions and the first 4 cells. A tree of drafted tokens: append(...,
cells=cells) puts a row into a cell that is not its position, and
attention(..., bits=bits) sees of the new tokens those whose bits are set
(draft.tree makes pos, cells, seq and bits); pos=pos beside a window.

    keep([cache, ...], lens, counts, path, kept)       # the accepted path's cells, in all layers: the new lengths
    copy_pages([cache, ...], src, dst, cells)          # pages (or their first cells) into others: forks

AppendCall, AttentionCall, KeepCall and CopyCall hold a call's argument
structure, as a C host does, to run it any number of times over the same
buffers.
"""
import ctypes

import numpy as np

from . import abi
from ._lib import call, load
from .device import DeviceTensor


class PagedCache:
    """One layer's pools and the sequences' page tables, as DeviceTensors:
    k, v (n_pages, P, Hkv, 128) f16, or (n_pages, Hkv, P, 128) with
    heads_first; table (n_seq, max_pages) int32 (None where only pages are
    copied)."""

    def __init__(self, k, v, table, heads_first=False):
        self.k, self.v, self.table, self.heads_first = k, v, table, heads_first
        self.axes = (3, 2, 1, 0) if heads_first else abi.KV_AXES

    def pool_descs(self):
        return [_as(t, self.axes).desc() for t in (self.k, self.v)]


def _as(t, axes):
    """The same memory with nnml dim i on numpy axis axes[i]."""
    return DeviceTensor(t.buf, t.type, t.shape, t.strides, t.offset, axes)


class AppendCall:
    def __init__(self, cache, q, k, v, pos, seq, q_out, *, q_w=None, k_w=None, eps=0.0, norm=True, rope=None,
                 cells=None, stream=None):
        a = self.args = abi.AlPagedAppendArgs()
        if q is not None:
            a.q, a.q_out = q.desc(), q_out.desc()
        a.k, a.v, a.pos, a.seq = k.desc(), v.desc(), pos.desc(), seq.desc()
        if norm and q_w is not None:
            a.q_w = q_w.desc()
        if norm and k_w is not None:
            a.k_w = k_w.desc()
        a.k_pool, a.v_pool = cache.pool_descs()
        a.table = cache.table.desc()
        a.eps, a.norm = eps, int(norm)
        if rope is not None:
            a.rope = ctypes.pointer(rope)
        a.stream = stream.handle if stream is not None else None
        self._ref, self._kept = ctypes.byref(a), (cache, q, k, v, pos, seq, q_out, q_w, k_w, rope, cells, stream)
        self._cells = None if cells is None else ctypes.byref(cells.desc())

    def run(self):
        if self._cells is None:
            call("al_paged_append_f32", self._ref)
        else:
            call("al_paged_append_cells_f32", self._ref, self._cells)


class AttentionCall:
    """window, first, bits (n_seq, T, words) int32 and pos (n_seq, T) int32:
    which cells a token sees, where that is not all before it."""

    def __init__(self, cache, q, lens, dst, *, scale, counts=None, sinks=None, logit_softcap=0.0, window=0, first=0,
                 bits=None, pos=None, stream=None, workspace=None):
        a = self.args = abi.AlPagedFattnArgs()
        a.q, a.dst = _as(q, abi.Q_AXES).desc(), _as(dst, abi.DST_AXES).desc()
        a.k_pool, a.v_pool = cache.pool_descs()
        a.table, a.lens = cache.table.desc(), lens.desc()
        if counts is not None:
            a.counts = counts.desc()
        if sinks is not None:
            a.sinks = sinks.desc()
        a.scale, a.logit_softcap = scale, logit_softcap
        a.stream = stream.handle if stream is not None else None
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.ptr, workspace.nbytes
        self._ref, self._kept = ctypes.byref(a), (cache, q, lens, dst, counts, sinks, bits, pos, stream, workspace)
        self._sees = None
        if window or first or bits is not None or pos is not None:
            r = abi.AlPagedSees(window, first)
            if bits is not None:
                r.bits = bits.desc()
            if pos is not None:
                r.pos = pos.desc()
            self._sees = ctypes.byref(r)

    def workspace_bytes(self):
        if self._sees is None:
            return int(load().al_paged_fattn_workspace_bytes(self._ref))
        return int(load().al_paged_fattn_sees_workspace_bytes(self._ref, self._sees))

    def run(self):
        if self._sees is None:
            call("al_paged_fattn_f16", self._ref)
        else:
            call("al_paged_fattn_sees_f16", self._ref, self._sees)


def _layers(caches):
    """The pools of all layers, and what has to live as long: caches of one
    shape."""
    caches = list(caches)
    if not caches:
        raise ValueError("no layers")
    like = [(c.k.shape, c.k.strides, c.v.shape, c.v.strides, c.heads_first) for c in caches]
    if any(x != like[0] for x in like):
        raise ValueError("the layers' pools have to be of one shape, with the same strides")
    r = abi.AlPagedLayers()
    r.k_pool, r.v_pool = caches[0].pool_descs()
    pointers = ctypes.c_void_p * len(caches)
    k, v = pointers(*[c.k.ptr for c in caches]), pointers(*[c.v.ptr for c in caches])
    r.k, r.v, r.n_layers = k, v, len(caches)
    return r, (caches, k, v)


class KeepCall:
    """caches: those of all layers, with one table; lens, kept, lens_out
    (n_seq,), path (n_seq, T) int32; counts (n_seq,) or None (T each)."""

    def __init__(self, caches, lens, counts, path, kept, lens_out=None, stream=None):
        a = self.args = abi.AlPagedKeepArgs()
        a.layers, pools = _layers(caches)
        if pools[0][0].table is None:
            raise ValueError("the sequences' table is missing")
        a.table, a.lens, a.path, a.kept = pools[0][0].table.desc(), lens.desc(), path.desc(), kept.desc()
        if counts is not None:
            a.counts = counts.desc()
        if lens_out is not None:
            a.lens_out = lens_out.desc()
        a.stream = stream.handle if stream is not None else None
        self._ref, self._kept = ctypes.byref(a), (pools, lens, counts, path, kept, lens_out, stream)

    def run(self):
        call("al_paged_keep_f16", self._ref)


class CopyCall:
    """src, dst, cells (n,) int32; cells None: whole pages."""

    def __init__(self, caches, src, dst, cells=None, stream=None):
        a = self.args = abi.AlPagedCopyArgs()
        a.layers, pools = _layers(caches)
        a.src, a.dst = src.desc(), dst.desc()
        if cells is not None:
            a.cells = cells.desc()
        a.stream = stream.handle if stream is not None else None
        self._ref, self._kept = ctypes.byref(a), (pools, src, dst, cells, stream)

    def run(self):
        call("al_paged_copy_f16", self._ref)


def append(cache, q, k, v, pos, seq, q_out=None, **kw):
    """Enqueues the append; returns q_out (allocated when None). q may be None."""
    if q is not None and q_out is None:
        q_out = DeviceTensor.empty(q.shape, np.float32)
    AppendCall(cache, q, k, v, pos, seq, q_out, **kw).run()
    return q_out


def attention(cache, q, lens, dst=None, **kw):
    """Enqueues the attention; returns dst, (n_seq, T, Hq, 128) f32
    (allocated when None: rows beyond counts then hold anything)."""
    if dst is None:
        dst = DeviceTensor.empty(q.shape, np.float32)
    AttentionCall(cache, q, lens, dst, **kw).run()
    return dst


def keep(caches, lens, counts, path, kept, lens_out=None, stream=None):
    """Enqueues the move; returns lens_out (allocated when None)."""
    if lens_out is None:
        lens_out = DeviceTensor.empty(lens.shape, np.int32)
    KeepCall(caches, lens, counts, path, kept, lens_out, stream).run()
    return lens_out


def copy_pages(caches, src, dst, cells=None, stream=None):
    """Enqueues the copy."""
    CopyCall(caches, src, dst, cells, stream).run()
