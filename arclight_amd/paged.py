"""A paged f16 KV cache over include/arclight_paged.h: appending a batch's
keys and values to it, and attention of the sequences' new tokens over it.

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

AppendCall and AttentionCall hold a call's argument structure, as a C host
does, to run it any number of times over the same buffers.
"""
import ctypes

import numpy as np

from . import abi
from ._lib import call, load
from .device import DeviceTensor


class PagedCache:
    """One layer's pools and the sequences' page tables, as DeviceTensors:
    k, v (n_pages, P, Hkv, 128) f16, or (n_pages, Hkv, P, 128) with
    heads_first; table (n_seq, max_pages) int32."""

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
                 stream=None):
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
        self._ref, self._kept = ctypes.byref(a), (cache, q, k, v, pos, seq, q_out, q_w, k_w, rope, stream)

    def run(self):
        call("al_paged_append_f32", self._ref)


class AttentionCall:
    def __init__(self, cache, q, lens, dst, *, scale, counts=None, sinks=None, logit_softcap=0.0, stream=None,
                 workspace=None):
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
        self._ref, self._kept = ctypes.byref(a), (cache, q, lens, dst, counts, sinks, stream, workspace)

    def workspace_bytes(self):
        return int(load().al_paged_fattn_workspace_bytes(self._ref))

    def run(self):
        call("al_paged_fattn_f16", self._ref)


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
