"""Trees of drafted tokens over include/arclight_draft.h: what a step needs
before attention, and their verification after it.

    pos, cells, seq, bits = tree(parents, lens, counts)          # (n_seq, T) int32 x 3, (n_seq, T, words) int32
    path, kept, next = verify(target, tokens, accept, sample, parents=parents, counts=counts)

parents (n_seq, T) int32: the node that each one follows, a smaller one; of
node 0, the last accepted token, -1. lens (n_seq,): cells of each sequence, the
nodes' among them. target (n_seq, T, V) f32: the probabilities of what follows
each node; draft: those that its children were drawn from (None: they were
chosen). accept (n_seq, T), sample (n_seq,) f32: random numbers in [0, 1).

A step of a server: paged.append(..., pos, seq, cells=cells), paged.attention(...,
bits=bits), verify, paged.keep(caches, lens, counts, path, kept).

TreeCall and VerifyCall hold a call's argument structure, as a C host does, to
run it any number of times over the same buffers.
"""
import ctypes

import numpy as np

from . import abi
from ._lib import call, load
from .device import DeviceTensor


class TreeCall:
    """Outputs that are None are left out."""

    def __init__(self, parents, lens, counts=None, pos=None, cells=None, seq=None, bits=None, stream=None):
        a = self.args = abi.AlDraftTreeArgs()
        a.parents, a.lens = parents.desc(), lens.desc()
        for name, t in (("counts", counts), ("pos", pos), ("cells", cells), ("seq", seq), ("bits", bits)):
            if t is not None:
                setattr(a, name, t.desc())
        a.stream = stream.handle if stream is not None else None
        self._ref, self._kept = ctypes.byref(a), (parents, lens, counts, pos, cells, seq, bits, stream)

    def run(self):
        call("al_draft_tree_i32", self._ref)


class VerifyCall:
    """parents None: chains; counts None: T nodes each."""

    def __init__(self, target, tokens, accept, sample, path, kept, next, *, parents=None, counts=None, draft=None, stream=None,
                 workspace=None):
        a = self.args = abi.AlDraftVerifyArgs()
        a.target, a.tokens, a.accept, a.sample = target.desc(), tokens.desc(), accept.desc(), sample.desc()
        a.path, a.kept, a.next = path.desc(), kept.desc(), next.desc()
        for name, t in (("parents", parents), ("counts", counts), ("draft", draft)):
            if t is not None:
                setattr(a, name, t.desc())
        a.stream = stream.handle if stream is not None else None
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.ptr, workspace.nbytes
        self._ref = ctypes.byref(a)
        self._kept = (target, tokens, accept, sample, path, kept, next, parents, counts, draft, stream, workspace)

    def workspace_bytes(self):
        return int(load().al_draft_verify_workspace_bytes(self._ref))

    def run(self):
        call("al_draft_verify_f32", self._ref)


def tree(parents, lens, counts=None, stream=None):
    """Enqueues it; returns pos, cells, seq and bits, allocated."""
    n, T = parents.shape
    pos, cells, seq = (DeviceTensor.empty((n, T), np.int32) for _ in range(3))
    bits = DeviceTensor.empty((n, T, max(1, (T + 31) // 32)), np.int32)
    TreeCall(parents, lens, counts, pos, cells, seq, bits, stream).run()
    return pos, cells, seq, bits


def verify(target, tokens, accept, sample, **kw):
    """Enqueues it; returns path (n_seq, T), kept and next (n_seq,), allocated."""
    path = DeviceTensor.empty(tokens.shape, np.int32)
    kept, next = (DeviceTensor.empty((tokens.shape[0],), np.int32) for _ in range(2))
    VerifyCall(target, tokens, accept, sample, path, kept, next, **kw).run()
    return path, kept, next
