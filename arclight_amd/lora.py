"""Low-rank adapters of many requests beside a shared projection, over
include/arclight_lora.h.

    ad = Adapters(a, b, scales, ranks)      # (n, R, K) and (n, N, R) f16, (n,) f32, (n,) int32
    y = apply(ad, x, ids, base)             # base + scale B (A x) of each row's adapter
    y = project(ad, wo, x, ids)             # the same beside the Q4_0 projection wo

x (T, K) f32, ids (T,) int32 (negative: no adapter), base and y (T, N) f32:
build_lora_mm (nnml/src/cgraph.cpp:497-500) with an adapter for each row.
ApplyCall and ProjectCall hold a call's argument structure, as a C host does,
to run it any number of times over the same buffers.
"""
import ctypes

import numpy as np

from . import abi
from ._lib import call, load
from .device import DeviceTensor


class Adapters:
    """Resident adapters as DeviceTensors: a (n, R, K), b (n, N, R) f16,
    scales (n,) f32 or None (1), ranks (n,) int32 or None (R)."""

    def __init__(self, a, b, scales=None, ranks=None):
        self.a, self.b, self.scales, self.ranks = a, b, scales, ranks
        self.N = b.shape[1]


class _Call:
    def __init__(self, entry, ad, x, ids, y, base, w, stream, workspace):
        a = self.args = abi.AlLoraArgs()
        a.a, a.b, a.x, a.ids, a.y = ad.a.desc(), ad.b.desc(), x.desc(), ids.desc(), y.desc()
        if ad.scales is not None:
            a.scales = ad.scales.desc()
        if ad.ranks is not None:
            a.ranks = ad.ranks.desc()
        if base is not None:
            a.base = base.desc()
        if w is not None:
            a.w = w.desc()
        a.stream = stream.handle if stream is not None else None
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.ptr, workspace.nbytes
        self._entry, self._ref, self._kept = entry, ctypes.byref(a), (ad, x, ids, y, base, w, stream, workspace)

    def workspace_bytes(self):
        return int(load().al_lora_workspace_bytes(self._ref))

    def run(self):
        call(self._entry, self._ref)


class ApplyCall(_Call):
    """base None: y's own content."""

    def __init__(self, ad, x, ids, base, y, stream=None, workspace=None):
        super().__init__("al_lora_f32", ad, x, ids, y, base, None, stream, workspace)


class ProjectCall(_Call):
    """w: a matmul.Q4_0Matrix or Q4_0View."""

    def __init__(self, ad, w, x, ids, y, stream=None, workspace=None):
        super().__init__("al_mul_mat_q4_0_lora_f32", ad, x, ids, y, None, w, stream, workspace)


def apply(ad, x, ids, base, y=None, stream=None):
    """Enqueues y = base + the adapters' products; returns y (allocated when
    None; base itself may be given). base None: y's own content, and then y has
    to be given."""
    if y is None:
        if base is None:
            raise ValueError("without base the products are added to y, which has to be given")
        y = DeviceTensor.empty((x.shape[0], ad.N), np.float32)
    ApplyCall(ad, x, ids, base, y, stream).run()
    return y


def project(ad, w, x, ids, y=None, stream=None):
    """Enqueues y = w x + the adapters' products; returns y."""
    if y is None:
        y = DeviceTensor.empty((x.shape[0], w.N), np.float32)
    ProjectCall(ad, w, x, ids, y, stream).run()
    return y
