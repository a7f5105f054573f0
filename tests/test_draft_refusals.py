"""What the entry points for drafts, windows and moved cells refuse, before any
device call (CPU), and the argument structures' layouts."""
import ctypes
import os
import subprocess

import pytest

from arclight_amd import _lib, abi
from tests.test_paged_refusals import POOL_FAULTS, SOME, T, append_args, fattn_args

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (run python -m arclight_amd.build)")
F32, F16, I32 = abi.AL_TYPE_F32, abi.AL_TYPE_F16, abi.AL_TYPE_I32


def fill(a, d):
    for n, v in d.items():
        setattr(a, n, v)
    return a


def refused(entry, status, name, *args):
    lib = _lib.load()
    assert getattr(lib, entry)(*(ctypes.byref(a) for a in args)) == status
    assert lib.al_last_error().decode().startswith(name), lib.al_last_error()


SEES = dict(window=5, first=2, bits=T(I32, [1, 4, 3]), pos=T(I32, [4, 3]))


def four(**kw):
    return fattn_args(q=T(F32, [128, 4, 32, 3]), dst=T(F32, [128, 32, 4, 3]), **kw)


@pytest.mark.parametrize("change, status", [
    (dict(window=-1), abi.AL_ERR_INVALID), (dict(first=-1), abi.AL_ERR_INVALID), (dict(bits=T(F32, [1, 4, 3])), abi.AL_ERR_INVALID),
    (dict(bits=T(I32, [0, 4, 3])), abi.AL_ERR_INVALID), (dict(bits=T(I32, [1, 5, 3])), abi.AL_ERR_INVALID),
    (dict(bits=T(I32, [1, 4, 2])), abi.AL_ERR_INVALID), (dict(bits=T(I32, [1, 4, 3], data=SOME + 2)), abi.AL_ERR_INVALID),
    (dict(bits=T(I32, [1, 4, 3], nb=[4, 6, 24, 72])), abi.AL_ERR_INVALID), (dict(pos=T(I32, [3, 3])), abi.AL_ERR_INVALID),
    (dict(pos=T(I32, [4, 4])), abi.AL_ERR_INVALID), (dict(pos=T(F32, [4, 3])), abi.AL_ERR_INVALID),
    (dict(pos=abi.empty_tensor()), abi.AL_ERR_INVALID),              # bits and a window, without positions
    (dict(bits=abi.empty_tensor()), abi.AL_ERR_INVALID),             # positions without bits
])
def test_a_rule_is_refused(change, status):
    refused("al_paged_fattn_sees_f16", status, "paged_fattn", four(), fill(abi.AlPagedSees(), {**SEES, **change}))


@pytest.mark.parametrize("change, status", POOL_FAULTS)
def test_a_rules_pools_are_refused(change, status):
    refused("al_paged_fattn_sees_f16", status, "paged_fattn", four(**change), fill(abi.AlPagedSees(), SEES))


def test_null_rules_and_cells():
    lib = _lib.load()
    assert lib.al_paged_fattn_sees_f16(ctypes.byref(four()), None) == abi.AL_ERR_INVALID
    assert lib.al_paged_fattn_sees_f16(None, ctypes.byref(abi.AlPagedSees())) == abi.AL_ERR_INVALID
    assert lib.al_paged_fattn_sees_workspace_bytes(ctypes.byref(four()), None) == 0
    assert lib.al_paged_append_cells_f32(ctypes.byref(append_args()), None) == abi.AL_ERR_INVALID
    assert lib.al_paged_append_cells_f32(None, ctypes.byref(T(I32, [4]))) == abi.AL_ERR_INVALID
    for cells in (T(I32, [3]), T(F32, [4]), T(I32, [4], data=None), T(I32, [4], data=SOME + 1)):
        refused("al_paged_append_cells_f32", abi.AL_ERR_INVALID, "paged_append", append_args(), cells)
    # nothing to do
    a = fattn_args(q=T(F32, [128, 0, 32, 3]), dst=T(F32, [128, 32, 0, 3]))
    assert lib.al_paged_fattn_sees_f16(ctypes.byref(a), ctypes.byref(fill(abi.AlPagedSees(), dict(window=3)))) == abi.AL_OK


def tree_args(**kw):
    d = dict(parents=T(I32, [9, 3]), lens=T(I32, [3]), counts=T(I32, [3]), pos=T(I32, [9, 3]), cells=T(I32, [9, 3]), seq=T(I32, [9, 3]),
             bits=T(I32, [1, 9, 3]))
    return fill(abi.AlDraftTreeArgs(), {**d, **kw})


@pytest.mark.parametrize("change, status", [
    (dict(parents=T(I32, [9, 3], data=None)), abi.AL_ERR_INVALID), (dict(parents=T(F32, [9, 3])), abi.AL_ERR_INVALID),
    (dict(lens=T(I32, [2])), abi.AL_ERR_INVALID), (dict(lens=T(I32, [3], data=None)), abi.AL_ERR_INVALID),
    (dict(counts=T(I32, [4])), abi.AL_ERR_INVALID), (dict(pos=T(I32, [8, 3])), abi.AL_ERR_INVALID), (dict(cells=T(I32, [9, 2])), abi.AL_ERR_INVALID),
    (dict(seq=T(F32, [9, 3])), abi.AL_ERR_INVALID), (dict(bits=T(I32, [0, 9, 3])), abi.AL_ERR_INVALID), (dict(bits=T(I32, [1, 9, 4])), abi.AL_ERR_INVALID),
    (dict(parents=T(I32, [1025, 3]), pos=T(I32, [1025, 3]), cells=T(I32, [1025, 3]), seq=T(I32, [1025, 3]), bits=T(I32, [33, 1025, 3])),
     abi.AL_ERR_UNSUPPORTED)])
def test_trees_are_refused(change, status):
    refused("al_draft_tree_i32", status, "draft_tree", tree_args(**change))


def verify_args(**kw):
    d = dict(target=T(F32, [100, 9, 3]), tokens=T(I32, [9, 3]), parents=T(I32, [9, 3]), accept=T(F32, [9, 3]), sample=T(F32, [3]), path=T(I32, [9, 3]),
             kept=T(I32, [3]), next=T(I32, [3]))
    return fill(abi.AlDraftVerifyArgs(), {**d, **kw})


@pytest.mark.parametrize("change, status", [
    (dict(target=T(F32, [100, 9, 3], data=None)), abi.AL_ERR_INVALID), (dict(target=T(F16, [100, 9, 3])), abi.AL_ERR_INVALID),
    (dict(target=T(F32, [0, 9, 3])), abi.AL_ERR_INVALID), (dict(target=T(F32, [100, 9, 3], nb=[8, 800, 7200, 21600])), abi.AL_ERR_INVALID),
    (dict(target=T(F32, [100, 9, 3], data=SOME + 2)), abi.AL_ERR_INVALID), (dict(draft=T(F32, [99, 9, 3])), abi.AL_ERR_INVALID),
    (dict(draft=T(F32, [100, 8, 3])), abi.AL_ERR_INVALID), (dict(tokens=T(I32, [9, 3], data=None)), abi.AL_ERR_INVALID),
    (dict(tokens=T(I32, [8, 3])), abi.AL_ERR_INVALID), (dict(parents=T(abi.AL_TYPE_I64, [9, 3])), abi.AL_ERR_INVALID),
    (dict(accept=T(I32, [9, 3])), abi.AL_ERR_INVALID), (dict(accept=T(F32, [9, 2])), abi.AL_ERR_INVALID), (dict(sample=T(I32, [3])), abi.AL_ERR_INVALID),
    (dict(sample=T(F32, [2])), abi.AL_ERR_INVALID), (dict(path=T(I32, [9, 4])), abi.AL_ERR_INVALID), (dict(kept=T(I32, [3], data=None)), abi.AL_ERR_INVALID),
    (dict(next=T(F32, [3])), abi.AL_ERR_INVALID), (dict(counts=T(I32, [4])), abi.AL_ERR_INVALID),
    (dict(target=T(F32, [2 ** 24 + 1, 9, 3])), abi.AL_ERR_UNSUPPORTED),
    (dict(target=T(F32, [100, 1025, 3]), tokens=T(I32, [1025, 3]), parents=abi.empty_tensor(), accept=T(F32, [1025, 3]), path=T(I32, [1025, 3])),
     abi.AL_ERR_UNSUPPORTED)])
def test_verification_is_refused(change, status):
    refused("al_draft_verify_f32", status, "draft_verify", verify_args(**change))


def layers(n=2, pools=None, **kw):
    ptrs = (ctypes.c_void_p * max(n, 1))(*([SOME] * max(n, 1) if pools is None else pools))
    r = fill(abi.AlPagedLayers(), {**dict(k_pool=T(F16, [128, 16, 8, 10]), v_pool=T(F16, [128, 16, 8, 10])), **kw})
    r.k, r.v, r.n_layers = ptrs, ptrs, n
    r.kept = ptrs
    return r


def keep_args(**kw):
    d = dict(layers=layers(), table=T(I32, [5, 3]), lens=T(I32, [3]), counts=T(I32, [3]), path=T(I32, [9, 3]), kept=T(I32, [3]),
             lens_out=T(I32, [3], data=2 * SOME))
    return fill(abi.AlPagedKeepArgs(), {**d, **kw})


LAYER_FAULTS = [(lambda: layers(0), abi.AL_ERR_INVALID), (lambda: layers(65536, [SOME] * 65536), abi.AL_ERR_INVALID),
                (lambda: layers(pools=[SOME, None]), abi.AL_ERR_INVALID), (lambda: layers(pools=[SOME, SOME + 8]), abi.AL_ERR_INVALID),
                (lambda: layers(k_pool=T(F32, [128, 16, 8, 10])), abi.AL_ERR_UNSUPPORTED),
                (lambda: layers(v_pool=T(F16, [128, 16, 8, 11])), abi.AL_ERR_INVALID),
                (lambda: layers(v_pool=T(F16, [128, 16, 8, 10], nb=[2, 264, 4224, 33792])), abi.AL_ERR_INVALID)]


@pytest.mark.parametrize("change, status", LAYER_FAULTS + [
    (dict(table=T(I32, [5, 3], data=None)), abi.AL_ERR_INVALID), (dict(path=T(I32, [9, 2])), abi.AL_ERR_INVALID),
    (dict(path=T(I32, [9, 3], data=None)), abi.AL_ERR_INVALID), (dict(lens=T(I32, [2])), abi.AL_ERR_INVALID),
    (dict(counts=T(F32, [3])), abi.AL_ERR_INVALID), (dict(kept=T(I32, [3], data=None)), abi.AL_ERR_INVALID),
    (dict(lens_out=T(I32, [3])), abi.AL_ERR_INVALID),                # lens itself
    (dict(lens_out=T(I32, [3], data=SOME + 8)), abi.AL_ERR_INVALID), (dict(path=T(I32, [65537, 3])), abi.AL_ERR_UNSUPPORTED)])
def test_keep_refuses(change, status):
    refused("al_paged_keep_f16", status, "paged_keep", keep_args(**(change if isinstance(change, dict) else dict(layers=change()))))


@pytest.mark.parametrize("change, status", LAYER_FAULTS + [
    (dict(src=T(I32, [2], data=None)), abi.AL_ERR_INVALID), (dict(dst=T(I32, [3])), abi.AL_ERR_INVALID), (dict(cells=T(I32, [1])), abi.AL_ERR_INVALID),
    (dict(src=T(I32, [65536]), dst=T(I32, [65536])), abi.AL_ERR_UNSUPPORTED)])
def test_copy_refuses(change, status):
    d = dict(layers=layers(), src=T(I32, [2]), dst=T(I32, [2]))
    refused("al_paged_copy_f16", status, "paged_copy", fill(abi.AlPagedCopyArgs(), {**d, **(change if isinstance(change, dict) else dict(layers=change()))}))


def test_null_arguments_and_empty_calls():
    lib = _lib.load()
    for entry in ("al_draft_tree_i32", "al_draft_verify_f32", "al_paged_keep_f16", "al_paged_copy_f16"):
        assert getattr(lib, entry)(None) == abi.AL_ERR_INVALID
    assert lib.al_draft_verify_workspace_bytes(None) == 0
    none = dict(parents=T(I32, [9, 0]), lens=T(I32, [0]), counts=T(I32, [0]), pos=T(I32, [9, 0]), cells=T(I32, [9, 0]), seq=T(I32, [9, 0]), bits=T(I32, [1, 9, 0]))
    assert lib.al_draft_tree_i32(ctypes.byref(tree_args(**none))) == abi.AL_OK
    none = dict(target=T(F32, [100, 9, 0]), tokens=T(I32, [9, 0]), parents=T(I32, [9, 0]), accept=T(F32, [9, 0]), sample=T(F32, [0]), path=T(I32, [9, 0]),
                kept=T(I32, [0]), next=T(I32, [0]))
    assert lib.al_draft_verify_f32(ctypes.byref(verify_args(**none))) == abi.AL_OK
    none = dict(table=T(I32, [5, 0]), lens=T(I32, [0]), counts=T(I32, [0]), path=T(I32, [9, 0]), kept=T(I32, [0]), lens_out=abi.empty_tensor())
    assert lib.al_paged_keep_f16(ctypes.byref(keep_args(**none))) == abi.AL_OK
    assert lib.al_paged_copy_f16(ctypes.byref(fill(abi.AlPagedCopyArgs(), dict(layers=layers(), src=T(I32, [0]), dst=T(I32, [0]))))) == abi.AL_OK


def test_struct_layouts_match_c(tmp_path):
    src = tmp_path / "probe.c"
    names = {"al_paged_sees": ("AlPagedSees", ["first", "bits", "pos"]), "al_paged_layers": ("AlPagedLayers", ["v_pool", "k", "v", "n_layers"]),
             "al_paged_keep_args": ("AlPagedKeepArgs", ["table", "path", "lens_out", "stream"]),
             "al_paged_copy_args": ("AlPagedCopyArgs", ["src", "cells", "stream"]),
             "al_draft_tree_args": ("AlDraftTreeArgs", ["lens", "bits", "stream"]),
             "al_draft_verify_args": ("AlDraftVerifyArgs", ["draft", "accept", "next", "stream", "workspace_bytes"])}
    body = "".join(f' printf("%zu {" ".join("%zu" for _ in f)}\\n", sizeof({s}), {", ".join(f"offsetof({s}, {x})" for x in f)});\n'
                   for s, (_, f) in names.items())
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "arclight_paged.h"\n#include "arclight_draft.h"\nint main(void) {\n' + body +
                   " return 0; }\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, (cls, f) in zip(lines, names.values()):
        c = getattr(abi, cls)
        assert [int(x) for x in line.split()] == [ctypes.sizeof(c)] + [getattr(c, x).offset for x in f]


def test_layers_of_different_shapes():
    from arclight_amd import paged

    class Pool:
        def __init__(self, shape, strides):
            self.shape, self.strides = shape, strides
    a, b = Pool((4, 16, 8, 128), (32768, 2048, 256, 2)), Pool((4, 16, 8, 128), (65536, 2048, 256, 2))
    with pytest.raises(ValueError, match="shape"):
        paged.CopyCall([paged.PagedCache(a, a, None), paged.PagedCache(a, b, None)], None, None)
    with pytest.raises(ValueError, match="layers"):
        paged.CopyCall([], None, None)
