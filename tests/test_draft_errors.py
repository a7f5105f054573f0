"""The texts of what the kernels of drafts, windows and moved cells record
(arclight_amd/csrc/device_errors.hpp, compiled by the host's compiler), beside
other kinds; and what the mirrors refuse themselves."""
import os
import shutil
import subprocess
from types import SimpleNamespace

import pytest

from arclight_amd import abi, paged

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path_factory.mktemp("draft_errors") / "probe")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-o", exe, os.path.join(HERE, "csrc", "device_errors.cpp")], check=True)

    def run(words):
        out = subprocess.run([exe, *(f"{k}={v}" for k, v in words.items())], capture_output=True, text=True, check=True).stdout
        status, text = out.rstrip("\n").split(" ", 1)
        return int(status), text
    return run


@pytest.mark.parametrize("what, value, text", [
    (1, 9, "draft: a node whose parent is 9,"), (2, -4, "draft: a tree of -4 nodes"), (3, 32000, "draft: a node of token 32000,"),
    (4, 3, "draft: sequence 3 has no probabilities")])
def test_drafts(report, what, value, text):
    status, got = report({12: 1, 13: what, 14: value})
    assert status == abi.AL_ERR_INVALID and got.startswith(text)
    status, got = report({12: 1, 13: what, 14: value, 2: 1, 4: 1, 5: 1, 6: 2})
    assert status == abi.AL_ERR_HIP and text in got and "gave up" in got and "sequence 2 has a page outside the pool" in got


@pytest.mark.parametrize("what, value, text", [
    (5, 70, "a token at position 70,"), (6, 71, "a token of cell 71,"), (7, 4, "new token 4 is not one that can be kept"), (8, 6, "a path of 6 tokens"),
    (9, 12, "page 12 of a copy"), (10, 17, "a copy of 17 cells")])
def test_cells(report, what, value, text):
    assert report({4: 1, 5: what, 6: value})[1].startswith("paged cache: " + text)


def _cache(shape, table=None):
    pool = SimpleNamespace(shape=shape, strides=(1,) * 4, ptr=4096)
    return SimpleNamespace(k=pool, v=pool, heads_first=False, table=table, pool_descs=lambda: (abi.empty_tensor(), abi.empty_tensor()))


def test_layers_that_do_not_go_together():
    a, b = _cache((8, 16, 2, 128)), _cache((9, 16, 2, 128))
    for caches in ([], [a, b]):
        with pytest.raises(ValueError):
            paged.CopyCall(caches, None, None)
        with pytest.raises(ValueError):
            paged.KeepCall(caches, None, None, None, None)
    with pytest.raises(ValueError, match="table"):
        paged.KeepCall([a, a], None, None, None, None)


@pytest.mark.parametrize("entry, names", [("al_draft_tree_i32", ("pos", "cells", "seq", "bits")), ("al_draft_verify_f32", ("path", "kept", "next"))])
def test_outputs_that_are_other_operands(entry, names):
    """Each operand at an address of its own, but one that two share (of memory
    that refused calls never touch)."""
    import ctypes

    from arclight_amd import _lib
    from tests.test_draft_refusals import tree_args, verify_args
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    for i, out in enumerate(names):
        a = tree_args() if entry == "al_draft_tree_i32" else verify_args()
        operands = [n for n, t in a._fields_ if t is abi.AlTensor and getattr(a, n).data]
        for j, n in enumerate(operands):
            getattr(a, n).data = 0x10000 * (j + 1)
        other = next(n for n in operands[i:] + operands if n not in names[:i + 1])
        getattr(a, out).data = getattr(a, other).data
        assert getattr(lib, entry)(ctypes.byref(a)) == abi.AL_ERR_INVALID
        assert "another operand's memory" in lib.al_last_error().decode()


def test_new_lengths_inside_the_path_or_the_table():
    import ctypes

    from arclight_amd import _lib
    from tests.test_draft_refusals import keep_args
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    for name in ("path", "table"):
        a = keep_args()
        getattr(a, name).data = 0x70000
        for at in (0x70000 - 8, 0x70000 + 4 * (5 if name == "table" else 9) * 3 - 4):
            a.lens_out.data = at
            assert lib.al_paged_keep_f16(ctypes.byref(a)) == abi.AL_ERR_INVALID
            assert "overlaps" in lib.al_last_error().decode()
