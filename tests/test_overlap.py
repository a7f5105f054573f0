"""Outputs in another operand's memory: overlap() of strided operands
(arclight_amd/csrc/overlap.hpp, compiled by the host's compiler) against their
bytes, and what the entry points for drafts refuse by it (CPU)."""
import ctypes
import os
import shutil
import subprocess

import pytest

from arclight_amd import _lib, abi
from tests.test_draft_refusals import tree_args, verify_args
from tests.test_paged_refusals import T

HERE = os.path.dirname(os.path.abspath(__file__))
built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
I32 = abi.AL_TYPE_I32


def test_against_the_bytes(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "probe")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", exe, os.path.join(HERE, "csrc", "overlap.cpp")], check=True)
    shared, gaps, wrong, careful = map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split())
    assert wrong == 0 and shared > 1000 and gaps > 1000 and careful < gaps


def _apart(a):
    """Every operand at an address of its own."""
    names = [n for n, t in a._fields_ if t is abi.AlTensor and getattr(a, n).data]
    for j, n in enumerate(names):
        getattr(a, n).data = 0x10000 * (j + 1)
    return names


def _refused(entry, a):
    lib = _lib.load()
    status = getattr(lib, entry)(ctypes.byref(a))
    text = lib.al_last_error().decode() if status != abi.AL_OK else ""
    return status == abi.AL_ERR_INVALID and "another operand's memory" in text


def _bytes(t):
    return 4 + sum((t.ne[i] - 1) * t.nb[i] for i in range(4))


CALLS = [("al_draft_tree_i32", tree_args, ("pos", "cells", "seq", "bits")), ("al_draft_verify_f32", verify_args, ("path", "kept", "next"))]


@built
@pytest.mark.parametrize("entry, args, outs", CALLS)
def test_outputs_that_begin_inside_another_operand(entry, args, outs):
    """An output from 4 bytes behind another operand's beginning on, on its last
    4 bytes, and with its own last 4 bytes in it."""
    for i, out in enumerate(outs):
        for n in _apart(args()):
            if n == out or n in outs[:i]:
                continue
            for where in ("inside", "last", "ends in it"):
                a = args()
                _apart(a)
                t, own = getattr(a, n), getattr(a, out)
                if where == "inside" and _bytes(t) <= 4:
                    continue
                own.data = t.data + {"inside": 4, "last": _bytes(t) - 4, "ends in it": 4 - _bytes(own)}[where]
                assert _refused(entry, a), (out, n, where)


# The accepted ones of these go on to the device: not with addresses that are none.
@built
@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="for machines without a GPU")
def test_operands_side_by_side_are_taken():
    """Behind one another without a gap, and tables of one record for each
    sequence, in one another's gaps."""
    a = tree_args()
    at = 0x10000
    for n in _apart(a):
        t = getattr(a, n)
        t.data, at = at, at + _bytes(t)
    assert not _refused("al_draft_tree_i32", a)
    # [sequence][pos | cells | seq | bits | parents] of 9 words each
    row = 5 * 36
    record = {n: T(I32, [9, 3], data=0x10000 + 36 * i, nb=[4, row, 3 * row, 3 * row]) for i, n in enumerate(("pos", "cells", "seq"))}
    record["bits"] = T(I32, [1, 9, 3], data=0x10000 + 108, nb=[4, 4, row, 3 * row])
    record["parents"] = T(I32, [9, 3], data=0x10000 + 144, nb=[4, row, 3 * row, 3 * row])
    a = tree_args(lens=T(I32, [3], data=0x20000), counts=T(I32, [3], data=0x30000), **record)
    assert not _refused("al_draft_tree_i32", a)
    a.bits.data -= 4
    assert _refused("al_draft_tree_i32", a)


@built
def test_outputs_of_no_nodes():
    """T = 0: kept and next are written all the same."""
    a = verify_args(target=T(abi.AL_TYPE_F32, [100, 0, 3]), tokens=T(I32, [0, 3]), parents=abi.empty_tensor(), accept=T(abi.AL_TYPE_F32, [0, 3]),
                    path=T(I32, [0, 3]))
    _apart(a)
    a.next.data = a.kept.data + 8
    assert _refused("al_draft_verify_f32", a)
