"""What the adapter entry points refuse, before any device call (CPU), and the
argument structure's layout."""
import ctypes
import os
import subprocess

import pytest

from arclight_amd import _lib, abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (run python -m arclight_amd.build)")
F32, F16, I32, Q4 = abi.AL_TYPE_F32, abi.AL_TYPE_F16, abi.AL_TYPE_I32, abi.AL_TYPE_Q4_0
SOME = 0x10000                      # an address that refused calls never touch


def T(typ, ne, data=SOME, nb=None):
    return abi.make_tensor(data, typ, ne, nb)


def args(**kw):
    a = abi.AlLoraArgs()
    d = dict(a=T(F16, [4096, 16, 5]), b=T(F16, [16, 2560, 5]), ids=T(I32, [3]), x=T(F32, [4096, 3]), base=T(F32, [2560, 3], SOME << 12),
             y=T(F32, [2560, 3]), w=T(Q4, [4096, 2560], nb=[18, 2304, 2304 * 2560, 2304 * 2560]))
    d.update(kw)
    for n, v in d.items():
        setattr(a, n, v)
    return a


FAULTS = [
    (dict(a=T(F16, [4096, 16, 5], data=None)), abi.AL_ERR_INVALID),
    (dict(ids=T(I32, [3], data=None)), abi.AL_ERR_INVALID),
    (dict(a=T(F32, [4096, 16, 5])), abi.AL_ERR_UNSUPPORTED),
    (dict(x=T(F16, [4096, 3])), abi.AL_ERR_UNSUPPORTED),
    (dict(b=T(F16, [8, 2560, 5])), abi.AL_ERR_INVALID),
    (dict(b=T(F16, [16, 2560, 4])), abi.AL_ERR_INVALID),
    (dict(x=T(F32, [2048, 3])), abi.AL_ERR_INVALID),
    (dict(y=T(F32, [2560, 4])), abi.AL_ERR_INVALID),
    (dict(a=T(F16, [4096, 12, 5]), b=T(F16, [12, 2560, 5])), abi.AL_ERR_UNSUPPORTED),
    (dict(a=T(F16, [4096, 136, 5]), b=T(F16, [136, 2560, 5])), abi.AL_ERR_UNSUPPORTED),
    (dict(a=T(F16, [4096, 16, 5], data=SOME + 2)), abi.AL_ERR_INVALID),
    (dict(b=T(F16, [16, 2560, 5], nb=[2, 36, 36 * 2560, 0])), abi.AL_ERR_INVALID),
    (dict(x=T(F32, [4096, 3], data=SOME + 4)), abi.AL_ERR_INVALID),
    (dict(y=T(F32, [2560, 3], nb=[4, 2560, 0, 0])), abi.AL_ERR_INVALID),
    (dict(ids=T(I32, [2])), abi.AL_ERR_INVALID),
    (dict(ranks=T(I32, [4])), abi.AL_ERR_INVALID),
    (dict(scales=T(F16, [5])), abi.AL_ERR_INVALID),
    (dict(a=T(F16, [4096, 16, 5], nb=[2, 1 << 28, 1 << 32, 5 << 32])), abi.AL_ERR_UNSUPPORTED),    # an adapter's A of 4 GB
    (dict(b=T(F16, [16, 2560, 5], nb=[2, 1 << 21, 2560 << 21, 12800 << 21])), abi.AL_ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("change, status", FAULTS + [
    (dict(base=T(F32, [2560, 2], SOME << 12)), abi.AL_ERR_INVALID),
    (dict(base=T(F32, [2560, 3], SOME + 4)), abi.AL_ERR_INVALID),     # overlaps y
    (dict(a=T(F16, [4100, 16, 5]), x=T(F32, [4100, 3])), abi.AL_ERR_UNSUPPORTED),
])
def test_apply_refuses(change, status):
    lib = _lib.load()
    assert lib.al_lora_f32(ctypes.byref(args(**change))) == status
    assert lib.al_last_error().decode().startswith("lora")


@pytest.mark.parametrize("change, status", FAULTS + [
    (dict(w=T(Q4, [4096, 2560], data=None, nb=[18, 2304, 0, 0])), abi.AL_ERR_INVALID),
    (dict(w=T(F16, [4096, 2560])), abi.AL_ERR_UNSUPPORTED),
    (dict(ids=T(I32, [65]), x=T(F32, [4096, 65]), y=T(F32, [2560, 65])), abi.AL_ERR_UNSUPPORTED),
    (dict(a=T(F16, [2560, 16, 5]), x=T(F32, [2560, 3])), abi.AL_ERR_INVALID),
])
def test_project_refuses(change, status):
    lib = _lib.load()
    assert lib.al_mul_mat_q4_0_lora_f32(ctypes.byref(args(**change))) == status


def test_null_arguments_and_empty_calls():
    lib = _lib.load()
    assert lib.al_lora_f32(None) == abi.AL_ERR_INVALID and lib.al_mul_mat_q4_0_lora_f32(None) == abi.AL_ERR_INVALID
    assert lib.al_lora_workspace_bytes(None) == 0
    a = args(ids=T(I32, [0]), x=T(F32, [4096, 0]), y=T(F32, [2560, 0]), base=T(F32, [2560, 0]))
    assert lib.al_lora_f32(ctypes.byref(a)) == abi.AL_OK


def test_struct_layout_matches_c(tmp_path):
    src = tmp_path / "probe.c"
    fields = ["ids", "base", "w", "stream", "workspace", "workspace_bytes"]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "arclight_lora.h"\nint main(void) {\n'
                   ' printf("%zu' + " %zu" * len(fields) + '", sizeof(al_lora_args), '
                   + ", ".join(f"offsetof(al_lora_args, {f})" for f in fields) + ");\n return 0; }\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(abi.AlLoraArgs)] + [getattr(abi.AlLoraArgs, f).offset for f in fields]


def test_base_beside_y_in_one_matrix_is_not_refused():
    """Columns of one wider matrix, in either order, are apart; those that
    share a column are not. (T = 3 rows; the workspace's size tells, or, where
    there is no device, the refusal's absence.)"""
    lib = _lib.load()
    N, row = 2560, 2 * 2560 * 4
    wide = lambda off: T(F32, [N, 3], SOME + off, [4, row, 0, 0])  # noqa: E731
    small = T(F32, [N, 3], SOME, [4, row, 0, 0])
    for base, y, refused in ((wide(N * 4), small, False), (small, wide(N * 4), False), (wide(N * 4 - 4), small, True),
                             (small, wide(N * 4 - 4), True), (wide(N * 4 + 4), small, True), (wide(row), small, True)):
        a = args(base=base, y=y, ids=T(I32, [3]), workspace=SOME, workspace_bytes=1)
        status = lib.al_lora_f32(ctypes.byref(a))                      # too small a workspace: nothing runs
        assert (status == abi.AL_ERR_INVALID) == refused and status != abi.AL_OK, (status, lib.al_last_error())
