"""What the paged-cache entry points refuse, before any device call (CPU), and
the argument structures' layouts."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from arclight_amd import _lib, abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (run python -m arclight_amd.build)")
F32, F16, I32 = abi.AL_TYPE_F32, abi.AL_TYPE_F16, abi.AL_TYPE_I32
SOME = 0x10000                      # an address that refused calls never touch


def T(typ, ne, data=SOME, nb=None):
    return abi.make_tensor(data, typ, ne, nb)


def fattn_args(**kw):
    a = abi.AlPagedFattnArgs()
    d = dict(q=T(F32, [128, 1, 32, 3]), dst=T(F32, [128, 32, 1, 3]), k_pool=T(F16, [128, 16, 8, 10]),
             v_pool=T(F16, [128, 16, 8, 10]), table=T(I32, [5, 3]), lens=T(I32, [3]), scale=0.1)
    d.update(kw)
    for n, v in d.items():
        setattr(a, n, v)
    return a


def append_args(**kw):
    a = abi.AlPagedAppendArgs()
    d = dict(q=T(F32, [128, 32, 4]), q_out=T(F32, [128, 32, 4]), k=T(F32, [128, 8, 4]), v=T(F32, [128, 8, 4]),
             pos=T(I32, [4]), seq=T(I32, [4]), k_pool=T(F16, [128, 16, 8, 10]), v_pool=T(F16, [128, 16, 8, 10]),
             table=T(I32, [5, 3]), eps=1e-6, norm=1)
    d.update(kw)
    for n, v in d.items():
        setattr(a, n, v)
    return a


POOL_FAULTS = [
    (dict(k_pool=T(F16, [128, 16, 8, 10], data=None)), abi.AL_ERR_INVALID),
    (dict(table=T(I32, [5, 3], data=None)), abi.AL_ERR_INVALID),
    (dict(k_pool=T(F32, [128, 16, 8, 10])), abi.AL_ERR_UNSUPPORTED),
    (dict(k_pool=T(F16, [64, 16, 8, 10])), abi.AL_ERR_UNSUPPORTED),
    (dict(v_pool=T(F16, [128, 16, 8, 9])), abi.AL_ERR_INVALID),
    (dict(k_pool=T(F16, [128, 12, 8, 10]), v_pool=T(F16, [128, 12, 8, 10])), abi.AL_ERR_UNSUPPORTED),
    (dict(k_pool=T(F16, [128, 16, 8, 10], data=SOME + 8)), abi.AL_ERR_INVALID),
    (dict(k_pool=T(F16, [128, 16, 8, 10], nb=[2, 264, 4224, 33792])), abi.AL_ERR_INVALID),
    (dict(k_pool=T(F16, [128, 16, 8, 10], nb=[4, 512, 8192, 65536])), abi.AL_ERR_INVALID),
    (dict(table=T(abi.AL_TYPE_I64, [5, 3])), abi.AL_ERR_INVALID),
    (dict(table=T(I32, [1 << 27, 3])), abi.AL_ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("change, status", POOL_FAULTS + [
    (dict(q=T(F32, [128, 1024, 4095, 3]), dst=T(F32, [128, 4095, 1024, 3]), k_pool=T(F16, [128, 16, 1, 10]),
          v_pool=T(F16, [128, 16, 1, 10])), abi.AL_ERR_UNSUPPORTED),    # rows x heads past 32 bits: the division is not exact
    (dict(q=T(F32, [128, 1, 32, 65]), dst=T(F32, [128, 32, 1, 65]), table=T(I32, [1 << 26, 65]), lens=T(I32, [65])),
     abi.AL_ERR_UNSUPPORTED),                                          # tiles of all sequences past 31 bits
    (dict(q=T(F32, [128, 1, 32, 3], data=None)), abi.AL_ERR_INVALID),
    (dict(lens=T(I32, [3], data=None)), abi.AL_ERR_INVALID),
    (dict(q=T(F16, [128, 1, 32, 3])), abi.AL_ERR_UNSUPPORTED),
    (dict(q=T(F32, [64, 1, 32, 3])), abi.AL_ERR_UNSUPPORTED),
    (dict(dst=T(F32, [128, 32, 1, 4])), abi.AL_ERR_INVALID),
    (dict(dst=T(F32, [128, 32, 1, 3], data=SOME + 4)), abi.AL_ERR_INVALID),
    (dict(q=T(F32, [128, 1, 30, 3]), dst=T(F32, [128, 30, 1, 3])), abi.AL_ERR_INVALID),
    (dict(q=T(F32, [128, 1, 32, 2]), dst=T(F32, [128, 32, 1, 2])), abi.AL_ERR_INVALID),
    (dict(lens=T(I32, [2])), abi.AL_ERR_INVALID),
    (dict(lens=T(abi.AL_TYPE_I64, [3])), abi.AL_ERR_INVALID),
    (dict(counts=T(I32, [4])), abi.AL_ERR_INVALID),
    (dict(sinks=T(F32, [8])), abi.AL_ERR_INVALID),
    (dict(logit_softcap=-1.0), abi.AL_ERR_INVALID),
    (dict(logit_softcap=float("nan")), abi.AL_ERR_INVALID),
])
def test_attention_refuses(change, status):
    lib = _lib.load()
    a = fattn_args(**change)
    assert lib.al_paged_fattn_f16(ctypes.byref(a)) == status
    assert lib.al_last_error().decode().startswith("paged_fattn")


@pytest.mark.parametrize("change, status", POOL_FAULTS + [
    (dict(k=T(F32, [128, 8, 4], data=None)), abi.AL_ERR_INVALID),
    (dict(k=T(F32, [128, 4, 4])), abi.AL_ERR_INVALID),
    (dict(v=T(F32, [128, 8, 3])), abi.AL_ERR_INVALID),
    (dict(q_out=T(F32, [128, 32, 4], data=None)), abi.AL_ERR_INVALID),
    (dict(q=T(F32, [128, 32, 5])), abi.AL_ERR_INVALID),
    (dict(pos=T(I32, [3])), abi.AL_ERR_INVALID),
    (dict(seq=T(I32, [4], data=None)), abi.AL_ERR_INVALID),
    (dict(q_w=T(F32, [64])), abi.AL_ERR_INVALID),
    (dict(norm=0, k_w=T(F32, [128])), abi.AL_ERR_INVALID),
    (dict(eps=-1.0), abi.AL_ERR_INVALID),
    (dict(rope=ctypes.pointer(abi.AlRopeParams(64, abi.AL_ROPE_NEOX, 4096, 1e6, 1.0, 0.0, 1.0, 32.0, 1.0))), abi.AL_ERR_UNSUPPORTED),
    (dict(rope=ctypes.pointer(abi.AlRopeParams(128, 7, 4096, 1e6, 1.0, 0.0, 1.0, 32.0, 1.0))), abi.AL_ERR_UNSUPPORTED),
])
def test_append_refuses(change, status):
    lib = _lib.load()
    a = append_args(**change)
    assert lib.al_paged_append_f32(ctypes.byref(a)) == status
    assert lib.al_last_error().decode().startswith("paged_append")


def test_null_arguments_and_empty_calls():
    lib = _lib.load()
    assert lib.al_paged_fattn_f16(None) == abi.AL_ERR_INVALID
    assert lib.al_paged_append_f32(None) == abi.AL_ERR_INVALID
    assert lib.al_paged_fattn_workspace_bytes(None) == 0
    # no sequences, no tokens: nothing to do
    a = fattn_args(q=T(F32, [128, 1, 32, 0]), dst=T(F32, [128, 32, 1, 0]), table=T(I32, [5, 0]), lens=T(I32, [0]))
    assert lib.al_paged_fattn_f16(ctypes.byref(a)) == abi.AL_OK
    a = fattn_args(q=T(F32, [128, 0, 32, 3]), dst=T(F32, [128, 32, 0, 3]))
    assert lib.al_paged_fattn_f16(ctypes.byref(a)) == abi.AL_OK
    a = append_args(q=T(F32, [128, 32, 0]), q_out=T(F32, [128, 32, 0]), k=T(F32, [128, 8, 0]), v=T(F32, [128, 8, 0]),
                    pos=T(I32, [0]), seq=T(I32, [0]))
    assert lib.al_paged_append_f32(ctypes.byref(a)) == abi.AL_OK


def test_struct_layouts_match_c(tmp_path):
    src = tmp_path / "probe.c"
    names = {"al_paged_append_args": ("AlPagedAppendArgs", ["k", "table", "eps", "norm", "rope", "stream"]),
             "al_paged_fattn_args": ("AlPagedFattnArgs", ["table", "dst", "scale", "stream", "workspace_bytes"])}
    body = "".join(f' printf("%zu {" ".join("%zu" for _ in f)}\\n", sizeof({s}), {", ".join(f"offsetof({s}, {x})" for x in f)});\n'
                   for s, (_, f) in names.items())
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "arclight_paged.h"\nint main(void) {\n' + body + " return 0; }\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, (cls, f) in zip(lines, names.values()):
        c = getattr(abi, cls)
        assert [int(x) for x in line.split()] == [ctypes.sizeof(c)] + [getattr(c, x).offset for x in f]


def test_page_index_by_multiplication_is_exact():
    """page_of_group's umulhi by ceil(2^32 / d) equals the division wherever
    the host lets a table through: at every page's first and last group."""
    for d in (2, 3, 5, 6, 7, 12, 31, 100, 8191, 131072):
        magic = (2 ** 32 + d - 1) // d
        top = min(2 ** 27, 2 ** 32 // d - 1)
        rng = np.random.default_rng(d)
        x = np.unique(np.concatenate([np.arange(0, min(top, 5000)), rng.integers(0, top, 20000), np.arange(max(0, top - 2000), top)]))
        edge = x // d * d
        x = np.unique(np.concatenate([x, edge, np.maximum(edge, 1) - 1])).astype(np.uint64)
        assert np.array_equal(x * np.uint64(magic) >> np.uint64(32), x // np.uint64(d))
