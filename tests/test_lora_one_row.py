"""A call of one row, whose strides are of no use: a base at y's address is y
(CPU: the sizes are accepted; GPU: the result)."""
import ctypes
import os

import numpy as np
import pytest

from arclight_amd import _lib, abi
from tests.test_lora_refusals import F32, I32, SOME, T, args

N = 2560


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (run python -m arclight_amd.build)")
@pytest.mark.parametrize("stride", [N * 4, 3 * N * 4, 4, 0])
def test_base_at_ys_address_is_y(stride):
    lib = _lib.load()
    a = args(ids=T(I32, [1]), x=T(F32, [4096, 1]), y=T(F32, [N, 1]), base=T(F32, [N, 1], SOME, [4, stride, 0, 0]),
             workspace=SOME, workspace_bytes=1)
    status = lib.al_lora_f32(ctypes.byref(a))                          # too small a workspace: nothing runs
    assert status not in (abi.AL_OK, abi.AL_ERR_INVALID), lib.al_last_error()


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (run python -m arclight_amd.build)")
def test_two_rows_of_other_strides_overlap():
    lib = _lib.load()
    a = args(ids=T(I32, [2]), x=T(F32, [4096, 2]), y=T(F32, [N, 2]), base=T(F32, [N, 2], SOME, [4, 3 * N * 4, 0, 0]),
             workspace=SOME, workspace_bytes=1)
    assert lib.al_lora_f32(ctypes.byref(a)) == abi.AL_ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("id_", [1, -1])
def test_one_row_of_a_wider_matrix(gpu, id_):
    from arclight_amd import device, lora
    print(f"\n[case] lora: one row, base is y with another stride, id {id_}", flush=True)
    rng = np.random.default_rng(2)
    put = device.DeviceTensor.from_numpy
    a, b = (rng.integers(-2, 3, s).astype(np.float16) for s in ((2, 8, 64), (2, 32, 8)))      # sums below 2^24: exact
    x, base = (rng.integers(-3, 4, s).astype(np.float32) for s in ((1, 64), (1, 32)))
    y = put(base)
    wide = device.DeviceTensor(y.buf, abi.AL_TYPE_F32, (1, 32), (100 * 4, 4))
    lora.apply(lora.Adapters(put(a.view(np.uint16)), put(b.view(np.uint16))), put(x), put(np.array([id_], np.int32)), wide, y)
    device.synchronize()
    want = base[0] + (0 if id_ < 0 else b[id_].astype(np.float32) @ (a[id_].astype(np.float32) @ x[0]))
    assert np.array_equal(y.numpy(np.float32)[0], want)
