"""What al_device_errors makes of the words that kernels recorded
(arclight_amd/csrc/device_errors.hpp, compiled by the host's compiler): every
kind is named, none hides another, and a merge that gave up keeps its status."""
import os
import shutil
import subprocess

import pytest

from arclight_amd import abi

HERE = os.path.dirname(os.path.abspath(__file__))
ROWS, MERGE, PAGED, LORA = {0: 1, 1: 70}, {2: 1}, {4: 1, 5: 2, 6: -3}, {8: 1, 9: 12}
TEXTS = {"rows": "set_rows: row index 70 ", "merge": "fattn: a merging workgroup gave up", "paged": "paged cache: a length of -3 cells",
         "lora": "lora: a row of adapter 12"}


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path_factory.mktemp("device_errors") / "probe")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-o", exe, os.path.join(HERE, "csrc", "device_errors.cpp")], check=True)

    def run(*kinds):
        words = {k: v for d in kinds for k, v in d.items()}
        out = subprocess.run([exe, *(f"{k}={v}" for k, v in words.items())], capture_output=True, text=True, check=True).stdout
        status, text = out.rstrip("\n").split(" ", 1)
        return int(status), text
    return run


@pytest.mark.parametrize("kinds, status", [
    ((), abi.AL_OK), (("rows",), abi.AL_ERR_INVALID), (("merge",), abi.AL_ERR_HIP), (("paged",), abi.AL_ERR_INVALID),
    (("lora",), abi.AL_ERR_INVALID), (("merge", "paged"), abi.AL_ERR_HIP), (("merge", "lora"), abi.AL_ERR_HIP),
    (("merge", "paged", "lora"), abi.AL_ERR_HIP), (("paged", "lora"), abi.AL_ERR_INVALID), (("rows", "merge"), abi.AL_ERR_INVALID),
    (("rows", "merge", "paged", "lora"), abi.AL_ERR_INVALID)])
def test_every_kind_is_reported(report, kinds, status):
    got, text = report(*({"rows": ROWS, "merge": MERGE, "paged": PAGED, "lora": LORA}[k] for k in kinds))
    assert got == status
    assert [k for k, t in TEXTS.items() if t in text] == [k for k in TEXTS if k in kinds], text


@pytest.mark.gpu
def test_two_kinds_at_once_on_the_device(gpu):
    """A page outside the pool and an adapter that is not there, in two calls
    before one report: both are named, and then both are cleared."""
    import numpy as np

    from arclight_amd import _lib, device, fattn, lora, paged
    put = device.DeviceTensor.from_numpy
    print("\n[case] two kinds of recorded errors", flush=True)
    pool = [put(np.zeros((2, 16, 1, 128), np.uint16)) for _ in range(2)]
    cache = paged.PagedCache(*pool, put(np.array([[5]], np.int32)))
    out = paged.attention(cache, put(np.ones((1, 1, 1, 128), np.float32)), put(np.array([3], np.int32)), scale=0.1)
    a, b = put(np.zeros((2, 8, 64), np.uint16)), put(np.zeros((2, 16, 8), np.uint16))
    y = lora.apply(lora.Adapters(a, b), put(np.ones((1, 64), np.float32)), put(np.array([2], np.int32)), put(np.ones((1, 16), np.float32)))
    device.synchronize()
    with pytest.raises(_lib.ArclightError) as e:
        fattn.device_errors()
    assert e.value.status == abi.AL_ERR_INVALID
    assert "sequence 0 has a page outside the pool" in str(e.value) and "adapter 2," in str(e.value)
    fattn.device_errors()
    assert np.all(np.isnan(out.numpy(np.float32))) and np.all(np.isnan(y.numpy(np.float32)))
