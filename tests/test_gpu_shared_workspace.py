"""One caller's workspace for calls of different kinds, one after another on a
stream: al_fattn_f16, whose counters and epochs at its start live from call to
call, the paged attention and the adapters, which leave them alone."""
import math

import numpy as np
import pytest

from oracle import oracle as O
from tests import paged_cases as P
from tests.fattn_cases import assert_parity

pytestmark = pytest.mark.gpu
COUNTERS = 256 << 10
D = 128


def _put(x):
    from arclight_amd import device
    return device.DeviceTensor.from_numpy(np.ascontiguousarray(x))


def _paged(rng):
    from arclight_amd import device, paged
    lens = [2000, 900]
    pool = P.Pool(rng, lens, 2, 16)
    q = rng.standard_normal((2, 1, 8, D)).astype(np.float32)
    out = device.DeviceTensor.empty(q.shape, np.float32)
    want = P.attention(pool, q, lens, [1, 1], 1 / math.sqrt(D))
    cache, dq, dl = pool.device(), _put(q), _put(np.array(lens, np.int32))
    return lambda ws: paged.AttentionCall(cache, dq, dl, out, scale=1 / math.sqrt(D), workspace=ws), out, want


def _lora(rng, T, project):
    from arclight_amd import device, lora, matmul
    K, N, R = 4096, 256, 16
    a, b = (rng.standard_normal(s).astype(np.float16) for s in ((2, R, K), (2, N, R)))
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    x, ids, base = _put(rng.standard_normal((T, K)).astype(np.float32)), _put(rng.integers(0, 2, T).astype(np.int32)), _put(np.zeros((T, N), np.float32))
    y = device.DeviceTensor.empty((T, N), np.float32)
    w = matmul.Q4_0Matrix(O.random_q4_0(rng, N, K).view(np.uint8), K, N)
    if project:
        return lambda ws: lora.ProjectCall(ad, w, x, ids, y, workspace=ws)
    return lambda ws: lora.ApplyCall(ad, x, ids, base, y, workspace=ws)


@pytest.mark.parametrize("what", ["paged", "adapters", "few adapters", "projection"])
def test_the_counters_are_left_alone(gpu, what):
    from arclight_amd import device, fattn
    print(f"\n[case] workspace's first 256 KiB, {what}", flush=True)
    rng = np.random.default_rng(40)
    make = _paged(rng)[0] if what == "paged" else _lora(rng, 100 if what == "adapters" else 20, what == "projection")
    need = make(None).workspace_bytes()
    assert need > COUNTERS
    ws = device.DeviceBuffer(need)
    ws.upload(np.full(need, 0xa5, np.uint8))
    make(ws).run()
    device.synchronize()
    fattn.device_errors()
    got = ws.download(np.empty(need, np.uint8))
    assert np.all(got[:COUNTERS] == 0xa5) and not np.all(got[COUNTERS:] == 0xa5)


def test_one_workspace_for_all(gpu):
    """A split decode before and after the others, each time as alone."""
    from arclight_amd import abi, device, fattn
    print("\n[case] one workspace for attention, paged attention and adapters", flush=True)
    rng = np.random.default_rng(41)
    q, k, v = O.make_inputs(41, T=1, Hq=32, Hkv=8, n_kv=4096)
    ref = O.attention(q, k, v, scale=1 / math.sqrt(D), kv_len=4000)
    dq, dk, dv = fattn.upload_q(q), fattn.upload_kv(k), fattn.upload_kv(v)
    dst = device.DeviceTensor.empty(q.shape, np.float32, axes=abi.DST_AXES)
    need = fattn.workspace_bytes(dq, dk, dv, None, None, dst, scale=1 / math.sqrt(D), kv_len=4000)
    assert need > COUNTERS
    paged_call, out, want = _paged(rng)
    others = [paged_call, _lora(rng, 100, False), _lora(rng, 20, True)]
    ws = device.DeviceBuffer(max([need] + [m(None).workspace_bytes() for m in others]))
    ws.zero()
    for i in range(3):
        dst.buf.zero()
        fattn.flash_attn_ext(dq, dk, dv, None, scale=1 / math.sqrt(D), kv_len=4000, dst=dst, workspace=ws)
        for m in others:
            m(ws).run()
        device.synchronize()
        fattn.device_errors()
        assert_parity(dst.numpy(np.float32), ref, what=f"decode {i}")
        got = out.numpy(np.float32)
        assert np.all(np.abs(got - want[0]) <= want[1])
