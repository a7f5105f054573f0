"""Threads that each call on hipStreamPerThread, one handle for as many streams
as there are threads: each has workspaces of its own, so that calls which
overlap give the bits that they give alone."""
import threading
import types

import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu
PER_THREAD = types.SimpleNamespace(handle=2)                          # hipStreamPerThread


def test_two_threads_on_their_default_streams(gpu):
    from arclight_amd import _lib, device, fattn, lora, matmul
    print("\n[case] projection and adapters on two threads' default streams", flush=True)
    lib, put = _lib.load(), device.DeviceTensor.from_numpy
    K, N, R, T = 4096, 2560, 32, 48

    class Side:
        def __init__(self, seed):
            rng = np.random.default_rng(seed)
            self.w = matmul.Q4_0Matrix(O.random_q4_0(rng, N, K).view(np.uint8), K, N)
            self.x, self.ids = put(rng.standard_normal((T, K)).astype(np.float32)), put(rng.integers(-1, 3, T).astype(np.int32))
            a, b = (rng.standard_normal(s).astype(np.float16) * np.float16(0.1) for s in ((3, R, K), (3, N, R)))
            self.ad = lora.Adapters(put(a.view(np.uint16)), put(b.view(np.uint16)))
            self.base = put(rng.standard_normal((T, N)).astype(np.float32))
            self.ys = [[device.DeviceTensor.empty((T, N), np.float32) for _ in range(20)] for _ in range(2)]
            self.error = None

        def calls(self, i, stream):
            matmul.mul_mat_q4_0(self.w, self.x, self.ys[0][i], stream=stream)
            lora.apply(self.ad, self.x, self.ids, self.base, self.ys[1][i], stream=stream)

        def thread(self, barrier):
            try:
                barrier.wait(30)
                for i in range(20):
                    self.calls(i, PER_THREAD)
                _lib.call("al_util_stream_synchronize", PER_THREAD.handle)
                _lib.call("al_fattn_release_stream", PER_THREAD.handle)
            except Exception as e:  # noqa: BLE001
                self.error = e

    sides = [Side(i) for i in range(2)]
    want = []
    for s in sides:
        s.calls(0, None)
        device.synchronize()
        want.append([y[0].numpy(np.float32).copy() for y in s.ys])
        for y in s.ys:
            y[0].buf.zero()
    device.synchronize()
    barrier = threading.Barrier(2)
    threads = [threading.Thread(target=s.thread, args=(barrier,)) for s in sides]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    device.synchronize()
    fattn.device_errors()
    for s, w in zip(sides, want):
        assert s.error is None, s.error
        for y, ref in zip(s.ys, w):
            assert all(np.array_equal(d.numpy(np.float32), ref) for d in y)
    assert lib.al_fattn_release_stream(PER_THREAD.handle) == 0          # this thread has none
