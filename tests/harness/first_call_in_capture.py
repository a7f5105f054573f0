"""A process whose first calls of the library are captured ones: the Q4_0
projection of 5 and of 20 tokens and an append to a paged cache, replayed
against eager calls afterwards. Prints "ok"."""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
from arclight_amd import device, fattn, matmul, paged  # noqa: E402

rng = np.random.default_rng(1)
put = device.DeviceTensor.from_numpy
K, N, D = 4096, 64, 128
blocks = rng.integers(0, 256, (N, K // 32, 18)).astype(np.uint8)
blocks[..., 1] = 0x30                                                 # scales of ordinary size
w = matmul.Q4_0Matrix(blocks, K, N)
x = [put(rng.standard_normal((T, K)).astype(np.float32)) for T in (5, 20)]
y = [device.DeviceTensor.empty((T, N), np.float32) for T in (5, 20)]
pools = [put(np.zeros((2, 16, 1, D), np.uint16)) for _ in range(2)]
cache = paged.PagedCache(*pools, put(np.array([[1, 0]], np.int32)))
k, pos, seq = put(rng.standard_normal((3, 1, D)).astype(np.float32)), put(np.array([0, 17, 5], np.int32)), put(np.zeros(3, np.int32))


def calls(stream):
    for a, b in zip(x, y):
        matmul.mul_mat_q4_0(w, a, b, stream=stream)
    paged.append(cache, None, k, k, pos, seq, norm=False, stream=stream)


def results():
    out = [t.numpy(np.float32).copy() for t in y] + [t.numpy(np.uint16).copy() for t in pools]
    for t in y + pools:
        t.buf.zero()
    device.synchronize()
    return out


st = device.Stream()
g = device.Graph(st, lambda: calls(st))
got = []
for _ in range(3):
    g.launch(st)
    st.synchronize()
    got.append(results())
calls(st)
st.synchronize()
fattn.device_errors()
want = results()
assert all(np.array_equal(a, b) for r in got for a, b in zip(r, want)) and np.any(want[0]) and np.any(want[1]) and np.any(want[2])
print("ok", flush=True)
