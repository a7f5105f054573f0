"""The Q4_0 projection of more than 8 tokens on several streams and in graphs:
each stream has memory of its own for the quantized activations, so that calls
which overlap give the bits that they give alone."""
import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu
K, N = 8192, 2560


def _case(name):
    print(f"\n[case] {name}", flush=True)


class Side:
    """A stream with its own weights, activations and (for "adapters")
    adapters; want: the bits that its call gives alone."""

    def __init__(self, seed, T, adapters):
        from arclight_amd import device, lora, matmul
        rng = np.random.default_rng(seed)
        self.stream = device.Stream()
        self.w = matmul.Q4_0Matrix(O.random_q4_0(rng, N, K).view(np.uint8), K, N)
        self.host_x = rng.standard_normal((T, K)).astype(np.float32)
        self.x = device.DeviceTensor.from_numpy(self.host_x)
        self.ad = None
        if adapters:
            a, b = (rng.standard_normal(s).astype(np.float16) * np.float16(0.1) for s in ((3, 16, K), (3, N, 16)))
            self.ad = lora.Adapters(device.DeviceTensor.from_numpy(a.view(np.uint16)), device.DeviceTensor.from_numpy(b.view(np.uint16)))
            self.ids = device.DeviceTensor.from_numpy(rng.integers(-1, 3, T).astype(np.int32))
        self.want = self.out(self.call())

    def call(self, y=None):
        from arclight_amd import lora, matmul
        if self.ad is not None:
            return lora.project(self.ad, self.w, self.x, self.ids, y, stream=self.stream)
        return matmul.mul_mat_q4_0(self.w, self.x, y, stream=self.stream)

    def out(self, y):
        self.stream.synchronize()
        return y.numpy(np.float32)

    def close(self):
        from arclight_amd import _lib
        assert _lib.load().al_fattn_release_stream(self.stream.handle) == 0
        self.stream.destroy()


@pytest.mark.parametrize("adapters", [False, True], ids=["plain", "adapters"])
@pytest.mark.parametrize("T", [16, 48])
def test_two_streams_at_once(gpu, T, adapters):
    from arclight_amd import device, fattn
    _case(f"projection on two streams, T={T}, adapters={adapters}")
    sides = [Side(T + i, T, adapters) for i in range(2)]
    assert not np.array_equal(sides[0].want, sides[1].want)
    ys = [[device.DeviceTensor.empty((T, N), np.float32) for _ in range(20)] for _ in sides]
    for i in range(20):
        for s, y in zip(sides, ys):
            s.call(y[i])
    device.synchronize()
    fattn.device_errors()
    for n, (s, y) in enumerate(zip(sides, ys)):
        for i, got in enumerate(y):
            assert np.array_equal(got.numpy(np.float32), s.want), f"stream {n}, call {i}"
        s.close()


@pytest.mark.parametrize("adapters", [False, True], ids=["plain", "adapters"])
def test_replays_beside_another_streams_calls(gpu, adapters):
    from arclight_amd import device, fattn
    T = 33
    _case(f"projection replayed beside another stream's calls, adapters={adapters}")
    one, other = Side(1, T, adapters), Side(2, T, adapters)
    y = device.DeviceTensor.empty((T, N), np.float32)
    y2 = [device.DeviceTensor.empty((T, N), np.float32) for _ in range(4)]
    g = device.Graph(one.stream, lambda: [one.call(y) for _ in range(4)])
    for i in range(5):
        y.buf.zero()
        device.synchronize()
        g.launch(one.stream)
        for d in y2:
            other.call(d)
        device.synchronize()
        assert np.array_equal(y.numpy(np.float32), one.want), f"replay {i}"
        assert all(np.array_equal(d.numpy(np.float32), other.want) for d in y2), f"beside replay {i}"
    fattn.device_errors()
    g.destroy()
    one.close()
    other.close()


def test_a_streams_first_call_in_a_capture(gpu):
    """The first call of more than 8 tokens on a stream may be a captured one;
    the memory is kept for the graph beside eager calls of other sizes, given
    back on request, and made anew by a later call."""
    from arclight_amd import _lib, device, matmul
    T = 20
    _case("projection: first call of a stream in a capture")
    s = Side(3, T, False)
    st = device.Stream()
    y = device.DeviceTensor.empty((T, N), np.float32)
    g = device.Graph(st, lambda: matmul.mul_mat_q4_0(s.w, s.x, y, stream=st))
    big = device.DeviceTensor.from_numpy(np.concatenate([s.host_x] * 3))
    for i in range(3):
        y.buf.zero()
        device.synchronize()
        g.launch(st)
        st.synchronize()
        assert np.array_equal(y.numpy(np.float32), s.want), f"replay {i}"
        got = s.out(matmul.mul_mat_q4_0(s.w, big, stream=s.stream))    # 60 tokens
        assert all(np.array_equal(got[j * T:(j + 1) * T], s.want) for j in range(3))
    g.destroy()
    for _ in range(2):
        assert _lib.load().al_fattn_release_stream(st.handle) == 0
        y.buf.zero()
        device.synchronize()
        matmul.mul_mat_q4_0(s.w, s.x, y, stream=st)
        st.synchronize()
        assert np.array_equal(y.numpy(np.float32), s.want)
    assert _lib.load().al_fattn_release_stream(st.handle) == 0
    st.destroy()
    s.close()
