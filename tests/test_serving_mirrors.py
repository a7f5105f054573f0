"""What the Python mirrors of the serving operators refuse themselves (CPU)."""
import numpy as np
import pytest

from arclight_amd import lora


class _Shape:
    def __init__(self, *shape):
        self.shape = shape


def test_apply_without_base_wants_y():
    """The products are added to y's own content, and memory that was just
    allocated has none."""
    ad = lora.Adapters(_Shape(2, 16, 64), _Shape(2, 32, 16))
    with pytest.raises(ValueError, match="y"):
        lora.apply(ad, _Shape(3, 64), _Shape(3), None)


@pytest.mark.gpu
def test_apply_without_base_adds_to_y(gpu):
    from arclight_amd import device
    print("\n[case] lora: added to y", flush=True)
    rng = np.random.default_rng(1)
    put = device.DeviceTensor.from_numpy
    a, b = (rng.integers(-2, 3, s).astype(np.float16) for s in ((2, 8, 64), (2, 32, 8)))      # sums below 2^24: exact
    x, base = (rng.integers(-3, 4, s).astype(np.float32) for s in ((3, 64), (3, 32)))
    ids = np.array([1, -1, 0], np.int32)
    y = put(base)
    assert lora.apply(lora.Adapters(put(a.view(np.uint16)), put(b.view(np.uint16))), put(x), put(ids), None, y) is y
    device.synchronize()
    want = base.copy()
    for t in (0, 2):
        want[t] += b[ids[t]].astype(np.float32) @ (a[ids[t]].astype(np.float32) @ x[t])
    assert np.array_equal(y.numpy(np.float32), want)
