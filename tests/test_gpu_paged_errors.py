"""Errors of the paged attention that test_gpu_paged.py does not make: counts
below zero, in every block of 64 slots."""
import math

import numpy as np
import pytest

from arclight_amd import abi
from tests import paged_cases as P
from tests.test_gpu_paged import MARK, _case, _check, _put

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("n, slot", [(1, 0), (4, 2), (4, 3), (70, 3), (70, 66), (200, 199)])
def test_negative_counts_are_reported(gpu, n, slot, T):
    """A slot with a negative count is recorded and has no rows; the others
    are right. (One slot: no sequence has work at all.)"""
    from arclight_amd import _lib, device, fattn, paged
    _case(f"paged attention, a negative count in slot {slot} of {n}, T={T}")
    rng = np.random.default_rng(30 + n + slot)
    lens = [int(x) for x in rng.integers(T, 40, n)]
    counts = [T] * n
    counts[slot] = -3
    pool = P.Pool(rng, lens, 2, 16)
    q = rng.standard_normal((n, T, 8, D)).astype(np.float32)
    out = _put(np.full(q.shape, MARK, np.float32))
    call = paged.AttentionCall(pool.device(), _put(q), _put(np.array(lens, np.int32)), out, counts=_put(np.array(counts, np.int32)),
                               scale=1 / math.sqrt(D))
    call.run()
    device.synchronize()
    with pytest.raises(_lib.ArclightError) as e:
        fattn.device_errors()
    assert e.value.status == abi.AL_ERR_INVALID and "-3 new tokens" in str(e.value)
    fattn.device_errors()                                              # reported once
    got = out.numpy(np.float32)
    assert np.all(got[slot] == MARK)
    keep = [s for s in range(n) if s != slot]
    if keep:
        ref = P.attention(pool, q, lens, [max(c, 0) for c in counts], 1 / math.sqrt(D))
        _check(got[keep], (ref[0][keep], ref[1][keep]), f"slot {slot} of {n}")
