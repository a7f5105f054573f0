"""Errors and values that test_gpu_paged.py does not give the attention: counts
below zero, in every block of 64 slots; logits of -inf; keys and values that are
not finite, for the rows that see them."""
import math

import numpy as np
import pytest

from arclight_amd import abi
from tests import paged_cases as P
from tests.test_gpu_paged import MARK, _attend, _case, _check, _put

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


@pytest.mark.parametrize("T, Hq, Hkv", [(1, 8, 2), (3, 8, 2), (1, 16, 16), (20, 4, 4)])
@pytest.mark.parametrize("n", [1, 33, 300, 5000])
@pytest.mark.parametrize("sinks", [None, 0.5])
def test_logits_that_overflow(gpu, n, T, Hq, Hkv, sinks):
    """Finite queries and keys whose products are below float32's range: those
    cells' weights are 0 wherever they lie, whole tiles and workgroups' parts
    among them; a row that sees nothing else is NaN, or 0 beside a sink.

    All other logits are 0, their probabilities 1 and their sums exact; what is
    left are the additions of values in chains (n 2^-23 of the mean size at the
    most: the matrix cores may cut instead of round), the sink's e^0.5 (2^-21)
    and a quotient and a product (2^-22)."""
    _case(f"paged attention, logits below the range, {n} cells, T={T}, sinks={sinks}")
    rng = np.random.default_rng(n + T)
    n = max(n, T)
    low = np.ones(n, bool)                                          # cells whose logits are -inf
    low[2 * n // 3::3] = False
    lens = [n, n, 7 + T]
    pool = P.Pool(rng, [1], Hkv, 16)
    per = (n + 15) // 16
    pool.n_pages, pool.max_pages = 3 * per + 3, per + 3
    pool.table = np.full((3, pool.max_pages), -7, np.int32)
    order = rng.permutation(pool.n_pages)
    for s in range(3):
        need = (lens[s] + 15) // 16
        pool.table[s, :need], order = order[:need], order[need:]
    pool.k = np.zeros((pool.n_pages, 16, Hkv, D), np.float16)
    pool.v = rng.standard_normal(pool.k.shape).astype(np.float16)
    cells = [low, np.ones(n, bool), np.zeros(lens[2], bool)]        # some, all, none
    for s, x in enumerate(cells):
        for c in np.flatnonzero(x):
            pool.k[pool.table[s, c // 16], c % 16, :, 3] = -6e4
    q = np.zeros((3, T, Hq, D), np.float32)
    q[..., 3] = 1e36
    q[..., 5] = 1.0                                                # (its keys are 0)
    with np.errstate(all="ignore"):
        got = _attend(pool, q, lens, sinks=None if sinks is None else [sinks] * Hq, scale=1.0)
    for s in range(3):
        v = pool.cells(pool.v, s, lens[s])
        for t in range(T):
            sees = lens[s] - T + 1 + t
            own = ~cells[s][:sees]
            for h in range(Hq):
                g = got[s, t, h].astype(np.float64)
                if not own.any():
                    assert np.all(np.isnan(g)) if sinks is None else np.all(g == 0), (s, t, h)
                    continue
                vv = v[:sees, h // (Hq // Hkv)][own]
                total = len(vv) + (0.0 if sinks is None else math.exp(sinks))
                tol = np.abs(vv).sum(0) / total * (len(vv) * 2.0 ** -23 + 2.0 ** -20)
                assert np.all(np.abs(g - vv.sum(0) / total) <= tol), (s, t, h)


@pytest.mark.parametrize("T, Hq, Hkv", [(1, 32, 8), (3, 32, 8), (6, 64, 8), (20, 4, 4)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_odd_values_reach_the_rows_that_see_them(gpu, value, T, Hq, Hkv):
    """Values that are not finite, in a cell that all tokens see, one that some
    see and the last one: not finite in their dims of the rows that see them,
    which are right in all other dims, as the other rows are in all."""
    _case(f"paged attention, values of {value} that rows see, T={T}")
    rng = np.random.default_rng(31)
    lens = [T, 60, 97, 700]
    pool = P.Pool(rng, lens, Hkv, 16)
    odd = {}
    for s, n in enumerate(lens):
        for c, d in ((n - 1, 5), (n - T // 2 - 1, 40), (max(n - T - 9, 0), 77)):
            pool.v[pool.table[s, c // 16], c % 16, :, d::64] = value
            odd.setdefault((s, c), []).append(d)
    finite = pool.v.copy()
    pool.v[~np.isfinite(pool.v)] = 0
    q = (rng.standard_normal((4, T, Hq, D)) * 0.5).astype(np.float32)   # (no weight is lost to 0)
    out, bound = P.attention(pool, q, lens, [T] * 4, 1 / math.sqrt(D))
    pool.v = finite
    got = _attend(pool, q, lens)
    reached = np.zeros(got.shape, bool)
    for (s, c), dims in odd.items():
        for t in range(T):
            if c < lens[s] - T + 1 + t:
                for d in dims:
                    reached[s, t, :, d::64] = True
    assert not np.any(np.isfinite(got[reached]))
    _check(got[~reached], (out[~reached], bound[~reached]), f"value {value}")


@pytest.mark.parametrize("T, Hq, Hkv", [(1, 32, 8), (6, 64, 8)])
def test_nan_keys_reach_the_rows_that_see_them(gpu, T, Hq, Hkv):
    _case(f"paged attention, NaN keys that rows see, T={T}")
    rng = np.random.default_rng(32)
    lens = [60, 700]
    pool = P.Pool(rng, lens, Hkv, 16)
    at = [(s, n - T // 2 - 1) for s, n in enumerate(lens)]
    q = (rng.standard_normal((2, T, Hq, D)) * 2).astype(np.float32)
    out, bound = P.attention(pool, q, lens, [T] * 2, 1 / math.sqrt(D))
    for s, c in at:
        pool.k[pool.table[s, c // 16], c % 16, :, 9] = np.nan
    got = _attend(pool, q, lens)
    for s, c in at:
        sees = [c < lens[s] - T + 1 + t for t in range(T)]
        assert np.all(np.isnan(got[s][sees]))
        other = [not x for x in sees]
        if any(other):
            _check(got[s][other], (out[s][other], bound[s][other]), f"sequence {s}")


def test_prompts_and_single_tokens_in_two_calls(gpu):
    """A step of prompts and single tokens over one pair of padded buffers: a
    call with T = 1 views and one of all T, each with counts of 0 for the
    other's sequences, write each its own rows, and what one call of all gives
    to the same bound."""
    from arclight_amd import device, fattn, paged
    _case("paged attention, prompts and single tokens in two calls")
    rng = np.random.default_rng(33)
    lens, counts, T, Hq, Hkv = [400, 50, 90, 1, 700, 64], [1, 50, 1, 1, 1, 30], 50, 8, 2
    pool = P.Pool(rng, lens, Hkv, 16)
    q = (rng.standard_normal((6, T, Hq, D)) * 2).astype(np.float32)
    ref = P.attention(pool, q, lens, counts, 1 / math.sqrt(D))
    cache, dq, out, dl = pool.device(), _put(q), _put(np.full(q.shape, MARK, np.float32)), _put(np.array(lens, np.int32))
    view = lambda t: device.DeviceTensor(t.buf, abi.AL_TYPE_F32, (6, 1, Hq, D), (T * Hq * D * 4, Hq * D * 4, D * 4, 4))  # noqa: E731
    one = [int(c == 1) for c in counts]
    more = [0 if c == 1 else c for c in counts]
    paged.attention(cache, view(dq), dl, view(out), counts=_put(np.array(one, np.int32)), scale=1 / math.sqrt(D))
    paged.attention(cache, dq, dl, out, counts=_put(np.array(more, np.int32)), scale=1 / math.sqrt(D))
    device.synchronize()
    fattn.device_errors()
    _check(out.numpy(np.float32), ref, "two calls")
    _check(_attend(pool, q, lens, counts), ref, "one call")
