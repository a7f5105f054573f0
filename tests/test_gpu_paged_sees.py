"""Attention over the paged cache of tokens that see other cells than all
before them: windows with first cells, trees of drafts, both; against the
definition in 64 bits (tests/tree_cases.py)."""
import math

import numpy as np
import pytest

from arclight_amd import abi
from tests import paged_cases as P
from tests import tree_cases as C
from tests.test_gpu_paged import MARK, _case, _check, _put

pytestmark = pytest.mark.gpu
D = 128
SCALE = 1 / math.sqrt(D)


def _attend(pool, q, lens, counts=None, sinks=None, cap=0.0, cache=None, errors=True, stream=None, workspace=None, bits=None, pos=None, **kw):
    from arclight_amd import device, fattn, paged
    out = _put(np.full(q.shape, MARK, np.float32))
    paged.attention(cache or pool.device(), _put(q.astype(np.float32)), _put(np.asarray(lens, np.int32)), out,
                    counts=None if counts is None else _put(np.asarray(counts, np.int32)),
                    sinks=None if sinks is None else _put(np.asarray(sinks, np.float32)), scale=SCALE, logit_softcap=cap,
                    bits=None if bits is None else _put(bits), pos=None if pos is None else _put(np.asarray(pos, np.int32)),
                    stream=stream, workspace=workspace, **kw)
    device.synchronize()
    if errors:
        fattn.device_errors()
    return out.numpy(np.float32)


def _free(pool, lens, counts, window, first):
    """What a server with a window frees: pages of cells that no token sees."""
    for s, n in enumerate(lens):
        c = counts[s]
        low = max(n - c + 1 - window, 0)
        for i in range(pool.max_pages):
            if i * pool.P >= first and (i + 1) * pool.P <= low:
                pool.table[s, i] = -9


WINDOWS = [
    # lens, counts, T, Hq, Hkv, P, heads_first, sinks, cap, window, first
    ([1], None, 1, 32, 8, 16, False, False, 0.0, 1, 0),
    ([40, 200, 33, 1], None, 1, 32, 8, 8, False, False, 0.0, 1, 0),
    ([700, 31, 32, 33, 64, 65], None, 1, 32, 8, 16, False, False, 0.0, 32, 4),
    ([700, 129, 300, 2], None, 1, 8, 8, 8, True, False, 0.0, 33, 1),
    ([300, 100, 2000, 31], None, 1, 64, 8, 24, True, True, 0.0, 64, 33),
    ([257, 64, 90], [1, 0, 1], 1, 5, 1, 256, False, True, 30.0, 100, 0),
    ([3000, 2500], None, 1, 16, 1, 16, False, False, 0.0, 1000, 70),
    ([2000], None, 1, 32, 8, 16, False, False, 0.0, 1900, 90),      # the window reaches the first cells' tile
    ([100, 7], None, 1, 32, 8, 16, False, False, 0.0, 5000, 3),     # a window longer than the sequence
    ([500], None, 1, 8, 2, 16, False, False, 0.0, 2 ** 31 - 1, 2 ** 31 - 1),
    ([400], None, 1, 8, 2, 16, False, False, 0.0, 20, 2 ** 31 - 1),  # all are first ones
    ([40, 3, 270, 1, 0], [4, 3, 2, 4, 0], 4, 32, 8, 16, False, False, 0.0, 17, 2),   # (more new tokens than cells)
    ([129, 40, 260], [6, 1, 0], 6, 64, 8, 32, False, True, 0.0, 3, 8),
    ([345, 200], None, 40, 8, 2, 16, True, False, 0.0, 50, 4),
    ([190], None, 70, 12, 4, 64, False, False, 15.0, 12, 0),
    ([300], None, 300, 4, 4, 16, False, False, 0.0, 64, 10),
    ([500, 333], [500, 20], 500, 8, 2, 48, False, True, 0.0, 100, 40),
]


@pytest.mark.parametrize("i", range(len(WINDOWS)))
def test_windows(gpu, i):
    lens, counts, T, Hq, Hkv, page, heads_first, sinks, cap, window, first = WINDOWS[i]
    _case(f"window {WINDOWS[i]}")
    rng = np.random.default_rng(200 + i)
    counts = counts or [T] * len(lens)
    pool = P.Pool(rng, lens, Hkv, page, heads_first)
    _free(pool, lens, counts, window, first)
    q = (rng.standard_normal((len(lens), T, Hq, D)) * 2.5).astype(np.float32)
    sk = rng.standard_normal(Hq) * 2 + 2 if sinks else None
    sees = [C.visible(n, c, T, window, first) for n, c in zip(lens, counts)]
    _check(_attend(pool, q, lens, counts, sk, cap, window=window, first=first),
           C.attention(pool, q, lens, counts, SCALE, sees, sk, cap), f"window {i}")


def _trees(rng, lens, counts, T, words=None, bushy=0.6):
    """parents, pos, bits of all sequences."""
    parents = [C.random_tree(rng, T, bushy) for _ in lens]
    made = [C.tree(par, n, min(c, n), words) for par, n, c in zip(parents, lens, counts)]
    return np.stack(parents), np.stack([m[0] for m in made]), np.stack([m[3] for m in made])


TREES = [
    # lens, counts, T, Hq, Hkv, P, heads_first, sinks, cap
    ([1], None, 1, 32, 8, 16, False, False, 0.0),
    ([9, 200, 40], None, 9, 32, 8, 16, False, False, 0.0),
    ([26, 300], None, 26, 32, 8, 16, False, False, 0.0),            # no cells before the tree
    ([500, 100, 70], [33, 1, 0], 33, 64, 8, 24, True, True, 0.0),
    ([64, 1000], [61, 64], 64, 8, 8, 32, False, False, 20.0),
    ([300, 77], [200, 65], 200, 4, 2, 16, False, True, 0.0),
    ([2500], None, 40, 16, 1, 16, False, False, 0.0),
    ([90, 31, 32, 33], [2, 2, 2, 2], 2, 32, 8, 8, True, False, 0.0),
]


@pytest.mark.parametrize("window, first", [(0, 0), (40, 5), (3, 0), (1, 20)])
@pytest.mark.parametrize("i", range(len(TREES)))
def test_trees(gpu, i, window, first):
    lens, counts, T, Hq, Hkv, page, heads_first, sinks, cap = TREES[i]
    _case(f"tree {TREES[i]}, window {window}, {first}")
    rng = np.random.default_rng(300 + i)
    counts = counts or [T] * len(lens)
    pool = P.Pool(rng, lens, Hkv, page, heads_first)
    _, pos, bits = _trees(rng, lens, counts, T)
    if window:
        _free(pool, lens, counts, window, first)
    q = (rng.standard_normal((len(lens), T, Hq, D)) * 2.5).astype(np.float32)
    sk = rng.standard_normal(Hq) * 2 + 2 if sinks else None
    sees = [C.visible(n, c, T, window, first, b, p if window else None) for n, c, b, p in zip(lens, counts, bits, pos)]
    if window == 3:                                                  # by the path, not by the cells' numbers
        assert any((s[:, n - c:] & (np.arange(c)[:, None] - np.arange(c) >= 3)).any() for s, n, c in zip(sees, lens, counts)) or T < 9
    _check(_attend(pool, q, lens, counts, sk, cap, bits=bits, pos=pos if window else None, window=window, first=first),
           C.attention(pool, q, lens, counts, SCALE, sees, sk, cap), f"tree {i}")


@pytest.mark.parametrize("sinks", [False, True])
def test_any_bits(gpu, sinks):
    """Rows that see nothing at all, later tokens, all tokens; bits behind the
    last token and words behind the last are not looked at; wider rows."""
    from arclight_amd import device, paged
    _case("any bits")
    rng = np.random.default_rng(11)
    lens, counts, T, Hq, Hkv = [37, 37, 90], [37, 37, 50], 50, 8, 2
    pool = P.Pool(rng, lens, Hkv, 16)
    bits = rng.integers(0, 2 ** 32, (3, T, 2), dtype=np.uint64).astype(np.uint32)
    bits[0, ::3] = 0
    bits[1, 5:40, 0] = 0
    bits[0, 1] = 0xffffffff
    bits = bits.view(np.int32)
    q = (rng.standard_normal((3, T, Hq, D)) * 2).astype(np.float32)
    sk = rng.standard_normal(Hq) * 2 if sinks else None
    sees = [C.visible(n, c, T, bits=b) for n, c, b in zip(lens, counts, bits)]
    assert any(not row.any() for s in sees for row in s) and any(s[t, n - c + t + 1:].any() for s, n, c in zip(sees, lens, counts) for t in range(30))
    ref = C.attention(pool, q, lens, counts, SCALE, sees, sk)
    _check(_attend(pool, q, lens, counts, sk, bits=bits), ref, "any bits")
    wide = np.full((3, T + 1, 5), -1, np.int32)
    wide[:, :T, :2] = bits
    wd = _put(wide)
    out = _put(np.full(q.shape, MARK, np.float32))
    paged.attention(pool.device(), _put(q), _put(np.array(lens, np.int32)), out, counts=_put(np.array(counts, np.int32)),
                    sinks=None if sk is None else _put(sk.astype(np.float32)), scale=SCALE,
                    bits=device.DeviceTensor(wd.buf, abi.AL_TYPE_I32, (3, T, 4), ((T + 1) * 20, 20, 4)))
    device.synchronize()
    _check(out.numpy(np.float32), ref, "any bits, wider")


@pytest.mark.parametrize("T, Hq, Hkv", [(12, 8, 2), (40, 16, 2)])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, T, Hq, Hkv):
    """NaN and infinities in some nodes' cells and below the windows: rows that
    do not see them are what they are without."""
    _case(f"odd values that some rows see, T={T}")
    rng = np.random.default_rng(12)
    lens, counts = [T, 150, 97], [T, T, T]
    pool = P.Pool(rng, lens, Hkv, 16)
    parents, pos, bits = _trees(rng, lens, counts, T)
    odd = (3, 5, T - 2)
    for s, n in enumerate(lens):
        for u, value in zip(odd, (np.nan, np.inf, -np.inf)):
            at = pool.table[s, (n - T + u) // 16], (n - T + u) % 16
            pool.v[at][:, ::5] = value
            pool.k[at][:, ::7] = value
    q = (rng.standard_normal((3, T, Hq, D)) * 2).astype(np.float32)
    for window in (0, 30):
        sees = [C.visible(n, T, T, window, 0, b, p if window else None) for n, b, p in zip(lens, bits, pos)]
        clean = np.stack([~s[:, [n - T + u for u in odd]].any(1) for s, n in zip(sees, lens)])
        assert clean.sum(1).min() >= 3                               # (of the inputs: there is something to compare)
        with np.errstate(all="ignore"):
            out, bound = C.attention(pool, q, lens, counts, SCALE, sees)
        got = _attend(pool, q, lens, bits=bits, pos=pos if window else None, window=window)
        _check(got[clean], (out[clean], bound[clean]), f"trees, window {window}")
    # a window's lower end, inside a tile: what lies below it is not a number
    n, window = 150, 60
    for c in range(n - T - window, n - T + 2 - window):
        at = pool.table[1, c // 16], c % 16
        pool.v[at], pool.k[at] = np.nan, np.inf
    for u in odd:
        at = pool.table[1, (n - T + u) // 16], (n - T + u) % 16
        pool.v[at], pool.k[at] = 1, 1
    sees = [C.visible(m, T, T, window) for m in lens]
    with np.errstate(all="ignore"):
        out, bound = C.attention(pool, q, lens, counts, SCALE, sees)
    got = _attend(pool, q, lens, window=window)
    _check(got[1, 1:], (out[1, 1:], bound[1, 1:]), "below a window")


def test_no_rule_is_the_plain_call(gpu):
    """first without a window, and a window longer than any position, see what
    the call without a rule sees; the former with its bits."""
    _case("no rule")
    rng = np.random.default_rng(13)
    lens, T = [300, 45], 3
    pool = P.Pool(rng, lens, 2, 16)
    q = rng.standard_normal((2, T, 8, D)).astype(np.float32)
    plain = _attend(pool, q, lens)
    assert np.array_equal(_attend(pool, q, lens, first=9), plain)
    ref = P.attention(pool, q, lens, [T] * 2, SCALE)
    _check(_attend(pool, q, lens, window=10000), ref, "long window")
    chain = np.stack([C.tree(np.arange(-1, T - 1), n, T)[3] for n in lens])
    _check(_attend(pool, q, lens, bits=chain), ref, "a chain's bits")


def test_wrong_positions_pages_and_lengths_are_reported(gpu):
    """The rows concerned are NaN, others are not; the error is recorded once."""
    from arclight_amd import fattn
    from arclight_amd._lib import ArclightError
    _case("wrong positions")
    rng = np.random.default_rng(14)
    lens, T, Hq = [100, 80, 60], 4, 8
    pool = P.Pool(rng, lens, 2, 16)
    _, pos, bits = _trees(rng, lens, [T] * 3, T)
    q = rng.standard_normal((3, T, Hq, D)).astype(np.float32)
    sees = [C.visible(n, T, T, 50, 0, b, p) for n, b, p in zip(lens, bits, pos)]
    ref = C.attention(pool, q, lens, [T] * 3, SCALE, sees)
    for bad in (lens[1], lens[1] - T - 1, -5, 2 ** 31 - 1, -2 ** 31):
        wrong = pos.astype(np.int64)
        wrong[1, 3] = bad                                            # (a leaf: no other row goes by it)
        keep = np.ones((3, T), bool)
        keep[1] = [not sees[1][t, lens[1] - 1] for t in range(T)]
        got = _attend(pool, q, lens, bits=bits, pos=wrong, window=50, errors=False)
        with pytest.raises(ArclightError, match="position"):
            fattn.device_errors()
        assert np.isnan(got[1, 3]).all()
        _check(got[keep], (ref[0][keep], ref[1][keep]), f"position {bad}")
    pool.table[2, 2] = pool.n_pages
    got = _attend(pool, q, lens, bits=bits, pos=pos, window=50, errors=False)
    with pytest.raises(ArclightError, match="page"):
        fattn.device_errors()
    assert np.isnan(got[2]).all()
    _check(got[:2], (ref[0][:2], ref[1][:2]), "page")
    got = _attend(pool, q, [100, 80, 10 ** 6], bits=bits, errors=False)
    with pytest.raises(ArclightError, match="length"):
        fattn.device_errors()
    assert np.isnan(got[2]).all() and np.isfinite(got[:2]).all()


def test_workspace_and_streams(gpu):
    """A caller's workspace of just the bytes asked for, and two streams at once."""
    from arclight_amd import device, fattn, paged
    _case("windows: workspace, streams")
    rng = np.random.default_rng(15)
    lens = [3000, 1200]
    pool = P.Pool(rng, lens, 2, 16)
    cache = pool.device()
    q = [rng.standard_normal((2, 1, 8, D)).astype(np.float32) for _ in range(2)]
    refs = [C.attention(pool, x, lens, [1, 1], SCALE, [C.visible(n, 1, 1, 900, 40) for n in lens]) for x in q]
    streams = [device.Stream() for _ in range(2)]
    outs, calls = [], []
    for x, st in zip(q, streams):
        out = _put(np.full(x.shape, MARK, np.float32))
        c = paged.AttentionCall(cache, _put(x), _put(np.array(lens, np.int32)), out, scale=SCALE, window=900, first=40, stream=st)
        ws = device.DeviceBuffer(c.workspace_bytes())
        c.args.workspace, c.args.workspace_bytes = ws.ptr, ws.nbytes - 1
        with pytest.raises(Exception, match="workspace"):
            c.run()
        c.args.workspace_bytes = ws.nbytes
        outs.append((out, ws))
        calls.append(c)
    device.synchronize()
    for _ in range(3):
        for c in calls:
            c.run()
    device.synchronize()
    fattn.device_errors()
    for (out, _), ref in zip(outs, refs):
        _check(out.numpy(np.float32), ref, "two streams")
    for st in streams:
        st.destroy()


def test_replayed_while_the_window_moves(gpu):
    """A captured call over buffers whose lengths, table and queries change:
    pages that fall behind the window leave the table."""
    from arclight_amd import device, fattn, paged
    _case("windows, replayed")
    rng = np.random.default_rng(16)
    page, window, first, n = 16, 40, 5, 3
    pool = P.Pool(rng, [400] * n, 2, page)
    full = pool.table.copy()
    cache = pool.device()
    st = device.Stream()
    buf = {k: device.DeviceTensor.from_numpy(np.zeros(s, t)) for k, s, t in
           (("q", (n, 1, 8, D), np.float32), ("lens", (n,), np.int32), ("out", (n, 1, 8, D), np.float32))}
    c = paged.AttentionCall(cache, buf["q"], buf["lens"], buf["out"], scale=SCALE, window=window, first=first, stream=st)
    graph = None
    for i, lens in enumerate(([1, 33, 100], [2, 90, 101], [50, 91, 300], [399, 92, 1], [400, 200, 64])):
        pool.table[:] = full
        _free(pool, lens, [1] * n, window, first)
        for s, m in enumerate(lens):
            pool.table[s, (m + page - 1) // page:] = -3
        q = rng.standard_normal((n, 1, 8, D)).astype(np.float32)
        buf["q"].buf.upload(q)
        buf["lens"].buf.upload(np.array(lens, np.int32))
        cache.table.buf.upload(pool.table)
        device.synchronize()
        if i == 1:
            graph = device.Graph(st, c.run)
        graph.launch(st) if graph else c.run()
        device.synchronize()
        fattn.device_errors()
        _check(buf["out"].numpy(np.float32), C.attention(pool, q, lens, [1] * n, SCALE, [C.visible(m, 1, 1, window, first) for m in lens]), f"step {i}")
    graph.destroy()
    st.destroy()


def test_a_long_cache_with_a_window(gpu):
    """Cells past 2^20 of a sequence, few pages of which are there, and pages
    beyond 4 GB of the pool."""
    from arclight_amd import device, fattn, paged
    _case("window of a long sequence")
    rng = np.random.default_rng(17)
    page, Hkv, Hq, n, window, first = 256, 2, 8, 1500001, 700, 300
    apart = 5 * 2 ** 29
    need = [i for i in range((n + page - 1) // page) if i * page < first or (i + 1) * page > n - window]
    table = np.full((1, (n + page - 1) // page), -1, np.int32)
    table[0, need] = np.arange(len(need))
    k, v = (rng.standard_normal((len(need), page, Hkv, D)).astype(np.float16) for _ in range(2))
    pools = []
    for x in (k, v):
        buf = device.DeviceBuffer(apart * (len(need) - 1) + page * Hkv * D * 2)
        for i in range(len(need)):
            buf.upload(np.ascontiguousarray(x[i]).view(np.uint16), apart * i)
        pools.append(device.DeviceTensor(buf, abi.AL_TYPE_F16, x.shape, (apart, Hkv * D * 2, D * 2, 2)))
    q = rng.standard_normal((1, 1, Hq, D)).astype(np.float32)
    out = paged.attention(paged.PagedCache(*pools, _put(table)), _put(q), _put(np.array([n], np.int32)), scale=SCALE, window=window, first=first)
    device.synchronize()
    fattn.device_errors()

    # the same cells, those between left out
    at = np.array(list(range(first)) + list(range(n - window, n)))
    small = P.Pool(rng, [0], Hkv, len(at), spare=1)
    small.table[:] = 0
    small.k, small.v = (x[table[0, at // page], at % page][None] for x in (k, v))
    _check(out.numpy(np.float32), C.attention(small, q, [len(at)], [1], SCALE, [np.ones((1, len(at)), bool)]), "long")
