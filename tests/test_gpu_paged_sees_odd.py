"""Windows and trees over the paged cache: values, sizes, strides and errors that
test_gpu_paged_sees.py does not give them, each for few query rows of a head and
for many, which two kernels take."""
import math

import numpy as np
import pytest

from arclight_amd import abi
from tests import paged_cases as P
from tests import tree_cases as C
from tests.test_gpu_paged import MARK, _case, _check, _put
from tests.test_gpu_paged_sees import SCALE, _attend, _trees

pytestmark = pytest.mark.gpu
D = 128
SIZES = [(1, 8, 2), (20, 4, 4), (45, 8, 2)]                             # tokens, heads: rows of a KV head 4, 20, 180


def _rule(rng, kind, lens, T, window=50, first=6):
    """Keyword arguments of the call, and what each token sees."""
    if kind == "window":
        return {"window": window, "first": first}, [C.visible(n, T, T, window, first) for n in lens]
    _, pos, bits = _trees(rng, lens, [T] * len(lens), T)
    if kind == "tree":
        return {"bits": bits}, [C.visible(n, T, T, bits=b) for n, b in zip(lens, bits)]
    return {"bits": bits, "pos": pos, "window": window, "first": first}, [C.visible(n, T, T, window, first, b, p) for n, b, p in zip(lens, bits, pos)]


@pytest.mark.parametrize("T, Hq, Hkv", SIZES)
@pytest.mark.parametrize("kind", ["window", "tree"])
@pytest.mark.parametrize("n", [60, 400, 3000])
@pytest.mark.parametrize("sinks", [None, 0.5])
def test_logits_that_overflow(gpu, n, T, Hq, Hkv, kind, sinks):
    """Finite queries and keys whose products are below float32's range: those
    cells' weights are 0 wherever they lie; a row that sees nothing else is NaN,
    or 0 beside a sink. All other logits are 0 and their probabilities 1: what is
    left are the additions of values in chains (n 2^-23 of the mean size), the
    sink's e^0.5 (2^-21) and a quotient and a product (2^-22)."""
    _case(f"logits below the range, {kind}, {n} cells, T={T}, sinks={sinks}")
    rng = np.random.default_rng(n + T)
    lens = [n, n, T + 7]
    pool = P.Pool(rng, lens, Hkv, 16)
    rule, sees = _rule(rng, kind, lens, T, window=n // 3)
    low = [np.ones(n, bool), np.ones(n, bool), np.zeros(T + 7, bool)]   # cells whose logits are -inf: some, all, none
    low[0][n // 2::3] = False
    for s, x in enumerate(low):
        for c in range(lens[s]):
            pool.k[pool.table[s, c // 16], c % 16] = 0
            if x[c]:
                pool.k[pool.table[s, c // 16], c % 16, :, 3] = -6e4
    q = np.zeros((3, T, Hq, D), np.float32)
    q[..., 3] = 1e36
    q[..., 5] = 1.0
    from arclight_amd import device, fattn, paged
    out = _put(np.full(q.shape, MARK, np.float32))
    put = {k: _put(x) if isinstance(x, np.ndarray) else x for k, x in rule.items()}
    paged.attention(pool.device(), _put(q), _put(np.array(lens, np.int32)), out, scale=1.0,
                    sinks=None if sinks is None else _put(np.full(Hq, sinks, np.float32)), **put)
    device.synchronize()
    fattn.device_errors()
    got = out.numpy(np.float32).astype(np.float64)
    for s in range(3):
        v = pool.cells(pool.v, s, lens[s])
        for t in range(T):
            own = sees[s][t] & ~low[s]
            for h in range(Hq):
                if not own.any():
                    assert np.all(np.isnan(got[s, t, h])) if sinks is None else np.all(got[s, t, h] == 0), (s, t, h)
                    continue
                vv = v[own, h // (Hq // Hkv)]
                total = len(vv) + (0.0 if sinks is None else math.exp(sinks))
                tol = np.abs(vv).sum(0) / total * (len(vv) * 2.0 ** -23 + 2.0 ** -20)
                assert np.all(np.abs(got[s, t, h] - vv.sum(0) / total) <= tol), (s, t, h)


@pytest.mark.parametrize("T, Hq, Hkv", SIZES)
@pytest.mark.parametrize("kind", ["window", "tree", "both"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_odd_values_reach_the_rows_that_see_them(gpu, value, T, Hq, Hkv, kind):
    """Values that are not finite, in cells that all, some and few tokens see:
    not finite in their dims of the rows that see them, which are right in all
    other dims, as the other rows are in all."""
    _case(f"values of {value} that rows see, {kind}, T={T}")
    rng = np.random.default_rng(31)
    lens = [T, 60, 150, 700]
    pool = P.Pool(rng, lens, Hkv, 16)
    rule, sees = _rule(rng, kind, lens, T)
    odd = {}
    for s, n in enumerate(lens):
        for c, d in ((n - 1, 5), (n - T // 2 - 1, 40), (max(n - T - 9, 0), 77), (max(n - T - 45, 0), 13), (min(2, n - 1), 30)):
            pool.v[pool.table[s, c // 16], c % 16, :, d::64] = value
            odd.setdefault((s, c), []).append(d)
    finite = pool.v.copy()
    pool.v[~np.isfinite(pool.v)] = 0
    q = (rng.standard_normal((4, T, Hq, D)) * 0.5).astype(np.float32)   # (no weight is lost to 0)
    out, bound = C.attention(pool, q, lens, [T] * 4, SCALE, sees)
    pool.v = finite
    got = _attend(pool, q, lens, **rule)
    reached = np.zeros(got.shape, bool)
    for (s, c), dims in odd.items():
        for t in range(T):
            if sees[s][t, c]:
                for d in dims:
                    reached[s, t, :, d::64] = True
    assert reached.any() and not np.any(np.isfinite(got[reached]))
    _check(got[~reached], (out[~reached], bound[~reached]), f"value {value}")


@pytest.mark.parametrize("T, Hq, Hkv", SIZES)
@pytest.mark.parametrize("size, scale", [(1e-30, 0.2e30), (3e4, 0.2 / 3e4), (1e30, 0.2e-30), (1, -0.125), (1, 0.0), (1e-12, 1e-12)])
def test_scales_and_rows_of_any_size(gpu, size, scale, T, Hq, Hkv):
    """Rows far outside float16's range with the scale that brings the scores
    back, beside zero rows; negative scales, none, scores of almost 0."""
    _case(f"rows of size {size}, scale {scale}, T={T}")
    from arclight_amd import device, fattn, paged
    rng = np.random.default_rng(10)
    lens = [T + 30, 177]
    pool = P.Pool(rng, lens, Hkv, 16)
    q = (rng.standard_normal((2, T, Hq, D)) * size).astype(np.float32)
    q[0, 0, 3] = 0
    out = _put(np.full(q.shape, MARK, np.float32))
    paged.attention(pool.device(), _put(q), _put(np.array(lens, np.int32)), out, scale=scale, window=64, first=3)
    device.synchronize()
    fattn.device_errors()
    _check(out.numpy(np.float32), C.attention(pool, q, lens, [T] * 2, float(np.float32(scale)), [C.visible(n, T, T, 64, 3) for n in lens]), "sizes")


@pytest.mark.parametrize("T, Hq, Hkv", SIZES)
def test_a_scale_that_is_no_number(gpu, T, Hq, Hkv):
    from arclight_amd import device, paged
    _case(f"scale NaN, T={T}")
    rng = np.random.default_rng(9)
    pool = P.Pool(rng, [T + 90], Hkv, 16)
    q = _put(rng.standard_normal((1, T, Hq, D)).astype(np.float32))
    out = paged.attention(pool.device(), q, _put(np.array([T + 90], np.int32)), scale=float("nan"), window=64)
    device.synchronize()
    assert np.isnan(out.numpy(np.float32)).all()


@pytest.mark.parametrize("apart", [5 * 2 ** 29, 5 * 2 ** 30])
@pytest.mark.parametrize("T, Hq, Hkv", SIZES)
def test_strided_operands_and_offsets_past_32_bits(gpu, T, Hq, Hkv, apart):
    """Queries and outputs as parts of wider rows, table rows of a wider table,
    pool pages 2.5 and 5 GB apart."""
    from arclight_amd import device, fattn, paged
    _case(f"strides, pages {apart >> 20} MB apart, T={T}")
    rng = np.random.default_rng(13)
    lens, page = [T + 20, T + 3], 64
    pool = P.Pool(rng, lens, Hkv, page, spare=0)
    pools = []
    for x in (pool.k, pool.v):
        buf = device.DeviceBuffer(apart * (pool.n_pages - 1) + page * Hkv * D * 2)
        for i in range(pool.n_pages):
            buf.upload(np.ascontiguousarray(x[i]).view(np.uint16), apart * i)
        pools.append(device.DeviceTensor(buf, abi.AL_TYPE_F16, x.shape, (apart, Hkv * D * 2, D * 2, 2)))
    wide = np.full((2, 9), -1, np.int32)
    wide[:, :pool.max_pages] = pool.table
    table = _put(wide)
    cache = paged.PagedCache(*pools, device.DeviceTensor(table.buf, abi.AL_TYPE_I32, (2, pool.max_pages), (36, 4)))
    q = rng.standard_normal((2, T, Hq + 3, D)).astype(np.float32)
    qd, out = _put(q), _put(np.full((2, T, Hq + 1, D + 4), MARK, np.float32))
    row = (D + 4) * 4
    _, pos, bits = _trees(rng, lens, [T] * 2, T)
    paged.attention(cache, device.DeviceTensor(qd.buf, abi.AL_TYPE_F32, (2, T, Hq, D), (T * (Hq + 3) * D * 4, (Hq + 3) * D * 4, D * 4, 4), D * 4),
                    _put(np.array(lens, np.int32)),
                    device.DeviceTensor(out.buf, abi.AL_TYPE_F32, (2, T, Hq, D), (T * (Hq + 1) * row, (Hq + 1) * row, row, 4)),
                    scale=SCALE, bits=_put(bits))
    device.synchronize()
    fattn.device_errors()
    got = out.numpy(np.float32)
    assert np.all(got[:, :, Hq] == MARK) and np.all(got[..., D:] == MARK)
    sees = [C.visible(n, T, T, bits=b) for n, b in zip(lens, bits)]
    _check(got[:, :, :Hq, :D], C.attention(pool, np.ascontiguousarray(q[:, :, 1:1 + Hq]), lens, [T] * 2, SCALE, sees), "strided")


@pytest.mark.parametrize("T, Hq, Hkv", SIZES)
@pytest.mark.parametrize("n, slot", [(4, 2), (70, 66)])
def test_negative_counts_are_reported(gpu, n, slot, T, Hq, Hkv):
    from arclight_amd import _lib, fattn
    _case(f"a negative count in slot {slot} of {n}, T={T}")
    rng = np.random.default_rng(30 + n)
    lens = [int(x) for x in rng.integers(T, T + 80, n)]
    counts = [T] * n
    counts[slot] = -3
    pool = P.Pool(rng, lens, Hkv, 16)
    q = rng.standard_normal((n, T, Hq, D)).astype(np.float32)
    got = _attend(pool, q, lens, counts, errors=False, window=40)
    with pytest.raises(_lib.ArclightError, match="-3 new tokens"):
        fattn.device_errors()
    fattn.device_errors()                                               # reported once
    counts[slot] = 0
    _check(got, C.attention(pool, q, lens, counts, SCALE, [C.visible(m, c, T, 40) for m, c in zip(lens, counts)]), "counts")


def test_prompts_in_windows_replayed(gpu):
    """A captured call of many query rows, whose lengths, counts and tables
    change: chunks of prompts of different lengths, an empty slot."""
    from arclight_amd import device, fattn, paged
    _case("prompts in windows, replayed")
    rng = np.random.default_rng(16)
    page, window, first, n, T, Hq, Hkv = 16, 70, 5, 3, 60, 8, 2
    pool = P.Pool(rng, [400] * n, Hkv, page)
    full = pool.table.copy()
    cache = pool.device()
    st = device.Stream()
    buf = {k: device.DeviceTensor.from_numpy(np.zeros(s, t)) for k, s, t in
           (("q", (n, T, Hq, D), np.float32), ("lens", (n,), np.int32), ("counts", (n,), np.int32), ("out", (n, T, Hq, D), np.float32))}
    c = paged.AttentionCall(cache, buf["q"], buf["lens"], buf["out"], counts=buf["counts"], scale=SCALE, window=window, first=first, stream=st)
    graph = None
    for i, (lens, counts) in enumerate((([60, 60, 60], [60, 60, 60]), ([61, 100, 399], [1, 40, 60]), ([120, 150, 0], [59, 50, 0]),
                                        ([400, 17, 300], [60, 17, 3]), ([3, 400, 64], [3, 60, 60]))):
        pool.table[:] = full
        for s, m in enumerate(lens):
            pool.table[s, (m + page - 1) // page:] = -3
        q = rng.standard_normal((n, T, Hq, D)).astype(np.float32)
        buf["q"].buf.upload(q)
        buf["out"].buf.upload(np.full((n, T, Hq, D), MARK, np.float32))
        buf["lens"].buf.upload(np.array(lens, np.int32))
        buf["counts"].buf.upload(np.array(counts, np.int32))
        cache.table.buf.upload(pool.table)
        device.synchronize()
        if i == 1:
            graph = device.Graph(st, c.run)
        graph.launch(st) if graph else c.run()
        device.synchronize()
        fattn.device_errors()
        _check(buf["out"].numpy(np.float32), C.attention(pool, q, lens, counts, SCALE, [C.visible(m, k, T, window, first) for m, k in zip(lens, counts)]),
               f"step {i}")
    graph.destroy()
    st.destroy()


@pytest.mark.parametrize("n, T, Hq, Hkv, window", [(70, 40, 8, 8, 30), (3, 700, 16, 2, 100), (40, 70, 4, 2, 20), (2, 2000, 8, 8, 65), (9, 129, 32, 8, 1000)])
def test_many_sequences_of_many_rows(gpu, n, T, Hq, Hkv, window):
    """Parts that end inside sequences, sequences left whole, more row groups
    than the card holds workgroups; against the same tokens one after another
    through the kernel of few rows, whose results are compared with the
    definition elsewhere: both are within 1e-5 of it by norm."""
    from arclight_amd import device, fattn, paged
    _case(f"{n} sequences of up to {T} tokens, window {window}")
    rng = np.random.default_rng(n + T)
    counts = [int(x) for x in rng.integers(T // 3, T + 1, n)]
    counts[0] = T
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 300, n))]
    pool = P.Pool(rng, [1] * n, Hkv, 32, max_pages=(max(lens) + 31) // 32)
    need = [(m + 31) // 32 for m in lens]
    pool.n_pages = sum(need)
    order, at = rng.permutation(pool.n_pages), 0
    for s, k in enumerate(need):
        pool.table[s, :k] = order[at:at + k]
        at += k
    pool.k, pool.v = (rng.standard_normal((pool.n_pages, 32, Hkv, D)).astype(np.float16) for _ in range(2))
    cache = pool.device()
    q = rng.standard_normal((n, T, Hq, D)).astype(np.float32) * 2
    qd, dl = _put(q), np.array(lens, np.int32)
    out, one = (_put(np.full(q.shape, MARK, np.float32)) for _ in range(2))
    paged.attention(cache, qd, _put(dl), out, counts=_put(np.array(counts, np.int32)), scale=SCALE, window=window, first=3)
    step = 4
    for t0 in range(0, T, step):                                        # tokens t0 to t0 + 3 of each sequence
        c = [max(0, min(step, k - t0)) for k in counts]
        ends = np.array([m - k + t0 + x for m, k, x in zip(lens, counts, c)], np.int32)
        k = min(step, T - t0)
        view = lambda x: device.DeviceTensor(x.buf, abi.AL_TYPE_F32, (n, k, Hq, D), (T * Hq * D * 4, Hq * D * 4, D * 4, 4), t0 * Hq * D * 4)  # noqa: E731
        paged.attention(cache, view(qd), _put(ends), view(one), counts=_put(np.array(c, np.int32)), scale=SCALE, window=window, first=3)
    device.synchronize()
    fattn.device_errors()
    a, b = out.numpy(np.float32).astype(np.float64), one.numpy(np.float32).astype(np.float64)
    for s in range(n):
        assert np.all(a[s, counts[s]:] == MARK) and np.linalg.norm(a[s, :counts[s]] - b[s, :counts[s]]) <= 2e-5 * np.linalg.norm(b[s, :counts[s]]), s


SHARES = [                                                              # tokens, heads, new tokens of each sequence, cells before them at most
    (100, 16, 4, [100, 1, 7, 33], 2500),
    (100, 16, 4, [9, 0, 32, 20], 2500),                                 # the last row groups have no rows
    (300, 4, 1, [5], 4000),
    (300, 4, 1, [300], 4000),
    (70, 8, 4, [70, 0, 0, 0, 0, 0, 0, 64], 1500),
    (40, 8, 1, [0] * 30 + [40] + [1] * 60 + [17] * 20, 300),            # two blocks of sequences, three row groups
    (130, 8, 8, [0, 0, 0], 900),
]


@pytest.mark.parametrize("i", range(len(SHARES)))
@pytest.mark.parametrize("window, first", [(0, 0), (700, 3)])
def test_row_groups_of_sequences_that_differ(gpu, i, window, first):
    """Sequences of few rows beside those of many: the row groups' shares of the
    card, and pieces of several groups' sequences, in a call and replayed with
    the counts the other way round."""
    from arclight_amd import device, fattn, paged
    T, Hq, Hkv, counts, before = SHARES[i]
    _case(f"counts {counts} of {T}, window {window}")
    rng = np.random.default_rng(i)
    n = len(counts)
    begin = [int(x) for x in rng.integers(before // 2, before, n)]
    pool = P.Pool(rng, [b + max(c, e) for b, c, e in zip(begin, counts, counts[::-1])], Hkv, 16)
    q = rng.standard_normal((n, T, Hq, D)).astype(np.float32) * 2
    bits = np.zeros((T, (T + 31) // 32), np.uint32)
    for t, u in zip(*np.nonzero(np.tril(rng.random((T, T)) < 0.7) | np.eye(T, dtype=bool))):
        bits[t, u // 32] |= np.uint32(1 << (u % 32))
    bits = bits.view(np.int32)
    buf = {"lens": _put(np.zeros(n, np.int32)), "counts": _put(np.zeros(n, np.int32)), "pos": _put(np.zeros((n, T), np.int32)),
           "out": _put(np.zeros(q.shape, np.float32))}
    st = device.Stream()
    call = paged.AttentionCall(pool.device(), _put(q), buf["lens"], buf["out"], counts=buf["counts"], scale=SCALE, stream=st, window=window,
                               first=first, bits=_put(np.ascontiguousarray(np.broadcast_to(bits, (n, *bits.shape)))), pos=buf["pos"] if window else None)
    graph = None
    for step in range(3):
        c = counts[::-1] if step == 1 else counts
        lens = [x + k for x, k in zip(begin, c)]
        pos = np.array(begin, np.int32)[:, None] + np.arange(T, dtype=np.int32)          # as in a chain
        for name, x in (("lens", lens), ("counts", c), ("pos", pos)):
            buf[name].buf.upload(np.array(x, np.int32))
        buf["out"].buf.upload(np.full(q.shape, MARK, np.float32))
        device.synchronize()
        if step == 1:
            graph = device.Graph(st, call.run)
        graph.launch(st) if graph else call.run()
        device.synchronize()
        fattn.device_errors()
        sees = [C.visible(m, k, T, window, first, bits, x if window else None) for m, k, x in zip(lens, c, pos)]
        _check(buf["out"].numpy(np.float32), C.attention(pool, q, lens, c, SCALE, sees), f"step {step}")
    graph.destroy()
    st.destroy()


LONGER = [(2, [], 300), (5, [0], 400), (8, [3, 7], 130), (11, [], 1000), (70, [0, 5, *range(12, 64), 65], 200)]


@pytest.mark.parametrize("n, gone, window, T, Hq, Hkv", [(*x, *y) for x in LONGER for y in ((1, 16, 8), (5, 16, 2))] + [(*x, 150, 96, 4) for x in LONGER[:3]])
def test_windows_that_all_sequences_are_longer_than(gpu, n, gone, window, T, Hq, Hkv):
    """Sequences that see as many cells as one another, with empty slots between
    them: each has workgroups of its own."""
    _case(f"{n} sequences beyond windows of {window}, T={T}")
    rng = np.random.default_rng(n + T)
    lens = [window + T + int(x) for x in rng.integers(0, 90, n)]
    counts = [T] * n
    for s in gone:
        lens[s], counts[s] = (0 if s % 2 else 40), 0
    pool = P.Pool(rng, lens, Hkv, 16)
    q = (rng.standard_normal((n, T, Hq, D)) * 2).astype(np.float32)
    got = _attend(pool, q, lens, counts, window=window, first=2)
    _check(got, C.attention(pool, q, lens, counts, SCALE, [C.visible(m, c, T, window, 2) for m, c in zip(lens, counts)]), "windows")


@pytest.mark.parametrize("what", ["few rows", "many rows", "verification"])
def test_a_workspaces_counters_are_left_alone(gpu, what):
    from arclight_amd import device, draft, fattn, paged
    _case(f"workspace's first 256 KiB, {what}")
    rng = np.random.default_rng(40)
    if what == "verification":
        n, T, V = 3, 6, 5000
        put = lambda x, t: _put(np.asarray(x, t))  # noqa: E731
        target, tokens = put(rng.random((n, T, V)) / V, np.float32), put(rng.integers(0, V, (n, T)), np.int32)
        parents, path = put(np.tile([-1, 0, 0, 1, 1, 2], (n, 1)), np.int32), put(np.zeros((n, T)), np.int32)
        kept, nxt = put(np.zeros(n), np.int32), put(np.zeros(n), np.int32)
        make = lambda ws: draft.VerifyCall(target, tokens, put(rng.random((n, T)), np.float32), put(rng.random(n), np.float32), path, kept, nxt,  # noqa: E731
                                           parents=parents, draft=target, workspace=ws)
    else:
        T = 1 if what == "few rows" else 60
        pool = P.Pool(rng, [3000, 900], 2, 16)
        cache, q = pool.device(), _put(rng.standard_normal((2, T, 8, D)).astype(np.float32))
        out, dl = device.DeviceTensor.empty((2, T, 8, D), np.float32), _put(np.array([3000, 900], np.int32))
        make = lambda ws: paged.AttentionCall(cache, q, dl, out, scale=SCALE, window=2500, workspace=ws)  # noqa: E731
    need, counters = make(None).workspace_bytes(), 256 << 10
    assert need > counters
    ws = device.DeviceBuffer(need + 4096)
    ws.upload(np.full(need + 4096, 0xa5, np.uint8))
    c = make(ws)
    c.args.workspace_bytes = need
    c.run()
    device.synchronize()
    fattn.device_errors()
    got = ws.download(np.empty(need + 4096, np.uint8))
    assert np.all(got[:counters] == 0xa5) and np.all(got[need:] == 0xa5) and not np.all(got[counters:need] == 0xa5)
