"""The paged KV cache on the GPU: attention and append against the plain forms
in 64 bits (tests/paged_cases.py), at the lengths, pages, masks and strides
where they can go wrong."""
import math

import numpy as np
import pytest

from arclight_amd import abi
from tests import paged_cases as P

pytestmark = pytest.mark.gpu
D = 128
MARK = 1234.5                       # what rows that are left alone hold


def _case(name):
    print(f"\n[case] {name}", flush=True)


def _put(x):
    from arclight_amd import device
    return device.DeviceTensor.from_numpy(np.ascontiguousarray(x))


def _attend(pool, q, lens, counts=None, sinks=None, cap=0.0, scale=1 / math.sqrt(D), cache=None, stream=None, workspace=None):
    from arclight_amd import device, fattn, paged
    out = _put(np.full(q.shape, MARK, np.float32))
    paged.attention(cache or pool.device(), _put(q.astype(np.float32)), _put(np.asarray(lens, np.int32)), out,
                    counts=None if counts is None else _put(np.asarray(counts, np.int32)),
                    sinks=None if sinks is None else _put(np.asarray(sinks, np.float32)), scale=scale, logit_softcap=cap,
                    stream=stream, workspace=workspace)
    device.synchronize()
    fattn.device_errors()
    return out.numpy(np.float32)


def _check(got, ref, what):
    out, bound = ref
    left = np.isnan(out)
    assert np.all(got[left] == MARK), f"{what}: rows of no token were written"
    err = np.abs(got.astype(np.float64) - out)[~left]
    worst = float((err / np.maximum(bound[~left], 1e-30)).max()) if err.size else 0.0
    print(f"{what}: worst error {worst:.3f} of the bound, largest {err.max() if err.size else 0:.2e}", flush=True)
    assert np.all(np.isfinite(got[~left])) and worst <= 1.0, what
    # The bound adds the roundings' largest sizes; they are independent, and
    # their root of squares stays below 1e-5 of the whole (scores of size 20
    # off by 20 sqrt(41) 2^-24 = 8e-6). One f16 rounding of the queries or of
    # the probabilities (2^-11 each) would be 20 times that.
    if err.size:
        assert np.linalg.norm(err) <= 1e-5 * np.linalg.norm(out[~left]) + 1e-30, what


CASES = [
    # lens, counts, T, Hq, Hkv, P, heads_first, sinks, cap
    ([1], None, 1, 32, 8, 16, False, False, 0.0),
    ([31, 32, 33, 0, 1, 7, 8, 9], None, 1, 32, 8, 16, False, False, 0.0),
    ([127, 128, 129, 300], None, 1, 8, 8, 8, True, False, 0.0),
    ([25, 49, 700, 24], None, 1, 32, 8, 24, False, True, 0.0),
    ([500, 100, 2000], None, 1, 64, 8, 48, True, False, 20.0),
    ([257, 64, 90], [1, 0, 1], 1, 5, 1, 256, False, True, 30.0),
    ([40, 3, 70, 1], [4, 3, 2, 4], 4, 32, 8, 16, False, False, 0.0),
    ([129, 40, 260], [6, 1, 0], 6, 64, 8, 32, False, True, 0.0),
    ([45, 200], None, 40, 8, 2, 16, True, False, 0.0),
    ([90], None, 70, 12, 4, 64, False, False, 15.0),
    ([33, 2, 5, 400], [3, 2, 8, 5], 8, 24, 8, 40, False, False, 0.0),
    ([3000], None, 1, 16, 1, 16, False, False, 0.0),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention_against_the_definition(gpu, i):
    lens, counts, T, Hq, Hkv, page, heads_first, sinks, cap = CASES[i]
    _case(f"paged attention {CASES[i]}")
    rng = np.random.default_rng(100 + i)
    pool = P.Pool(rng, lens, Hkv, page, heads_first)
    q = (rng.standard_normal((len(lens), T, Hq, D)) * 2.5).astype(np.float32)
    sk = rng.standard_normal(Hq) * 2 + 2 if sinks else None
    scale = 1 / math.sqrt(D)
    ref = P.attention(pool, q, lens, counts or [T] * len(lens), scale, sk, cap)
    _check(_attend(pool, q, lens, counts, sk, cap), ref, f"case {i}")


def test_attention_of_many_sequences(gpu):
    """More sequences than a wave has lanes, of very different lengths, empty
    slots among them: chunks found across blocks of 64."""
    _case("paged attention, 150 sequences")
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(1, 90, 150)]
    lens[70], lens[149], lens[3] = 3000, 1500, 0
    counts = [int(x) for x in rng.integers(0, 2, 150)]
    counts[70] = counts[149] = counts[3] = 1
    pool = P.Pool(rng, lens, 2, 16)
    q = (rng.standard_normal((150, 1, 8, D)) * 2).astype(np.float32)
    _check(_attend(pool, q, lens, counts), P.attention(pool, q, lens, counts, 1 / math.sqrt(D)), "150 sequences")


def test_attention_of_a_long_sequence(gpu):
    """One axis split over all workgroups and joined; probabilities far below
    the largest, which f16 alone would lose, carry part of the result."""
    _case("paged attention, 50000 cells")
    rng = np.random.default_rng(8)
    n = 50000
    pool = P.Pool(rng, [100], 1, 64)
    pool.n_pages = pool.max_pages = (n + 63) // 64
    pool.table = rng.permutation(pool.n_pages).astype(np.int32)[None]
    pool.k = (rng.standard_normal((pool.n_pages, 64, 1, D)) * 0.05).astype(np.float16)
    pool.v = (rng.standard_normal((pool.n_pages, 64, 1, D)) + 1).astype(np.float16)
    q = rng.standard_normal((1, 1, 4, D)).astype(np.float32)
    c = n // 3                                                      # one cell 14 above the others
    key = q[0, 0, 0] / np.linalg.norm(q[0, 0, 0]) ** 2 * 14 * math.sqrt(D)
    pool.k[pool.table[0, c // 64], c % 64, 0] = key
    _check(_attend(pool, q, [n]), P.attention(pool, q, [n], [1], 1 / math.sqrt(D)), "50000 cells")


@pytest.mark.parametrize("T, Hq, Hkv", [(3, 32, 8), (6, 64, 8), (20, 4, 4)])
def test_cells_a_row_does_not_see_do_not_reach_it(gpu, T, Hq, Hkv):
    """NaN and infinities in later tokens' keys and values (the cells past
    the last hold NaN in every case): each token's row is what it is without
    them, tokens that see them are not compared."""
    _case(f"paged attention, odd values in later tokens' cells, T={T}")
    rng = np.random.default_rng(9)
    lens = [T, 60, 97]
    pool = P.Pool(rng, lens, Hkv, 16)
    for s, n in enumerate(lens):
        for back, value in ((1, np.nan), (2, np.inf)):
            c = n - back
            pool.v[pool.table[s, c // 16], c % 16, :, ::5] = value
            pool.k[pool.table[s, c // 16], c % 16, :, ::7] = -value
    q = (rng.standard_normal((3, T, Hq, D)) * 2).astype(np.float32)
    clean = T - 2                                                   # tokens that see neither
    with np.errstate(all="ignore"):
        out, bound = P.attention(pool, q, lens, [T] * 3, 1 / math.sqrt(D))
    got = _attend(pool, q, lens)
    _check(got[:, :clean], (out[:, :clean], bound[:, :clean]), f"T={T}")


@pytest.mark.parametrize("size", [1e-30, 1e-12, 3e4, 1e30])
def test_query_rows_of_any_size(gpu, size):
    """Rows far outside f16's range, with the scale that brings the scores
    back, beside rows of ordinary size and zero rows."""
    _case(f"paged attention, rows of size {size}")
    rng = np.random.default_rng(10)
    pool = P.Pool(rng, [77], 2, 16)
    q = rng.standard_normal((1, 1, 8, D)) * size
    q[0, 0, 3] = 0
    scale = 0.2 / size
    _check(_attend(pool, q.astype(np.float32), [77], scale=scale),
           P.attention(pool, q.astype(np.float32), [77], [1], float(np.float32(scale))), f"size {size}")


def test_negative_scale(gpu):
    rng = np.random.default_rng(11)
    pool = P.Pool(rng, [300], 4, 32)
    q = rng.standard_normal((1, 2, 8, D)).astype(np.float32)
    _check(_attend(pool, q, [300], scale=-0.125), P.attention(pool, q, [300], [2], -0.125), "scale -1/8")


def test_shared_pages(gpu):
    """Two sequences with the same first pages, and one whose table names one
    page twice."""
    _case("paged attention, shared pages")
    rng = np.random.default_rng(12)
    pool = P.Pool(rng, [64, 80, 48], 2, 16)
    pool.table[1, :3] = pool.table[0, :3]
    pool.table[2, 1] = pool.table[2, 0]
    q = rng.standard_normal((3, 1, 8, D)).astype(np.float32)
    _check(_attend(pool, q, [64, 80, 48]), P.attention(pool, q, [64, 80, 48], [1, 1, 1], 1 / math.sqrt(D)), "shared pages")


def test_strided_operands_and_offsets_past_32_bits(gpu):
    """Queries and outputs as parts of wider rows, table rows of a wider
    table, and pool pages 2.5 GB apart, so that the last ones lie beyond 4 GB."""
    from arclight_amd import device, fattn, paged
    _case("paged attention, strides, pages past 4 GB")
    rng = np.random.default_rng(13)
    lens, Hq, Hkv, page = [40, 61], 8, 2, 32
    pool = P.Pool(rng, lens, Hkv, page, spare=0)
    apart = 5 * 2 ** 29
    pools = []
    for x in (pool.k, pool.v):
        buf = device.DeviceBuffer(apart * (pool.n_pages - 1) + page * Hkv * D * 2)
        for i in range(pool.n_pages):
            buf.upload(np.ascontiguousarray(x[i]).view(np.uint16), apart * i)
        pools.append(device.DeviceTensor(buf, abi.AL_TYPE_F16, x.shape, (apart, Hkv * D * 2, D * 2, 2)))
    wide = np.full((2, 9), -1, np.int32)
    wide[:, :2] = pool.table
    table = _put(wide)
    cache = paged.PagedCache(*pools, device.DeviceTensor(table.buf, abi.AL_TYPE_I32, (2, 2), (36, 4)))
    q = rng.standard_normal((2, 1, Hq + 3, D)).astype(np.float32)
    qd, out = _put(q), _put(np.full((2, 2, Hq, D + 4), MARK, np.float32))
    row = (D + 4) * 4
    paged.attention(cache, device.DeviceTensor(qd.buf, abi.AL_TYPE_F32, (2, 1, Hq, D), ((Hq + 3) * D * 4, 99 * 16, D * 4, 4), D * 4),
                    _put(np.array(lens, np.int32)),
                    device.DeviceTensor(out.buf, abi.AL_TYPE_F32, (2, 1, Hq, D), (2 * Hq * row, Hq * row, row, 4)),
                    scale=0.1)
    device.synchronize()
    fattn.device_errors()
    got = out.numpy(np.float32)
    _check(got[:, :1, :, :D], P.attention(pool, q[:, :, 1:1 + Hq], lens, [1, 1], float(np.float32(0.1))), "strided")
    assert np.all(got[:, 1] == MARK) and np.all(got[..., D:] == MARK)


def test_wrong_pages_and_lengths_are_reported(gpu):
    """A page outside the pool, a length beyond the table, a count beyond T:
    nothing is read there, the sequence's rows are NaN, the others are right."""
    from arclight_amd import _lib, device, fattn, paged
    _case("paged attention, wrong pages, lengths and counts")
    rng = np.random.default_rng(14)
    lens = [50, 300, 20, 33]
    pool = P.Pool(rng, lens, 2, 16)
    q = rng.standard_normal((4, 1, 8, D)).astype(np.float32)
    ref = P.attention(pool, q, lens, [1] * 4, 1 / math.sqrt(D))
    for what, table, ln, counts, s in (
            ("page past the pool", lambda t: t.__setitem__((1, 5), pool.n_pages), lens, [1] * 4, 1),
            ("negative page", lambda t: t.__setitem__((0, 0), -1), lens, [1] * 4, 0),
            ("length", lambda t: None, [50, 300, pool.max_pages * 16 + 1, 33], [1] * 4, 2),
            ("negative length", lambda t: None, [50, 300, 20, -3], [1] * 4, 3),
            ("count", lambda t: None, lens, [1, 1, 2, 1], 2)):
        good = pool.table.copy()
        if what == "length":                                       # every entry a page, so that clamping can read them
            pool.table[2, 2:] = 0
        table(pool.table)
        cache = pool.device()
        pool.table = good
        out = _put(np.full(q.shape, MARK, np.float32))
        paged.attention(cache, _put(q), _put(np.array(ln, np.int32)), out, counts=_put(np.array(counts, np.int32)),
                        scale=1 / math.sqrt(D))
        device.synchronize()
        with pytest.raises(_lib.ArclightError) as e:
            fattn.device_errors()
        assert e.value.status == abi.AL_ERR_INVALID and "paged cache" in str(e.value), what
        fattn.device_errors()                                      # reported once
        got = out.numpy(np.float32)
        assert np.all(np.isnan(got[s])), what
        keep = [i for i in range(4) if i != s]
        _check(got[keep], (ref[0][keep], ref[1][keep]), what)


def test_workspace_of_the_caller(gpu):
    from arclight_amd import _lib, device, paged
    _case("paged attention, caller's workspace")
    rng = np.random.default_rng(15)
    lens = [2000, 900]
    pool = P.Pool(rng, lens, 2, 16)
    q = rng.standard_normal((2, 1, 8, D)).astype(np.float32)
    cache = pool.device()
    c = paged.AttentionCall(cache, _put(q), _put(np.array(lens, np.int32)), _put(np.zeros_like(q)), scale=0.1)
    need = c.workspace_bytes()
    assert need > 0
    ws = device.DeviceBuffer(need)
    ws.upload(np.full(need, 0xff, np.uint8))                       # NaN records
    ref = P.attention(pool, q, lens, [1, 1], float(np.float32(0.1)))
    _check(_attend(pool, q, lens, scale=0.1, cache=cache, workspace=ws), ref, "workspace")
    small = device.DeviceBuffer(need - 16)
    with pytest.raises(_lib.ArclightError) as e:
        _attend(pool, q, lens, scale=0.1, cache=cache, workspace=small)
    assert e.value.status == abi.AL_ERR_WORKSPACE


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with the library's workspace of its stream."""
    from arclight_amd import device, fattn, paged
    _case("paged attention on two streams")
    rng = np.random.default_rng(16)
    sides = []
    for i in range(2):
        st = device.Stream()
        lens = [5000 + 1000 * i]
        pool = P.Pool(rng, [16], 2, 16)
        pool.max_pages = pool.n_pages = (lens[0] + 15) // 16
        pool.table = rng.permutation(pool.n_pages).astype(np.int32)[None]
        pool.k = rng.standard_normal((pool.n_pages, 16, 2, D)).astype(np.float16)
        pool.v = rng.standard_normal((pool.n_pages, 16, 2, D)).astype(np.float16)
        q = rng.standard_normal((1, 1, 8, D)).astype(np.float32)
        out = _put(np.zeros_like(q))
        sides.append((st, pool, lens, q, out, paged.AttentionCall(pool.device(), _put(q), _put(np.array(lens, np.int32)), out, scale=0.1, stream=st)))
    for _ in range(20):
        for s in sides:
            s[5].run()
    device.synchronize()
    fattn.device_errors()
    for st, pool, lens, q, out, _ in sides:
        _check(out.numpy(np.float32), P.attention(pool, q, lens, [1], float(np.float32(0.1))), "stream")
        st.destroy()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def _tokens(rng, lens, counts, pad):
    seq = [s for s, c in enumerate(counts) for _ in range(c)]
    pos = [p for n, c in zip(lens, counts) for p in range(n - c, n)]
    at = list(rng.permutation(len(seq) + pad))                      # rows in no order, padding between them
    sq, ps = np.full(len(at), -1, np.int32), np.full(len(at), -5, np.int32)
    for i, (s, p) in enumerate(zip(seq, pos)):
        sq[at[i]], ps[at[i]] = s, p
    return sq, ps


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("Hq, Hkv, P_, mode, eps, weights, with_q", [
    (32, 8, 16, "neox", 1e-6, True, True), (64, 8, 24, "normal", 1e-5, True, True), (5, 5, 8, "neox", None, False, True),
    (12, 4, 64, "normal", None, False, True), (9, 3, 256, None, 1e-6, False, True), (8, 2, 16, "neox", 1e-6, True, False)])
def test_append_against_the_definition(gpu, Hq, Hkv, P_, mode, eps, weights, with_q, heads_first):
    from arclight_amd import device, fattn, paged
    _case(f"paged append Hq={Hq} Hkv={Hkv} P={P_} {mode} eps={eps} heads_first={heads_first}")
    rng = np.random.default_rng(20)
    lens, counts = [30, 1, 300, 0, 65, 2000], [30, 1, 7, 0, 3, 1]
    pool = P.Pool(rng, lens, Hkv, P_, heads_first)
    seq, pos = _tokens(rng, lens, counts, pad=3)
    T = len(seq)
    q, k, v = (rng.standard_normal((T, H, D)).astype(np.float32) * 3 for H in (Hq, Hkv, Hkv))
    qw, kw = (rng.standard_normal(D).astype(np.float32) if weights else None for _ in range(2))
    rope = None if mode is None else abi.qwen3_rope()
    if mode == "normal":
        rope.mode = abi.AL_ROPE_NORMAL
    cache = pool.device()
    q_out = _put(np.full(q.shape, MARK, np.float32)) if with_q else None
    paged.append(cache, _put(q) if with_q else None, _put(k), _put(v), _put(pos), _put(seq), q_out,
                 q_w=None if qw is None else _put(qw), k_w=None if kw is None else _put(kw), eps=eps or 0.0,
                 norm=eps is not None, rope=rope)
    device.synchronize()
    fattn.device_errors()
    mine = seq >= 0
    real = np.where(mine, pos, 0)
    # the producers' bar: 1e-5 + 1e-6 of the size, which holds sines and
    # cosines off by an ulp or two and float32 sums of squares
    bar = lambda y: 1e-5 + 1e-6 * np.abs(y)  # noqa: E731
    if with_q:
        ref = P.norm_rotate(q, qw, real, eps, mode)
        got = q_out.numpy(np.float32)
        assert np.all(got[~mine] == MARK)
        assert np.all(np.abs(got[mine] - ref[mine]) <= bar(ref[mine]) * 3)   # |x| up to 3 times larger than a unit row's
    kr = P.norm_rotate(k, kw, real, eps, mode)
    got_k, got_v = pool.download(cache)
    want_k, want_v = pool.k.copy(), pool.v.copy()
    tol = np.zeros(want_k.shape)
    for t in np.flatnonzero(mine):
        at = pool.table[seq[t], pos[t] // P_], pos[t] % P_
        want_k[at], want_v[at] = kr[t].astype(np.float16), v[t].astype(np.float16)
        tol[at] = bar(kr[t]) * 3 + np.abs(kr[t]) * 2.0 ** -10           # one float16 step
    new = tol > 0
    assert np.array_equal(got_v.view(np.uint16), want_v.view(np.uint16))
    assert np.array_equal(got_k.view(np.uint16)[~new], want_k.view(np.uint16)[~new]), "other cells were written"
    assert np.all(np.abs(got_k[new].astype(np.float64) - want_k[new]) <= tol[new])


@pytest.mark.parametrize("T", [1, 37])
def test_append_gives_the_rings_bits(gpu, T):
    """Queries and cells are, bit for bit, what al_attn_inputs_f32 gives for
    the same tokens with the pool seen as a ring's rows."""
    from arclight_amd import device, fattn, paged, prologue
    _case(f"paged append against the ring's producers, T={T}")
    rng = np.random.default_rng(21)
    Hq, Hkv, page, lens = 32, 8, 16, [9000]
    pool = P.Pool(rng, [16], Hkv, page)
    pool.max_pages = pool.n_pages = (lens[0] + page - 1) // page
    pool.table = rng.permutation(pool.n_pages).astype(np.int32)[None]
    pool.k = np.zeros((pool.n_pages, page, Hkv, D), np.float16)
    pool.v = pool.k.copy()
    seq, pos = np.zeros(T, np.int32), np.arange(lens[0] - T, lens[0], dtype=np.int32)
    q, k, v = (rng.standard_normal((T, H, D)).astype(np.float32) for H in (Hq, Hkv, Hkv))
    w = [_put(rng.standard_normal(D).astype(np.float32)) for _ in range(2)]
    cache = pool.device()
    dq, dk, dv, dp = _put(q), _put(k), _put(v), _put(pos)
    q_out = paged.append(cache, dq, dk, dv, dp, _put(seq), q_w=w[0], k_w=w[1], eps=1e-6, rope=abi.qwen3_rope())
    rows = (pool.table[0, pos // page].astype(np.int64) * page + pos % page)
    n = pool.n_pages * page
    rk = [_put(np.zeros((n, Hkv * D), np.uint16)) for _ in range(2)]
    rq = _put(np.zeros_like(q))
    prologue.attn_inputs(dq, w[0], dk, w[1], _put(v.reshape(T, -1)), dp, _put(rows), rq, rk[0], rk[1], eps=1e-6, rope=abi.qwen3_rope())
    device.synchronize()
    fattn.device_errors()
    assert np.array_equal(q_out.numpy(np.float32).view(np.uint32), rq.numpy(np.float32).view(np.uint32))
    for mine, ring in zip((cache.k, cache.v), rk):
        assert np.array_equal(mine.numpy(np.uint16).reshape(n, -1), ring.numpy(np.uint16))


def test_append_reports_what_it_cannot_place(gpu):
    from arclight_amd import _lib, device, fattn, paged
    _case("paged append, wrong sequences, positions and pages")
    rng = np.random.default_rng(22)
    pool = P.Pool(rng, [20, 40], 2, 16)
    k = rng.standard_normal((3, 2, D)).astype(np.float32)
    good = (np.array([0, 1, 1], np.int32), np.array([19, 5, 39], np.int32))
    for what, i, s, p in (("sequence", 1, 2, 5), ("position", 2, 1, pool.max_pages * 16), ("negative position", 2, 1, -1),
                          ("page", 0, 0, 35)):                      # sequence 0 has no third page
        seq, pos = good[0].copy(), good[1].copy()
        seq[i], pos[i] = s, p
        cache = pool.device()
        paged.append(cache, None, _put(k), _put(k), _put(pos), _put(seq), norm=False)
        device.synchronize()
        with pytest.raises(_lib.ArclightError) as e:
            fattn.device_errors()
        assert e.value.status == abi.AL_ERR_INVALID, what
        got_k, got_v = pool.download(cache)
        want = pool.k.copy(), pool.v.copy()
        for t in range(3):
            if t != i:
                at = pool.table[seq[t], pos[t] // 16], pos[t] % 16
                want[0][at] = want[1][at] = k[t].astype(np.float16)
        assert np.array_equal(got_k.view(np.uint16), want[0].view(np.uint16)), what
        assert np.array_equal(got_v.view(np.uint16), want[1].view(np.uint16)), what


@pytest.mark.parametrize("replayed", [False, True])
def test_decode_steps_of_a_batch(gpu, replayed):
    """Steps of append and attention as a server makes them: sequences grow,
    one ends and its slot and pages go to another; with the two launches
    captured once and replayed."""
    from arclight_amd import device, fattn, paged
    _case(f"paged decode steps, replayed={replayed}")
    rng = np.random.default_rng(23)
    n, Hq, Hkv, page, max_pages = 6, 16, 4, 16, 20
    pool = P.Pool(rng, [0] * n, Hkv, page, spare=70, max_pages=max_pages)
    free = list(range(70))
    lens = [0, 15, 16, 200, 33, 100]
    pool.k[:], pool.v[:] = np.nan, np.nan
    for s, m in enumerate(lens):
        for i in range((m + page - 1) // page):
            pool.table[s, i] = free.pop()
        for c in range(m):
            at = pool.table[s, c // page], c % page
            pool.k[at], pool.v[at] = rng.standard_normal((2, Hkv, D))
    cache = pool.device()
    stream = device.Stream()
    w = [rng.standard_normal(D).astype(np.float32) for _ in range(2)]
    dw = [_put(x) for x in w]
    buf = {k: device.DeviceTensor.empty(s, t) for k, s, t in (
        ("q", (n, Hq, D), np.float32), ("k", (n, Hkv, D), np.float32), ("v", (n, Hkv, D), np.float32), ("pos", (n,), np.int32),
        ("seq", (n,), np.int32), ("lens", (n,), np.int32), ("counts", (n,), np.int32), ("q_out", (n, Hq, D), np.float32),
        ("out", (n, 1, Hq, D), np.float32))}
    app = paged.AppendCall(cache, buf["q"], buf["k"], buf["v"], buf["pos"], buf["seq"], buf["q_out"], q_w=dw[0], k_w=dw[1],
                           eps=1e-6, rope=abi.qwen3_rope(), stream=stream)
    q_rows = device.DeviceTensor(buf["q_out"].buf, abi.AL_TYPE_F32, (n, 1, Hq, D))
    att = paged.AttentionCall(cache, q_rows, buf["lens"], buf["out"], counts=buf["counts"], scale=1 / math.sqrt(D), stream=stream)

    def step():
        app.run()
        att.run()

    graph = None
    for i in range(6):
        active = [s for s in range(n) if not (s == 2 and i in (2, 3))]   # slot 2 is empty for two steps
        if i == 4:                                                     # and then another sequence's, from its first token on
            lens[2] = 0
            pool.table[2] = -7
        for s in active:
            if lens[s] % page == 0 and pool.table[s, lens[s] // page] < 0:
                pool.table[s, lens[s] // page] = free.pop()
        host = {k: rng.standard_normal(buf[k].shape).astype(np.float32) for k in ("q", "k", "v")}
        host["seq"] = np.array([s if s in active else -1 for s in range(n)], np.int32)
        host["pos"] = np.array(lens, np.int32)
        for s in active:
            lens[s] += 1
        host["lens"] = np.array(lens, np.int32)
        host["counts"] = (host["seq"] >= 0).astype(np.int32)
        host["out"] = np.full(buf["out"].shape, MARK, np.float32)
        for k, x in host.items():
            buf[k].buf.upload(x)
        cache.table.buf.upload(pool.table)
        device.synchronize()
        if replayed and graph is None and i == 1:
            graph = device.Graph(stream, step)
        if graph is not None:
            graph.launch(stream)
        else:
            step()
        device.synchronize()
        fattn.device_errors()
        kr = P.norm_rotate(host["k"], w[1], host["pos"], 1e-6, "neox")
        for s in active:
            at = pool.table[s, (lens[s] - 1) // page], (lens[s] - 1) % page
            pool.k[at], pool.v[at] = kr[s].astype(np.float16), host["v"][s].astype(np.float16)
        got_k, got_v = pool.download(cache)
        seen = ~np.isnan(pool.k)
        assert np.array_equal(seen, ~np.isnan(got_k)) and np.array_equal(got_v.view(np.uint16), pool.v.view(np.uint16))
        assert np.all(np.abs(got_k[seen].astype(np.float64) - pool.k[seen]) <= np.abs(pool.k[seen].astype(np.float64)) * 2.0 ** -10 + 3e-5)
        pool.k = np.where(seen, got_k, pool.k)                         # the attention over the cells as they are
        q = buf["q_out"].numpy(np.float32)
        ref_q = P.norm_rotate(host["q"], w[0], host["pos"], 1e-6, "neox")
        assert np.all(np.abs(q[active] - ref_q[active]) <= 3e-5 + 1e-6 * np.abs(ref_q[active]))
        counts = host["counts"].tolist()
        _check(buf["out"].numpy(np.float32), P.attention(pool, q[:, None], lens, counts, 1 / math.sqrt(D)), f"step {i}")
    if graph is not None:
        graph.destroy()
    stream.destroy()


@pytest.mark.parametrize("n, longest, T, Hq, Hkv", [(2, 40, 1, 8, 8), (70, 500, 1, 32, 8), (64, 512, 1, 4, 4), (65, 513, 1, 4, 4),
                                                    (300, 60, 1, 8, 2), (130, 200, 7, 8, 8), (40, 300, 20, 8, 2), (200, 33, 3, 64, 8)])
def test_sequences_left_whole_or_cut(gpu, n, longest, T, Hq, Hkv):
    """Short sequences, some to a workgroup, over one block of 64 lanes and
    more; the longest at, below and above where they are cut; empty slots at
    both ends and between; counts from none to all."""
    _case(f"paged attention, {n} sequences of up to {longest}")
    rng = np.random.default_rng(17)
    lens = [int(x) for x in rng.integers(0, longest + 1, n)]
    lens[n // 2] = longest
    counts = [int(min(x, c)) for x, c in zip(lens, rng.integers(0, T + 1, n))]
    counts[n // 2] = T
    counts[0] = 0
    if n > 2:
        counts[-1] = counts[n // 3] = 0
    pool = P.Pool(rng, lens, Hkv, 16)
    q = (rng.standard_normal((n, T, Hq, D)) * 2).astype(np.float32)
    ref = P.attention(pool, q, lens, counts, 1 / math.sqrt(D))
    _check(_attend(pool, q, lens, counts), ref, f"{n} sequences")
    if T == 1:                                                         # every one of the batch with a token
        _check(_attend(pool, q, lens), P.attention(pool, q, lens, [1] * n, 1 / math.sqrt(D)), f"{n} sequences, all")
    only = [0] * n                                                     # one alone
    only[n // 2] = T
    _check(_attend(pool, q, lens, only), P.attention(pool, q, lens, only, 1 / math.sqrt(D)), "one of them")


def test_append_past_32_bits(gpu):
    """Pages 2.5 GB apart: the cells of the last ones lie beyond 4 GB."""
    from arclight_amd import device, fattn, paged
    _case("paged append, pages past 4 GB")
    rng = np.random.default_rng(24)
    Hkv, page, n_pages = 2, 8, 3
    apart = 5 * 2 ** 29
    pools = []
    for _ in range(2):
        buf = device.DeviceBuffer(apart * (n_pages - 1) + page * Hkv * D * 2)
        for i in range(n_pages):
            buf.upload(np.full((page, Hkv, D), 0x3c00, np.uint16), apart * i)
        pools.append(device.DeviceTensor(buf, abi.AL_TYPE_F16, (n_pages, page, Hkv, D), (apart, Hkv * D * 2, D * 2, 2)))
    cache = paged.PagedCache(*pools, _put(np.array([[1, 2, 0]], np.int32)))
    pos = np.array([17, 0, 15, 8], np.int32)                        # pages 0, 1, 2, 2
    k, v = (rng.standard_normal((4, Hkv, D)).astype(np.float32) for _ in range(2))
    paged.append(cache, None, _put(k), _put(v), _put(pos), _put(np.zeros(4, np.int32)), norm=False)
    device.synchronize()
    fattn.device_errors()
    for t, x in zip(pools, (k, v)):
        for at in range(n_pages):
            want = np.full((page, Hkv, D), 0x3c00, np.uint16)
            for i, p_ in enumerate(pos):
                if [1, 2, 0][p_ // page] == at:
                    want[p_ % page] = x[i].astype(np.float16).view(np.uint16)
            assert np.array_equal(t.buf.download(np.empty((page, Hkv, D), np.uint16), apart * at), want), at
