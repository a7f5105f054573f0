"""Low-rank adapters of many requests on the GPU against the definition in 64
bits: alone and beside the Q4_0 projection, for one row to many, any order of
adapters, ranks below the slot's, odd sizes and strides."""
from types import SimpleNamespace

import numpy as np
import pytest

from arclight_amd import abi
from oracle import oracle as O
from tests.test_oracle_q4 import abs_bound, dequant_q4_0, dequant_q8_0

pytestmark = pytest.mark.gpu
EPS32 = 2.0 ** -24


def _case(name):
    print(f"\n[case] {name}", flush=True)


def _put(x):
    from arclight_amd import device
    return device.DeviceTensor.from_numpy(np.ascontiguousarray(x))


def _adapters(rng, n, R, K, N, ranks):
    """Slots whose parts beyond the rank hold NaN."""
    a = (rng.standard_normal((n, R, K)) / np.sqrt(K)).astype(np.float16)
    b = (rng.standard_normal((n, N, R)) / np.sqrt(R)).astype(np.float16)
    for i, r in enumerate(ranks):
        a[i, r:], b[i, :, r:] = np.nan, np.nan
    return a, b


def _ref(x, a, b, scales, ranks, ids, base):
    """(y, bound): float64, and what float32 may be off: v is a sum of K
    products whose chains hold at most K / 4 + 32 additions, rounded by its
    scale; y one of at most 128 products added to base, v's error through it."""
    y = base.astype(np.float64).copy()
    bound = np.abs(y) * EPS32
    x = x.astype(np.float64)
    for t, i in enumerate(ids):
        if i < 0:
            continue
        r = ranks[i]
        aa, bb = a[i, :r].astype(np.float64), b[i, :, :r].astype(np.float64)
        s = float(scales[i])
        v = aa @ x[t] * s
        dv = (np.abs(aa) @ np.abs(x[t])) * abs(s) * (x.shape[1] / 4 + 40) * EPS32
        y[t] += bb @ v
        bound[t] += np.abs(bb) @ dv + (np.abs(bb) @ np.abs(v) + np.abs(base[t])) * 40 * EPS32
    return y, bound


def _check(got, ref, what):
    y, bound = ref
    err = np.abs(got.astype(np.float64) - y)
    worst = float((err / np.maximum(bound, 1e-30)).max())
    print(f"{what}: worst error {worst:.4f} of the bound, relative {np.linalg.norm(err) / np.linalg.norm(y):.1e}", flush=True)
    assert np.all(np.isfinite(got)) and worst <= 1.0, what
    # independent roundings: their root of squares is far below the bound's sum
    assert np.linalg.norm(err) <= 2e-6 * np.linalg.norm(y), what


def _ids(rng, T, n, how):
    if how == "runs":
        return np.sort(rng.integers(-1, n, T)).astype(np.int32)
    if how == "one":
        return np.full(T, n - 1, np.int32)
    return rng.integers(-1, n, T).astype(np.int32)


CASES = [
    # K, N, R, adapters, T, ids, ranks below R
    (4096, 2560, 16, 3, 1, "one", False),
    (2560, 4096, 8, 5, 7, "any", True),
    (4096, 4096, 64, 20, 33, "any", True),
    (2568, 130, 24, 4, 17, "any", False),
    (8, 1, 8, 1, 5, "any", False),
    (136, 333, 128, 7, 100, "any", True),
    (5120, 1023, 40, 9, 64, "runs", True),
    (2560, 1024, 32, 30, 250, "any", True),
    (4096, 260, 16, 3, 1111, "runs", False),
    (512, 512, 96, 2, 5000, "runs", True),
    (512, 256, 16, 40, 4500, "any", True),
]


@pytest.mark.parametrize("i", range(len(CASES)))
@pytest.mark.parametrize("in_place", [False, True])
def test_apply_against_the_definition(gpu, i, in_place):
    from arclight_amd import device, fattn, lora
    K, N, R, n, T, how, mixed = CASES[i]
    _case(f"lora {CASES[i]} in_place={in_place}")
    rng = np.random.default_rng(200 + i)
    ranks = rng.integers(0, R + 1, n) if mixed else np.full(n, R)
    a, b = _adapters(rng, n, R, K, N, ranks)
    scales = (rng.random(n) * 2).astype(np.float32)
    ids = _ids(rng, T, n, how)
    x = (rng.standard_normal((T, K)) * 10.0 ** rng.integers(-3, 4, (T, 1))).astype(np.float32)
    base = rng.standard_normal((T, N)).astype(np.float32)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)), _put(scales), _put(ranks.astype(np.int32)))
    d = _put(base)
    y = lora.apply(ad, _put(x), _put(ids), d if not in_place else None, d if in_place else None)
    device.synchronize()
    fattn.device_errors()
    _check(y.numpy(np.float32), _ref(x, a, b, scales, ranks, ids, base), f"case {i}")


def test_defaults_strides_and_sizes_beyond_f16(gpu):
    """No ranks and no scales; rows of x, base and y as parts of wider rows
    that are left alone; activations of 1e20 beside 1e-20."""
    from arclight_amd import device, fattn, lora
    _case("lora: strides, sizes")
    rng = np.random.default_rng(230)
    K, N, R, n, T = 640, 96, 16, 3, 21
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    ids = _ids(rng, T, n, "any")
    wide = rng.standard_normal((T, K + 8)).astype(np.float32)
    wide *= 10.0 ** np.where(np.arange(T) % 2, 20, -20)[:, None].astype(np.float32)
    base, out = np.zeros((T, N + 3), np.float32), np.full((T, N + 5), 77.0, np.float32)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    xd, bd, yd = _put(wide), _put(base), _put(out)
    view = lambda t, cols, w, off: device.DeviceTensor(t.buf, abi.AL_TYPE_F32, (T, cols), (w * 4, 4), off)  # noqa: E731
    lora.apply(ad, view(xd, K, K + 8, 16), _put(ids), view(bd, N, N + 3, 4), view(yd, N, N + 5, 8))
    device.synchronize()
    fattn.device_errors()
    got = yd.numpy(np.float32)
    assert np.all(got[:, :2] == 77.0) and np.all(got[:, 2 + N:] == 77.0)
    y, bound = _ref(wide[:, 4:4 + K], a, b, np.ones(n), [R] * n, ids, np.zeros((T, N)))
    for k in (0, 1):                                                   # the small and the large rows
        _check(got[k::2, 2:2 + N], (y[k::2], bound[k::2]), f"rows {k}")


def test_odd_values_stay_in_their_row(gpu):
    """A row of NaN and infinities does not reach the rows of its tile, with
    the same adapter or another."""
    from arclight_amd import device, lora
    rng = np.random.default_rng(231)
    K, N, R, n, T = 256, 64, 8, 2, 40
    a, b = _adapters(rng, n, R, K, N, [R, 5])
    ids = _ids(rng, T, n, "any")
    x, base = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    x[3], x[20, 7], base[30, 5] = np.nan, np.inf, np.inf
    ids[[3, 20]] = [0, 1]
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)), None, _put(np.array([R, 5], np.int32)))
    y = lora.apply(ad, _put(x), _put(ids), _put(base))
    device.synchronize()
    got = y.numpy(np.float32)
    keep = np.setdiff1d(np.arange(T), [3, 20, 30])
    ref = _ref(x[keep], a, b, np.ones(n), [R, 5], ids[keep], base[keep])
    _check(got[keep], ref, "other rows")
    assert np.all(np.isnan(got[3])) and not np.any(np.isfinite(got[20])) and np.isinf(got[30, 5])


@pytest.mark.parametrize("T", [1, 5, 20, 70])
def test_unknown_adapters_are_reported(gpu, T):
    from arclight_amd import _lib, device, fattn, lora
    _case(f"lora: unknown adapters, T={T}")
    rng = np.random.default_rng(232)
    K, N, R, n = 4096, 96, 16, 3
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    x, base = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    for what, bad, ranks in (("id", n, [R] * n), ("rank", 1, [R, R + 1, R]), ("negative rank", 1, [R, -1, R])):
        ids = _ids(rng, T, n, "any")
        ids[ids == 1] = 0
        ids[T // 2] = bad
        ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)), None, _put(np.array(ranks, np.int32)))
        y = lora.apply(ad, _put(x), _put(ids), _put(base))
        device.synchronize()
        with pytest.raises(_lib.ArclightError) as e:
            fattn.device_errors()
        assert e.value.status == abi.AL_ERR_INVALID and "lora" in str(e.value), what
        got = y.numpy(np.float32)
        assert np.all(np.isnan(got[T // 2])), what
        keep = np.arange(T) != T // 2
        if keep.any():
            _check(got[keep], _ref(x[keep], a, b, np.ones(n), [R] * n, ids[keep], base[keep]), what)


PROJ = [(4096, 2560, 16, 8, 1), (4096, 4096, 32, 4, 3), (4096, 2560, 8, 12, 8), (8192, 5120, 64, 20, 9), (4096, 100, 24, 6, 16),
        (8192, 1000, 16, 50, 48), (12288, 257, 128, 3, 64), (16384, 64, 8, 2, 2), (16384, 48, 128, 3, 8), (4096, 300, 128, 5, 1), (8192, 31, 72, 9, 6),
        (4096, 40, 40, 2, 60)]


@pytest.mark.parametrize("i", range(len(PROJ)))
def test_project_against_the_definition(gpu, i):
    """The projection's own bar (against the oracle's) and the adapters'."""
    from arclight_amd import device, fattn, lora, matmul
    K, N, R, n, T = PROJ[i]
    _case(f"project {PROJ[i]}")
    rng = np.random.default_rng(240 + i)
    ranks = rng.integers(0, R + 1, n)
    a, b = _adapters(rng, n, R, K, N, ranks)
    scales = (rng.random(n) * 2).astype(np.float32)
    ids = _ids(rng, T, n, "any")
    ids[0] = n - 1
    x = rng.standard_normal((T, K)).astype(np.float32)
    wo = O.random_q4_0(rng, N, K)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)), _put(scales), _put(ranks.astype(np.int32)))
    y = lora.project(ad, matmul.Q4_0Matrix(wo.view(np.uint8), K, N), _put(x), _put(ids))
    device.synchronize()
    fattn.device_errors()
    got = y.numpy(np.float32)
    base = O.mul_mat_q4_0(wo, x)
    ref, bound = _ref(x, a, b, scales, ranks, ids, base)
    bound += (K // 32 + 16) * 2 * EPS32 * abs_bound(dequant_q4_0(wo), dequant_q8_0(O.quantize_q8_0(x)))
    err = np.abs(got.astype(np.float64) - ref)
    print(f"worst {float((err / bound).max()):.4f} of the bound", flush=True)
    assert np.all(err <= bound)
    assert np.linalg.norm(err) <= 2e-6 * np.linalg.norm(ref)


@pytest.mark.parametrize("T", [1, 8, 40])
def test_rows_without_adapters_are_the_projection(gpu, T):
    """Bit for bit, where no row has an adapter."""
    from arclight_amd import device, lora, matmul
    rng = np.random.default_rng(250)
    K, N = 4096, 2560
    a, b = _adapters(rng, 2, 8, K, N, [8, 8])
    x = rng.standard_normal((T, K)).astype(np.float32)
    w = matmul.Q4_0Matrix(O.random_q4_0(rng, N, K).view(np.uint8), K, N)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    y = lora.project(ad, w, _put(x), _put(np.full(T, -1, np.int32)))
    y0 = matmul.mul_mat_q4_0(w, _put(x))
    device.synchronize()
    assert np.array_equal(y.numpy(np.float32).view(np.uint32), y0.numpy(np.float32).view(np.uint32))


@pytest.mark.parametrize("project", [False, True])
@pytest.mark.parametrize("T", [1, 30])
def test_replayed_with_other_adapters(gpu, T, project):
    """A captured call replayed with other activations and other ids."""
    from arclight_amd import device, fattn, lora, matmul
    _case(f"lora replayed, T={T}, project={project}")
    rng = np.random.default_rng(260)
    K, N, R, n = 4096, 512, 16, 6
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    wo = O.random_q4_0(rng, N, K)
    w = matmul.Q4_0Matrix(wo.view(np.uint8), K, N)
    x, ids, base, y = (_put(np.zeros(s, t)) for s, t in (((T, K), np.float32), ((T,), np.int32), ((T, N), np.float32), ((T, N), np.float32)))
    st = device.Stream()
    c = lora.ProjectCall(ad, w, x, ids, y, st) if project else lora.ApplyCall(ad, x, ids, base, y, st)
    c.run()
    st.synchronize()
    g = device.Graph(st, c.run)
    for i in range(5):
        hx, hb = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
        hi = _ids(rng, T, n, "any")
        for d, h in ((x, hx), (base, hb), (ids, hi)):
            d.buf.upload(h)
        device.synchronize()
        g.launch(st)
        st.synchronize()
        fattn.device_errors()
        ref = _ref(hx, a, b, np.ones(n), [R] * n, hi, O.mul_mat_q4_0(wo, hx) if project else hb)
        if project:
            ref = ref[0], ref[1] + (K // 32 + 16) * 2 * EPS32 * abs_bound(dequant_q4_0(wo), dequant_q8_0(O.quantize_q8_0(hx)))
        _check(y.numpy(np.float32), ref, f"replay {i}")
    g.destroy()
    st.destroy()


def test_workspace_of_the_caller(gpu):
    from arclight_amd import _lib, device, lora, matmul
    rng = np.random.default_rng(270)
    K, N, R, n, T = 4096, 256, 16, 4, 20
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    x, ids = rng.standard_normal((T, K)).astype(np.float32), _ids(rng, T, n, "any")
    wo = O.random_q4_0(rng, N, K)
    w = matmul.Q4_0Matrix(wo.view(np.uint8), K, N)
    y = _put(np.zeros((T, N), np.float32))
    need = lora.ProjectCall(ad, w, _put(x), _put(ids), y).workspace_bytes()
    ws = device.DeviceBuffer(need)
    ws.upload(np.full(need, 0xff, np.uint8))
    lora.ProjectCall(ad, w, _put(x), _put(ids), y, workspace=ws).run()
    device.synchronize()
    ref = _ref(x, a, b, np.ones(n), [R] * n, ids, O.mul_mat_q4_0(wo, x))
    bound = ref[1] + (K // 32 + 16) * 2 * EPS32 * abs_bound(dequant_q4_0(wo), dequant_q8_0(O.quantize_q8_0(x)))
    _check(y.numpy(np.float32), (ref[0], bound), "workspace")
    with pytest.raises(_lib.ArclightError) as e:
        lora.ProjectCall(ad, w, _put(x), _put(ids), y, workspace=device.DeviceBuffer(need - 256)).run()
    assert e.value.status == abi.AL_ERR_WORKSPACE


@pytest.mark.parametrize("T", [65, 256, 384, 385, 513, 900])
@pytest.mark.parametrize("how", ["each its own", "in turn", "none", "two kinds of none"])
def test_groups_of_rows(gpu, T, how):
    """Every row of another adapter, 33 in turn, no row with one, with the
    last row's alone: base is copied, in a workspace of the size that is asked
    for and no more, that held other values."""
    from arclight_amd import device, fattn, lora
    _case(f"lora groups: T={T}, {how}")
    rng = np.random.default_rng(280 + T)
    K, N, R = 64, 20, 8
    n = T if how == "each its own" else 33
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    ids = {"each its own": rng.permutation(n), "in turn": np.arange(T) % 33, "none": np.full(T, -1),
           "two kinds of none": np.where(np.arange(T) == T - 1, 5, -1 - np.arange(T) % 2 * 1000)}[how].astype(np.int32)
    x, base = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    xd, idd, bd, y = _put(x), _put(ids), _put(base), _put(np.full((T, N), 7.0, np.float32))
    need = lora.ApplyCall(ad, xd, idd, bd, y).workspace_bytes()
    ws = device.DeviceBuffer(need + 4096)
    ws.upload(np.full(need + 4096, 0xa5, np.uint8))
    fit = SimpleNamespace(ptr=ws.ptr, nbytes=need)
    for _ in range(2):
        lora.ApplyCall(ad, xd, idd, bd, y, workspace=fit).run()
    device.synchronize()
    fattn.device_errors()
    tail = np.zeros(need + 4096, np.uint8)
    ws.download(tail)
    assert np.all(tail[need:] == 0xa5)
    _check(y.numpy(np.float32), _ref(x, a, b, np.ones(n), [R] * n, ids, base), how)


def test_a_growing_workspace_leaves_the_graphs_theirs(gpu):
    """A captured call replayed after calls on its stream that need a larger
    workspace of the library's, and buffers that would take a freed one's
    place."""
    from arclight_amd import _lib, device, fattn, lora
    _case("lora: a workspace that grows")
    rng = np.random.default_rng(290)
    K, N, R, n, T = 512, 64, 16, 4, 50
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
    x, ids, base = rng.standard_normal((T, K)).astype(np.float32), _ids(rng, T, n, "any"), rng.standard_normal((T, N)).astype(np.float32)
    ref = _ref(x, a, b, np.ones(n), [R] * n, ids, base)
    y = _put(np.zeros((T, N), np.float32))
    st = device.Stream()
    small = lora.ApplyCall(ad, _put(x), _put(ids), _put(base), y, st)
    small.run()
    st.synchronize()
    g = device.Graph(st, small.run)
    kept = []
    for i, rows in enumerate((50000, 120000)):                         # v of 26 and 61 MB
        a1, b1 = _adapters(rng, 2, 128, 8, 4, [128] * 2)
        x1, i1, base1 = rng.standard_normal((rows, 8)).astype(np.float32), _ids(rng, rows, 2, "any"), np.zeros((rows, 4), np.float32)
        y1 = _put(base1)
        big = lora.ApplyCall(lora.Adapters(_put(a1.view(np.uint16)), _put(b1.view(np.uint16))), _put(x1), _put(i1), _put(base1), y1, st)
        assert big.workspace_bytes() > (20 << 20) * (i + 1)
        big.run()
        st.synchronize()
        some = rng.choice(rows, 500, replace=False)
        some[0] = rows - 1
        _check(y1.numpy(np.float32)[some], _ref(x1[some], a1, b1, np.ones(2), [128] * 2, i1[some], base1[some]), f"{rows} rows")
        kept += [_put(np.full(5 << 20, 1e30, np.float32)) for _ in range(2)]
        for _ in range(2):
            y.buf.zero()
            device.synchronize()
            g.launch(st)
            st.synchronize()
            _check(y.numpy(np.float32), ref, "replay")
    assert all(np.all(k.numpy(np.float32) == np.float32(1e30)) for k in kept)
    fattn.device_errors()
    g.destroy()
    assert _lib.load().al_fattn_release_stream(st.handle) == 0
    small.run()
    st.synchronize()
    _check(y.numpy(np.float32), ref, "after the release")
    assert _lib.load().al_fattn_release_stream(st.handle) == 0
    st.destroy()


def test_two_streams_and_columns_of_one_matrix(gpu):
    """Calls on two streams, each with the library's workspace of its stream;
    base and y are columns of one matrix, either first."""
    from arclight_amd import device, fattn, lora
    _case("lora on two streams")
    rng = np.random.default_rng(300)
    K, N, R, n, T = 2048, 512, 32, 5, 130
    sides = []
    for i in range(2):
        a, b = _adapters(rng, n, R, K, N, [R] * n)
        x, ids = rng.standard_normal((T, K)).astype(np.float32), _ids(rng, T, n, "any")
        wide = rng.standard_normal((T, 2 * N)).astype(np.float32)
        d = _put(wide)
        cols = [device.DeviceTensor(d.buf, abi.AL_TYPE_F32, (T, N), (2 * N * 4, 4), off) for off in (0, N * 4)]
        st = device.Stream()
        ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)))
        base, y = cols[i], cols[1 - i]
        sides.append((st, lora.ApplyCall(ad, _put(x), _put(ids), base, y, st), d, wide, i, _ref(x, a, b, np.ones(n), [R] * n, ids, wide[:, i * N:(i + 1) * N])))
    for _ in range(20):
        for s in sides:
            s[1].run()
    device.synchronize()
    fattn.device_errors()
    for st, _, d, wide, i, ref in sides:
        got = d.numpy(np.float32)
        assert np.array_equal(got[:, i * N:(i + 1) * N], wide[:, i * N:(i + 1) * N])
        _check(got[:, (1 - i) * N:(2 - i) * N], ref, f"stream {i}")
        st.destroy()


@pytest.mark.parametrize("K, N, R", [(4096, 2560, 16), (4096, 4099, 32), (8192, 33, 24), (12288, 20, 16), (4096, 70, 48), (8192, 4100, 8),
                                     (16384, 5, 16), (4096, 4097, 40), (4096, 96, 64)])
def test_one_token_through_the_projection(gpu, K, N, R):
    """Sizes on both sides of where one token's launches become one; each rank
    from none to the slot's, scales, no adapter, and adapters that are not to
    be used."""
    from arclight_amd import _lib, device, fattn, lora, matmul
    _case(f"project one token {K} {N} {R}")
    rng = np.random.default_rng(310)
    ranks = np.array([0, 1, 7, 8, R - 1, R, R + 1, -2])
    n = len(ranks)
    a, b = _adapters(rng, n, R, K, N, np.clip(ranks, 0, R))
    scales = (rng.random(n) * 2).astype(np.float32)
    wo = O.random_q4_0(rng, N, K)
    w = matmul.Q4_0Matrix(wo.view(np.uint8), K, N)
    ad = lora.Adapters(_put(a.view(np.uint16)), _put(b.view(np.uint16)), _put(scales), _put(ranks.astype(np.int32)))
    x = (rng.standard_normal((1, K)) * 3).astype(np.float32)
    xd, base = _put(x), O.mul_mat_q4_0(wo, x)
    more = (K // 32 + 16) * 2 * EPS32 * abs_bound(dequant_q4_0(wo), dequant_q8_0(O.quantize_q8_0(x)))
    for i in (-1, *range(n), n, 1 << 30):
        y = _put(np.full((1, N), 5.0, np.float32))
        lora.project(ad, w, xd, _put(np.array([i], np.int32)), y)
        device.synchronize()
        if i >= 6:
            with pytest.raises(_lib.ArclightError) as e:
                fattn.device_errors()
            assert e.value.status == abi.AL_ERR_INVALID and np.all(np.isnan(y.numpy(np.float32))), i
            continue
        fattn.device_errors()
        ref, bound = _ref(x, a, b, scales, ranks, [i], base)
        err = np.abs(y.numpy(np.float32).astype(np.float64) - ref)
        assert np.all(err <= bound + more), (i, float((err / (bound + more)).max()))


@pytest.mark.parametrize("T", [40, 70])
def test_rows_past_32_bits(gpu, T):
    """Rows of x, base and y 2^27 bytes apart, adapters 3 GB apart."""
    from arclight_amd import device, fattn, lora
    _case(f"lora: offsets past 4 GB, T={T}")
    rng = np.random.default_rng(320)
    K, N, R, n, apart, slot = 256, 64, 8, 3, 1 << 27, 3 << 30
    a, b = _adapters(rng, n, R, K, N, [R] * n)
    ids = _ids(rng, T, n, "any")
    x, base = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    rows = device.DeviceBuffer(apart * (T - 1) + 4096)                 # x at 0, base at 1024, y at 2048 of each row
    for t in range(T):
        rows.upload(x[t], apart * t)
        rows.upload(base[t], apart * t + 1024)
    slots = device.DeviceBuffer(slot * (n - 1) + 8192)                 # A at 0, B at 4096 of each slot
    for i in range(n):
        slots.upload(a[i].view(np.uint16), slot * i)
        slots.upload(b[i].view(np.uint16), slot * i + 4096)
    view = lambda cols, off: device.DeviceTensor(rows, abi.AL_TYPE_F32, (T, cols), (apart, 4), off)  # noqa: E731
    ad = lora.Adapters(device.DeviceTensor(slots, abi.AL_TYPE_F16, (n, R, K), (slot, K * 2, 2)),
                       device.DeviceTensor(slots, abi.AL_TYPE_F16, (n, N, R), (slot, R * 2, 2), 4096))
    lora.ApplyCall(ad, view(K, 0), _put(ids), view(N, 1024), view(N, 2048)).run()
    device.synchronize()
    fattn.device_errors()
    got = np.stack([rows.download(np.empty(N, np.float32), apart * t + 2048) for t in range(T)])
    _check(got, _ref(x, a, b, np.ones(n), [R] * n, ids, base), "offsets")
