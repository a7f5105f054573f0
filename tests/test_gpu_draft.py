"""Trees of drafted tokens on the GPU: their tables and their verification
against the definitions (tests/tree_cases.py); whole numbers, equal to the
last."""
import numpy as np
import pytest

from arclight_amd import abi
from tests import tree_cases as C
from tests.test_gpu_paged import _case, _put

pytestmark = pytest.mark.gpu
MARK = -77


def _sync(errors=True):
    from arclight_amd import device, fattn
    device.synchronize()
    if errors:
        fattn.device_errors()


@pytest.mark.parametrize("n, T, words, bushy", [(1, 1, 1, 0.5), (3, 2, 1, 0.5), (5, 31, 1, 0.6), (4, 32, 2, 0.3), (70, 33, 2, 0.8), (3, 64, 5, 0.0),
                                                (4, 65, 3, 0.7), (2, 500, 16, 0.9), (2, 1024, 32, 0.0), (2, 1024, 33, 0.95)])
def test_tree(gpu, n, T, words, bushy):
    from arclight_amd import draft
    _case(f"tree tables {n} x {T}")
    rng = np.random.default_rng(T * 7 + n)
    parents = np.stack([C.random_tree(rng, T, bushy) for _ in range(n)])
    parents[0, T // 2] = -1                                          # a second root
    counts = rng.integers(0, T + 1, n)
    counts[0] = T
    lens = counts + rng.integers(0, 2 ** 20, n)
    lens[-1] = counts[-1]
    outs = [_put(np.full((n, T), MARK, np.int32)) for _ in range(3)] + [_put(np.full((n, T, words), MARK, np.int32))]
    draft.TreeCall(_put(parents), _put(lens.astype(np.int32)), _put(counts.astype(np.int32)), *outs).run()
    _sync()
    got = [o.numpy(np.int32) for o in outs]
    for s in range(n):
        pos, cells, seq, bits = C.tree(parents[s], int(lens[s]), int(counts[s]), words)
        for g, w in zip(got, (pos, cells, np.where(seq < 0, -1, s), bits)):
            assert np.array_equal(g[s], w), s


def test_tree_parts_and_strides(gpu):
    """Outputs that are left out, operands in wider rows."""
    from arclight_amd import device, draft
    _case("tree tables, strides")
    rng = np.random.default_rng(5)
    n, T = 3, 40
    parents = np.full((n, T + 3), 99, np.int32)
    for s in range(n):
        parents[s, :T] = C.random_tree(rng, T)
    lens = np.array([40, 50, 1000], np.int32)
    pd, pos = _put(parents), _put(np.full((n, T + 1), MARK, np.int32))
    bits = _put(np.full((n, T + 2, 3), MARK, np.int32))
    view = lambda t, shape, strides: device.DeviceTensor(t.buf, abi.AL_TYPE_I32, shape, strides)  # noqa: E731
    draft.TreeCall(view(pd, (n, T), ((T + 3) * 4, 4)), _put(lens), None, view(pos, (n, T), ((T + 1) * 4, 4)), None, None,
                   view(bits, (n, T, 2), ((T + 2) * 12, 12, 4))).run()
    _sync()
    p, b = pos.numpy(np.int32), bits.numpy(np.int32)
    assert np.all(p[:, T:] == MARK) and np.all(b[:, T:] == MARK) and np.all(b[:, :, 2] == MARK)
    for s in range(n):
        want = C.tree(parents[s, :T], int(lens[s]), T)
        assert np.array_equal(p[s, :T], want[0]) and np.array_equal(b[s, :T, :2], want[3])


def test_tree_reports_wrong_parents_and_counts(gpu):
    from arclight_amd import draft, fattn
    from arclight_amd._lib import ArclightError
    _case("tree tables, wrong parents")
    T = 5
    for bad, value in ((0, 0), (2, 2), (2, 2 ** 31 - 1), (4, 7)):
        parents = np.array([[-1, 0, 1, 1, 0], [-1, 0, 0, 0, 0]], np.int32)
        parents[0, bad] = value
        got = [t.numpy(np.int32) for t in draft.tree(_put(parents), _put(np.array([9, 9], np.int32)))]
        with pytest.raises(ArclightError, match="parent"):
            _sync() or fattn.device_errors()
        for s in range(2):
            pos, cells, _, bits = C.tree(parents[s], 9, T)
            assert np.array_equal(got[0][s], pos) and np.array_equal(got[1][s], cells) and np.array_equal(got[3][s], bits)
    for count, length in ((-1, 9), (6, 9), (4, 3)):
        parents = np.array([[-1, 0, 1, 1, 0]] * 2, np.int32)
        got = [t.numpy(np.int32) for t in draft.tree(_put(parents), _put(np.array([length, 9], np.int32)), _put(np.array([count, 5], np.int32)))]
        with pytest.raises(ArclightError, match="tree of"):
            _sync() or fattn.device_errors()
        assert not got[0][0].any() and np.all(got[2][0] == -1) and not got[3][0].any() and np.all(got[2][1] == 1)


def _probabilities(rng, *shape):
    x = rng.standard_normal(shape) * 2.5
    x = np.exp(x - x.max(-1, keepdims=True))
    return (x / x.sum(-1, keepdims=True)).astype(np.float32)


def _verify(target, tokens, accept, sample, parents=None, counts=None, draft=None, errors=True, stream=None):
    from arclight_amd import draft as D
    i32 = lambda x: None if x is None else _put(np.asarray(x, np.int32))  # noqa: E731
    out = D.verify(_put(target), i32(tokens), _put(accept.astype(np.float32)), _put(sample.astype(np.float32)), parents=i32(parents),
                   counts=i32(counts), draft=None if draft is None else _put(draft), stream=stream)
    _sync(errors)
    return [t.numpy(np.int32) for t in out]


def _same(got, target, tokens, accept, sample, parents=None, counts=None, draft=None):
    path, kept, nxt = got
    accept, sample = accept.astype(np.float32), sample.astype(np.float32)
    depths = []
    for s in range(target.shape[0]):
        want, follow = C.verify(target[s], tokens[s], accept[s], sample[s], None if parents is None else parents[s],
                                None if counts is None else int(counts[s]), None if draft is None else draft[s])
        assert kept[s] == len(want) and list(path[s, :len(want)]) == want and np.all(path[s, len(want):] == -1), (s, path[s], want)
        assert nxt[s] == follow, (s, nxt[s], follow)
        depths.append(len(want))
    return depths


def _children(rng, target, parents, drafted=None):
    """Tokens for the nodes: drawn from the draft's row of the parent, or among
    the target's likely ones, some of them twice."""
    n, T, V = target.shape
    out = np.full((n, T), 7 % V)
    for s in range(n):
        for u in range(1, T):
            v = max(int(parents[s, u]), 0)
            if drafted is not None:
                p = drafted[s, v].astype(np.float64)
                out[s, u] = rng.choice(V, p=p / p.sum())
            else:
                out[s, u] = np.argsort(-target[s, v])[min(int(rng.integers(0, 4)), V - 1)]
    return out


@pytest.mark.parametrize("n, T, V", [(1, 1, 1), (2, 1, 5), (4, 2, 2), (6, 7, 33), (3, 26, 2048), (5, 20, 2049), (2, 40, 5000), (9, 12, 1000),
                                     (2, 3, 160001), (2, 300, 300)])
@pytest.mark.parametrize("kind", ["tree", "chain", "drafted chain", "drafted tree"])
def test_verify(gpu, n, T, V, kind):
    _case(f"verify {kind} {n} x {T} of {V}")
    rng = np.random.default_rng(n * 1000 + T + V)
    target = _probabilities(rng, n, T, V)
    parents = np.stack([C.random_tree(rng, T, 0.8) for _ in range(n)])
    if "chain" in kind:
        parents = np.tile(np.arange(-1, T - 1), (n, 1))
    draft = None
    if "drafted" in kind:
        draft = target * np.exp(rng.standard_normal(target.shape) * 0.7)
        draft = (draft / draft.sum(-1, keepdims=True)).astype(np.float32)
    tokens = _children(rng, target, parents, draft)
    counts = rng.integers(0, T + 1, n)
    counts[0] = T
    given = None if "chain" in kind else parents
    depths = []
    for again in range(3):
        accept, sample = rng.random((n, T)), rng.random(n)
        if again == 1:
            accept *= 0.3
        c = None if again == 2 else counts
        got = _verify(target, tokens, accept, sample, given, c, draft)
        depths += _same(got, target, tokens, accept, sample, given, c, draft)
        twice = _verify(target, tokens, accept, sample, given, c, draft)
        assert all(np.array_equal(a, b) for a, b in zip(got, twice))
    print(f"accepted paths of {sorted(set(depths))} nodes", flush=True)


def test_verify_on_the_border(gpu):
    """Probabilities whose sums are exact, random numbers on the borders: a
    child is rejected at accept = p, the token that follows is the first whose
    sum is above, tokens of no weight are never drawn."""
    _case("verify, borders")
    V = 8
    row = np.array([0.0, 0.25, 0.0, 0.25, 0.125, 0.125, 0.25, 0.0], np.float32)
    sample = np.array([0.0, 0.2499, 0.25, 0.5, 0.625, 0.75, 0.99, 1.0, 1.5, -1.0, np.nan, np.inf], np.float32)
    n = len(sample)
    target = np.tile(row, (n, 1, 1))
    tokens, accept = np.zeros((n, 1), int), np.zeros((n, 1))
    got = _verify(target, tokens, accept, sample)
    assert list(got[2]) == [1, 1, 3, 4, 5, 6, 6, 6, 6, 1, 6, 6]
    _same(got, target, tokens, accept, sample)
    # accept: below, at, above p; children of no weight; what two rejections leave
    target = np.tile(row, (7, 5, 1))
    parents = np.tile(np.array([-1, 0, 0, 0, 0]), (7, 1))
    tokens = np.tile(np.array([0, 1, 1, 3, 0]), (7, 1))              # 1 twice, 0 has no weight
    accept = np.array([[0, 0.2499, 0, 0, 0], [0, 0.25, 0, 0, 0], [0, 0.25, 0, 0.33, 0], [0, 0.25, 0, 0.334, 0], [0, 0.3, 0.0, 0.9, -1.0],
                       [0, np.nan, np.nan, np.nan, np.nan], [0, -1, 0, 0, 0]])
    sample = np.array([0.1, 0.1, 0.1, 0.1, 0.5, 0.0, 0.0])
    got = _verify(target, tokens, accept, sample, parents)
    assert list(got[0][:, 1]) == [1, 3, 3, -1, -1, -1, 1] and list(got[2][3:6]) == [4, 6, 4]
    _same(got, target, tokens, accept, sample, parents)


def test_verify_where_nothing_is_left(gpu):
    """All of the probability on a rejected token, a draft equal to the target:
    the target's own row is drawn from. Rows without any, infinities, NaN."""
    from arclight_amd import fattn
    from arclight_amd._lib import ArclightError
    _case("verify, nothing left")
    V, n = 3000, 3
    target = np.zeros((n, 3, V), np.float32)
    target[:, :, 2500] = 1.0
    tokens, accept, sample = np.full((n, 3), 2500), np.full((n, 3), 1.0), np.full(n, 0.5)
    parents = np.tile(np.array([-1, 0, 0]), (n, 1))
    for given, draft in ((None, None), (parents, None), (None, target.copy()), (parents, target.copy())):
        got = _verify(target, tokens, accept, sample, given, None, draft)
        assert list(got[1]) == [1] * n and list(got[2]) == [2500] * n
        _same(got, target, tokens, accept, sample, given, None, draft)
    rng = np.random.default_rng(3)
    target = _probabilities(rng, 4, 2, V)
    target[0, 0, ::3] = np.nan
    target[0, 0, 1::3] *= -1
    target[1, 0] = 0
    target[2, 0, 7] = np.inf
    target[3, 0] = np.nan
    tokens, accept, sample = np.full((4, 2), 2), np.full((4, 2), 1.0), np.full(4, 0.5)
    got = _verify(target, tokens, accept, sample, errors=False)
    with pytest.raises(ArclightError, match="probabilities"):
        fattn.device_errors()
    assert list(got[2][1:]) == [-1] * 3 and got[2][0] % 3 == 2
    _same([g[:1] for g in got], target[:1], tokens[:1], accept[:1], sample[:1])


def test_verify_reports_wrong_nodes(gpu):
    from arclight_amd import fattn
    from arclight_amd._lib import ArclightError
    _case("verify, wrong nodes")
    rng = np.random.default_rng(4)
    target = _probabilities(rng, 2, 4, 50)
    accept, sample = np.zeros((2, 4)), rng.random(2)
    tokens, parents = _children(rng, target, np.tile(np.array([-1, 0, 0, 1]), (2, 1))), np.tile(np.array([-1, 0, 0, 1]), (2, 1))
    for what, text, change in (("tokens", "vocabulary", 50), ("tokens", "vocabulary", -1), ("tokens", "vocabulary", -2 ** 31), ("parents", "parent", 1),
                               ("parents", "parent", 2 ** 31 - 1), ("counts", "tree of", 5), ("counts", "tree of", -2)):
        t, p, c = tokens.copy(), parents.copy(), np.array([4, 4])
        if what == "counts":
            c[0] = change
        else:
            {"tokens": t, "parents": p}[what][0, 1] = change
        for draft in (None, target[:, ::-1].copy()):
            got = _verify(target, t, accept, sample, p, c, draft, errors=False)
            with pytest.raises(ArclightError, match=text):
                fattn.device_errors()
            assert got[0][0, 1] in (-1, 2)
            _same(got, target, t, accept, sample, p, c, draft)


def test_verify_strides_and_rows_past_4_gb(gpu):
    """Rows that begin at any multiple of 4 bytes, a sequence's rows beyond 4 GB
    of the first's, operands in wider rows, beside a workspace of just the bytes
    asked for."""
    from arclight_amd import device, draft
    _case("verify, strides")
    rng = np.random.default_rng(6)
    n, T, V = 2, 3, 4099
    target = _probabilities(rng, n, T, V)
    apart, row = 5 * 2 ** 30 + 4, (V + 2) * 4
    buf = device.DeviceBuffer(apart + T * row + 64)
    for s in range(n):
        for t in range(T):
            buf.upload(target[s, t], 4 + apart * s + row * t)
    tokens = _children(rng, target, np.tile(np.arange(-1, T - 1), (n, 1)))
    wide = np.full((n, T + 2), -9, np.int32)
    wide[:, :T] = tokens
    path = _put(np.full((n, T + 1), MARK, np.int32))
    td = _put(wide)
    kept, nxt = _put(np.zeros(n, np.int32)), _put(np.zeros(n, np.int32))
    accept, sample = rng.random((n, T)).astype(np.float32) * 0.2, rng.random(n).astype(np.float32)
    c = draft.VerifyCall(device.DeviceTensor(buf, abi.AL_TYPE_F32, (n, T, V), (apart, row, 4), 4),
                         device.DeviceTensor(td.buf, abi.AL_TYPE_I32, (n, T), ((T + 2) * 4, 4)), _put(accept), _put(sample),
                         device.DeviceTensor(path.buf, abi.AL_TYPE_I32, (n, T), ((T + 1) * 4, 4)), kept, nxt)
    ws = device.DeviceBuffer(c.workspace_bytes())
    c.args.workspace, c.args.workspace_bytes = ws.ptr, ws.nbytes - 1
    with pytest.raises(Exception, match="workspace"):
        c.run()
    c.args.workspace_bytes = ws.nbytes
    c.run()
    _sync()
    p = path.numpy(np.int32)
    assert np.all(p[:, T] == MARK)
    _same([p[:, :T], kept.numpy(np.int32), nxt.numpy(np.int32)], target, tokens, accept, sample)


def test_verify_distribution(gpu):
    """What verification is for: with tokens drawn from a draft, accepted or
    followed tokens have the target's distribution, whatever the draft's. 40000
    trees of one node and two children each; the count of each of 6 tokens is off
    by at most 5 standard deviations."""
    _case("verify, distribution")
    rng = np.random.default_rng(8)
    n, V = 40000, 6
    p, q = (np.array(x, np.float32) for x in ([0.4, 0.05, 0.2, 0.05, 0.2, 0.1], [0.1, 0.3, 0.1, 0.3, 0.1, 0.1]))
    target, draft = np.tile(p, (n, 3, 1)), np.tile(q, (n, 3, 1))
    parents = np.tile(np.array([-1, 0, 0]), (n, 1))
    tokens = np.concatenate([np.zeros((n, 1), int), rng.choice(V, (n, 2), p=q.astype(np.float64) / q.astype(np.float64).sum())], 1)
    for given, d in ((tokens, draft), (np.tile([0, 1, 4], (n, 1)), None)):
        path, kept, nxt = _verify(target, given, rng.random((n, 3)), rng.random(n), parents, None, d)
        first = np.where(kept == 2, given[np.arange(n), np.maximum(path[:, 1], 0)], nxt)
        count = np.bincount(first, minlength=V)
        assert np.all(np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))), count


@pytest.mark.parametrize("drafted", [False, True])
def test_verify_replayed(gpu, drafted):
    """A captured call over buffers whose content changes, eager calls of the
    same stream between the replays."""
    from arclight_amd import device, draft
    _case(f"verify, replayed, drafted={drafted}")
    rng = np.random.default_rng(9)
    n, T, V = 4, 9, 3001
    st = device.Stream()
    buf = {k: device.DeviceTensor.from_numpy(np.zeros(s, t)) for k, s, t in
           (("target", (n, T, V), np.float32), ("draft", (n, T, V), np.float32), ("tokens", (n, T), np.int32), ("parents", (n, T), np.int32),
            ("counts", (n,), np.int32), ("accept", (n, T), np.float32), ("sample", (n,), np.float32), ("path", (n, T), np.int32),
            ("kept", (n,), np.int32), ("next", (n,), np.int32))}
    c = draft.VerifyCall(*(buf[k] for k in ("target", "tokens", "accept", "sample", "path", "kept", "next")), parents=buf["parents"],
                         counts=buf["counts"], draft=buf["draft"] if drafted else None, stream=st)
    graph = None
    for i in range(5):
        h = {"target": _probabilities(rng, n, T, V), "parents": np.stack([C.random_tree(rng, T, 0.8) for _ in range(n)]),
             "counts": rng.integers(1, T + 1, n).astype(np.int32), "accept": (rng.random((n, T)) * 0.6).astype(np.float32),
             "sample": rng.random(n).astype(np.float32)}
        h["draft"] = _probabilities(rng, n, T, V)
        h["tokens"] = _children(rng, h["target"], h["parents"], h["draft"] if drafted else None).astype(np.int32)
        for k, x in h.items():
            buf[k].buf.upload(x)
        device.synchronize()
        if i == 1:
            graph = device.Graph(st, c.run)
        graph.launch(st) if graph else c.run()
        _sync()
        _same([buf[k].numpy(np.int32) for k in ("path", "kept", "next")], h["target"], h["tokens"], h["accept"], h["sample"], h["parents"],
              h["counts"], h["draft"] if drafted else None)
        _verify(h["target"], h["tokens"], h["accept"], h["sample"], h["parents"], stream=st)
    graph.destroy()
    st.destroy()


def test_two_threads_with_streams_of_their_own(gpu):
    """Verification and attention of trees by two threads at once, on streams of
    their own and the library's workspaces: each call's results are those of the
    same call alone, bit for bit."""
    import threading

    from arclight_amd import device, draft, paged
    from tests import paged_cases as P
    _case("two threads")
    rng = np.random.default_rng(12)
    n, T, V, Hq, Hkv = 4, 30, 5000, 16, 4
    lens = [900, 30, 2100, 333]
    pool = P.Pool(rng, lens, Hkv, 16)
    cache, dl = pool.device(), _put(np.array(lens, np.int32))
    work = []
    for _ in range(2):
        parents = np.stack([C.random_tree(rng, T) for _ in range(n)])
        target = _probabilities(rng, n, T, V)
        tokens = _put(rng.integers(0, V, (n, T)).astype(np.int32))
        st = device.Stream()
        path, kept, nxt = (_put(np.zeros(s, np.int32)) for s in ((n, T), (n,), (n,)))
        v = draft.VerifyCall(_put(target.astype(np.float32)), tokens, _put(rng.random((n, T)).astype(np.float32)), _put(rng.random(n).astype(np.float32)),
                             path, kept, nxt, parents=_put(parents.astype(np.int32)), stream=st)
        q, out = _put(rng.standard_normal((n, T, Hq, 128)).astype(np.float32)), _put(np.zeros((n, T, Hq, 128), np.float32))
        bits = np.stack([C.tree(p, m, T)[3] for p, m in zip(parents, lens)])
        a = paged.AttentionCall(cache, q, dl, out, scale=0.09, bits=_put(bits), stream=st)
        v.run(), a.run()
        _sync()
        work.append((st, v, a, (path, kept, nxt, out), [x.numpy(t) for x, t in zip((path, kept, nxt, out), (np.int32,) * 3 + (np.float32,))]))
    wrong = []

    def run(st, v, a, outs, want):
        try:
            for _ in range(40):
                v.run(), a.run()
        except Exception as e:                                          # noqa: BLE001 (shown by the main thread)
            wrong.append(e)
    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    _sync()
    assert not wrong, wrong
    for st, _, _, outs, want in work:
        for x, w in zip(outs, want):
            assert np.array_equal(x.numpy(w.dtype), w)
        st.destroy()


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("T", [9, 300])
def test_nodes_behind_the_count_hold_anything(gpu, T, drafted):
    """Tokens, parents and numbers of nodes that are not there: not followed, and
    nothing recorded."""
    _case(f"verification, nodes behind the count, T={T}, drafted={drafted}")
    rng = np.random.default_rng(T)
    n, V = 6, 700
    target = _probabilities(rng, n, T, V)
    drafts = _probabilities(rng, n, T, V) if drafted else None
    parents = np.stack([C.random_tree(rng, T, 0.6) for _ in range(n)])
    tokens = _children(rng, target, parents, drafts)
    accept, sample, counts = rng.random((n, T)), rng.random(n), np.array([0, 1, 2, T // 2, T - 1, T])
    for s, c in enumerate(counts):
        parents[s, c:] = rng.choice([-2 ** 31, -9, T, 2 ** 31 - 1, c, 0], T - c)
        tokens[s, c:] = rng.choice([-2 ** 31, -1, V, 2 ** 31 - 1, 3], T - c)
        accept[s, c:] = rng.choice([np.nan, np.inf, -1.0, 0.5], T - c)
    got = _verify(target, tokens, accept, sample, parents, counts, drafts)
    some = counts > 0
    _same([x[some] for x in got], target[some], tokens[some], accept[some], sample[some], parents[some], counts[some], None if drafts is None else drafts[some])
    assert got[1][0] == 0 and got[2][0] == -1 and np.all(got[0][0] == -1)
