"""Steps of a server that drafts, as they would be run: the trees' tables, the
append by cell, attention in a layer that sees all and in one with a window,
verification, the accepted paths' cells kept in both layers and the next
step's lengths from them; eager and captured."""
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


@pytest.mark.parametrize("mode", ["neox", "normal", None])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append_by_cell(gpu, heads_first, mode):
    """Rows rotated by their positions in cells that are others, padding rows
    among them; cells that the table does not have."""
    from arclight_amd import device, fattn, paged
    from arclight_amd._lib import ArclightError
    _case(f"append by cell, {mode}")
    rng = np.random.default_rng(3)
    lens, Hq, Hkv, page = [40, 70], 8, 2, 24
    pool = P.Pool(rng, lens, Hkv, page, heads_first)
    pool.k[:], pool.v[:] = np.nan, np.nan
    cells = np.concatenate([rng.permutation(40)[:9], rng.permutation(70)[:20], [5, 5]]).astype(np.int32)
    seq = np.array([0] * 9 + [1] * 20 + [-1, -1], np.int32)
    pos = rng.integers(0, 5000, len(seq)).astype(np.int32)
    q, k, v = (rng.standard_normal((len(seq), H, D)).astype(np.float32) for H in (Hq, Hkv, Hkv))
    rope = None if mode is None else abi.qwen3_rope()
    if rope is not None:
        rope.mode = abi.AL_ROPE_NEOX if mode == "neox" else abi.AL_ROPE_NORMAL
    cache = pool.device()
    out = paged.append(cache, _put(q), _put(k), _put(v), _put(pos), _put(seq), eps=1e-6, rope=rope, cells=_put(cells))
    device.synchronize()
    fattn.device_errors()
    mine = seq >= 0
    kr, qr = (P.norm_rotate(x, None, pos, 1e-6, mode) for x in (k, q))
    for t in np.flatnonzero(mine):
        at = pool.table[seq[t], cells[t] // page], cells[t] % page
        pool.k[at], pool.v[at] = kr[t].astype(np.float16), v[t].astype(np.float16)
    got_k, got_v = pool.download(cache)
    assert np.array_equal(got_v.view(np.uint16), pool.v.view(np.uint16))
    seen = ~np.isnan(pool.k)
    assert np.array_equal(seen, ~np.isnan(got_k))
    # one float16 step, and 3e-5 of the producers' float32
    assert np.all(np.abs(got_k[seen].astype(np.float64) - pool.k[seen]) <= np.abs(pool.k[seen].astype(np.float64)) * 2.0 ** -10 + 3e-5)
    assert np.all(np.abs(out.numpy(np.float32)[mine] - qr[mine]) <= 3e-5 + 1e-6 * np.abs(qr[mine]))
    for bad, text in ((pool.max_pages * page, "cell"), (-1, "cell"), (40 + page, "page")):
        wrong = cells.copy()
        wrong[0] = bad
        paged.append(cache, None, _put(k), _put(v), _put(pos), _put(seq), None, eps=1e-6, rope=rope, cells=_put(wrong))
        device.synchronize()
        with pytest.raises(ArclightError, match=text):
            fattn.device_errors()


@pytest.mark.parametrize("replayed", [False, True])
def test_steps_of_a_server_that_drafts(gpu, replayed):
    from arclight_amd import device, draft, fattn, paged
    _case(f"steps with trees, replayed={replayed}")
    rng = np.random.default_rng(40)
    n, T, Hq, Hkv, page, V, window, first = 4, 11, 8, 2, 16, 700, 24, 3
    W = (T + 31) // 32
    pools = [P.Pool(rng, [0] * n, Hkv, page, spare=60, max_pages=10) for _ in range(2)]
    free, table = list(rng.permutation(60)), np.full((n, 10), -4, np.int32)
    lens = [20, 0, 57, 130]
    for s, m in enumerate(lens):
        for i in range((m + page - 1) // page):
            table[s, i] = free.pop()
        for c in range(m):
            for pool in pools:
                pool.k[table[s, c // page], c % page], pool.v[table[s, c // page], c % page] = rng.standard_normal((2, Hkv, D))
    for pool in pools:
        pool.table = table
    caches = [pool.device() for pool in pools]
    td = caches[0].table
    caches = [paged.PagedCache(c.k, c.v, td) for c in caches]
    st = device.Stream()
    shapes = {"parents": (n, T), "counts": (n,), "lens": (n,), "pos": (n, T), "cells": (n, T), "seq": (n, T), "bits": (n, T, W), "tokens": (n, T),
              "path": (n, T), "kept": (n,), "next": (n,), "lens_out": (n,)}
    buf = {k: device.DeviceTensor.from_numpy(np.zeros(s, np.int32)) for k, s in shapes.items()}
    floats = {"q0": (n * T, Hq, D), "q1": (n * T, Hq, D), "k0": (n * T, Hkv, D), "k1": (n * T, Hkv, D), "v0": (n * T, Hkv, D), "v1": (n * T, Hkv, D),
              "r0": (n * T, Hq, D), "r1": (n * T, Hq, D), "o0": (n, T, Hq, D), "o1": (n, T, Hq, D), "target": (n, T, V), "accept": (n, T), "sample": (n,)}
    buf |= {k: device.DeviceTensor.from_numpy(np.zeros(s, np.float32)) for k, s in floats.items()}
    flat = {k: device.DeviceTensor(buf[k].buf, abi.AL_TYPE_I32, (n * T,)) for k in ("pos", "cells", "seq")}
    calls = [draft.TreeCall(*(buf[k] for k in ("parents", "lens", "counts", "pos", "cells", "seq", "bits")), stream=st)]
    for i, c in enumerate(caches):
        calls.append(paged.AppendCall(c, buf[f"q{i}"], buf[f"k{i}"], buf[f"v{i}"], flat["pos"], flat["seq"], buf[f"r{i}"], eps=1e-6,
                                      rope=abi.qwen3_rope(), cells=flat["cells"], stream=st))
        q = device.DeviceTensor(buf[f"r{i}"].buf, abi.AL_TYPE_F32, (n, T, Hq, D))
        rule = {"window": window, "first": first, "pos": buf["pos"]} if i else {}
        calls.append(paged.AttentionCall(c, q, buf["lens"], buf[f"o{i}"], counts=buf["counts"], scale=SCALE, bits=buf["bits"], stream=st, **rule))
    calls.append(draft.VerifyCall(*(buf[k] for k in ("target", "tokens", "accept", "sample", "path", "kept", "next")), parents=buf["parents"],
                                  counts=buf["counts"], stream=st))
    calls.append(paged.KeepCall(caches, buf["lens"], buf["counts"], buf["path"], buf["kept"], buf["lens_out"], stream=st))

    def step():
        for c in calls:
            c.run()

    graph, longest = None, 0
    for i in range(7):
        counts = [T if s != i % n else int(rng.integers(0, T)) for s in range(n)]
        parents = np.stack([C.random_tree(rng, T, 0.7) for _ in range(n)])
        for s in range(n):
            have = (lens[s] + page - 1) // page
            lens[s] += counts[s]
            for j in range(have, (lens[s] + page - 1) // page):
                table[s, j] = free.pop()
        target = rng.random((n, T, V)) ** 40
        target = (target / target.sum(-1, keepdims=True)).astype(np.float32)
        tokens = rng.integers(0, V, (n, T))
        for s in range(n):
            for u in range(1, T):
                tokens[s, u] = np.argsort(-target[s, parents[s, u]])[rng.integers(0, 3)]
        host = {"parents": parents, "counts": np.array(counts, np.int32), "lens": np.array(lens, np.int32), "tokens": tokens.astype(np.int32),
                "target": target, "accept": (rng.random((n, T)) * 0.1).astype(np.float32), "sample": rng.random(n).astype(np.float32)}
        host |= {k: rng.standard_normal(floats[k]).astype(np.float32) for k in ("q0", "q1", "k0", "k1", "v0", "v1")}
        host |= {k: np.full(floats[k], MARK, np.float32) for k in ("o0", "o1")}
        for k, x in host.items():
            buf[k].buf.upload(x)
        td.buf.upload(table)
        device.synchronize()
        if replayed and i == 1:
            graph = device.Graph(st, step)
        graph.launch(st) if graph else step()
        device.synchronize()
        fattn.device_errors()
        # each stage against its definition, on what the stage before it gave
        made = [C.tree(parents[s], lens[s], counts[s], W) for s in range(n)]
        got = {k: buf[k].numpy(np.int32) for k in ("pos", "cells", "seq", "bits", "path", "kept", "next", "lens_out")}
        for s in range(n):
            assert all(np.array_equal(got[k][s], m) for k, m in zip(("pos", "cells", "bits"), (made[s][0], made[s][1], made[s][3])))
            assert np.array_equal(got["seq"][s], np.where(made[s][2] < 0, -1, s))
        seq = got["seq"].reshape(-1)
        for layer, pool in enumerate(pools):
            kr = P.norm_rotate(host[f"k{layer}"], None, got["pos"].reshape(-1), 1e-6, "neox")
            before = pool.k.copy(), pool.v.copy()
            for t in np.flatnonzero(seq >= 0):
                c = got["cells"].reshape(-1)[t]
                at = table[seq[t], c // page], c % page
                before[0][at], before[1][at] = kr[t].astype(np.float16), host[f"v{layer}"][t].astype(np.float16)
            # the accepted cells lie where they are kept
            moved = [x.copy() for x in before]
            for s in range(n):
                b = lens[s] - counts[s]
                for j in range(got["kept"][s]):
                    a, z = b + int(got["path"][s, j]), b + j
                    for new, old in zip(moved, before):
                        new[table[s, z // page], z % page] = old[table[s, a // page], a % page]
            dk, dv = pool.download(caches[layer])
            seen = ~np.isnan(moved[0])
            assert np.array_equal(dv.view(np.uint16)[seen], moved[1].view(np.uint16)[seen]) and np.array_equal(seen, ~np.isnan(dk))
            assert np.all(np.abs(dk[seen].astype(np.float64) - moved[0][seen]) <= np.abs(moved[0][seen].astype(np.float64)) * 2.0 ** -10 + 3e-5)
            # attention read the cells before the move: those that stayed are the device's
            stay = dk.copy()
            whole = P.Pool.__new__(P.Pool)
            whole.__dict__.update(pool.__dict__)
            whole.k, whole.v = before
            # (keys that moved away are taken from where they went)
            for s in range(n):
                b = lens[s] - counts[s]
                back = {int(got["path"][s, j]): j for j in range(got["kept"][s])}
                for u in range(counts[s]):
                    z = back.get(u)
                    at = table[s, (b + u) // page], (b + u) % page
                    if z is not None:
                        before[0][at] = stay[table[s, (b + z) // page], (b + z) % page]
                    elif u >= got["kept"][s]:
                        before[0][at] = stay[at]
            q = buf[f"r{layer}"].numpy(np.float32).reshape(n, T, Hq, D)
            rule = (window, first) if layer else (0, 0)
            sees = [C.visible(m, c, T, *rule, b, p if layer else None) for m, c, b, p in zip(lens, counts, got["bits"], got["pos"])]
            # a key in a place that was written over is the host's, within a float16 step of the device's: its cells' rows are not compared
            lost = [[lens[s] - counts[s] + u for u in range(min(counts[s], got["kept"][s])) if u not in set(got["path"][s].tolist())] for s in range(n)]
            ref, bound = C.attention(whole, q, lens, counts, SCALE, sees)
            out = buf[f"o{layer}"].numpy(np.float32)
            clean = np.array([[t >= counts[s] or not sees[s][t, lost[s]].any() for t in range(T)] for s in range(n)])
            _check(out[clean], (ref[clean], bound[clean]), f"step {i}, layer {layer}")
            pool.k, pool.v = dk.copy(), dv.copy()
        for s in range(n):
            want, follow = C.verify(target[s], tokens[s], host["accept"][s], host["sample"][s], parents[s], counts[s])
            assert list(got["path"][s, :len(want)]) == want and got["kept"][s] == len(want) and got["next"][s] == follow
            longest = max(longest, len(want))
            lens[s] += got["kept"][s] - counts[s]
            assert got["lens_out"][s] == lens[s]
            for j in range((lens[s] + page - 1) // page, 10):            # pages behind the kept cells are free again
                if table[s, j] >= 0:
                    free.insert(0, table[s, j])
                    table[s, j] = -4
    assert longest >= 3
    if graph:
        graph.destroy()
    st.destroy()


def test_forks_of_a_sequence(gpu):
    """A sequence forked in the middle of a page: the fork shares its full
    pages, has a copy of the last one, and both go on with tokens of their own."""
    from arclight_amd import device, fattn, paged
    _case("a fork")
    rng = np.random.default_rng(41)
    page, Hq, Hkv, m = 16, 8, 2, 41
    pool = P.Pool(rng, [m, 0], Hkv, page, spare=1, max_pages=3)
    spare = (set(range(pool.n_pages)) - set(pool.table[0].tolist())).pop()
    pool.table[1] = pool.table[0]
    pool.table[1, 2] = spare
    cache = pool.device()
    paged.copy_pages([cache], _put(pool.table[0, 2:3].copy()), _put(pool.table[1, 2:3].copy()), _put(np.array([m % page], np.int32)))
    pool.k[spare, :m % page], pool.v[spare, :m % page] = pool.k[pool.table[0, 2], :m % page], pool.v[pool.table[0, 2], :m % page]
    k, v = (rng.standard_normal((2, Hkv, D)).astype(np.float32) for _ in range(2))
    paged.append(cache, None, _put(k), _put(v), _put(np.array([m, m], np.int32)), _put(np.array([0, 1], np.int32)), norm=False)
    for s in range(2):
        at = pool.table[s, m // page], m % page
        pool.k[at], pool.v[at] = k[s].astype(np.float16), v[s].astype(np.float16)
    q = rng.standard_normal((2, 1, Hq, D)).astype(np.float32)
    out = paged.attention(cache, _put(q), _put(np.array([m + 1] * 2, np.int32)), scale=SCALE)
    device.synchronize()
    fattn.device_errors()
    for x, y in zip(pool.download(cache), (pool.k, pool.v)):
        assert np.array_equal(x.view(np.uint16), y.view(np.uint16))
    _check(out.numpy(np.float32), P.attention(pool, q, [m + 1] * 2, [1, 1], SCALE), "fork")
