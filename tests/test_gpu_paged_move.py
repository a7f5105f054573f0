"""Cells moved in all layers on the GPU: an accepted path's, and pages. Copies,
equal to the last bit; what is not named stays as it was."""
import numpy as np
import pytest

from arclight_amd import abi
from tests.test_gpu_paged import _case, _put

pytestmark = pytest.mark.gpu
D = 128
MARK = -77


class Layers:
    def __init__(self, rng, n_layers, n_pages, page, Hkv, heads_first=False, table=None):
        from arclight_amd import paged
        shape = (n_pages, Hkv, page, D) if heads_first else (n_pages, page, Hkv, D)
        self.page, self.heads_first, self.table = page, heads_first, table
        self.host = [[rng.integers(0, 2 ** 16, shape, dtype=np.uint16) for _ in range(2)] for _ in range(n_layers)]
        td = None if table is None else _put(table)
        self.caches = [paged.PagedCache(_put(k), _put(v), td, heads_first=heads_first) for k, v in self.host]

    def cell(self, x, page, at):
        return x[page, :, at] if self.heads_first else x[page, at]

    def check(self, want):
        for (k, v), c in zip(want, self.caches):
            assert np.array_equal(c.k.numpy(np.uint16), k) and np.array_equal(c.v.numpy(np.uint16), v)

    def moved(self, moves):
        """The host's layers after ((page, cell), (page, cell)) moves at once."""
        out = [[x.copy() for x in kv] for kv in self.host]
        for new, old in zip(out, self.host):
            for a, b in zip(new, old):
                for src, dst in moves:
                    self.cell(a, *dst)[...] = self.cell(b, *src)
        return out


def _tables(rng, lens, page, spare=1):
    need = [(n + page - 1) // page for n in lens]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(max(need), 1)), -5, np.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    return table, at + spare


def _path(rng, c, k, front):
    """k rising nodes of c from 0 on, the first ones next to one another."""
    rest = sorted(rng.choice(np.arange(1, c), k - 1, replace=False)) if k > 1 else []
    return ([0] + list(range(1, k)) if front else [0] + [int(x) for x in rest])[:k]


@pytest.mark.parametrize("layers, lens, counts, T, page, Hkv, heads_first", [
    (1, [1], None, 1, 16, 8, False), (3, [30, 9, 100], [9, 9, 1], 9, 8, 8, False), (2, [300, 33], None, 33, 24, 2, True),
    (66, [50, 20, 7], [20, 20, 0], 20, 16, 1, False), (2, [400, 300, 90], [200, 130, 65], 200, 256, 5, True), (1, [40] * 70, None, 26, 16, 4, False)])
def test_keep(gpu, layers, lens, counts, T, page, Hkv, heads_first):
    """Paths that begin in their places, whose cells overlap (a cell that is the
    place of a later entry), of all nodes, of none."""
    from arclight_amd import device, fattn, paged
    _case(f"keep {layers} layers {lens[:4]} of {T}")
    rng = np.random.default_rng(T + layers)
    counts = counts or [T] * len(lens)
    table, n_pages = _tables(rng, lens, page)
    L = Layers(rng, layers, n_pages, page, Hkv, heads_first, table)
    path, kept, moves = np.full((len(lens), T), MARK, np.int32), [], []
    for s, (n, c) in enumerate(zip(lens, counts)):
        k = 0 if c == 0 else int(rng.integers(1, c + 1)) if s else c
        p = _path(rng, c, k, s % 4 == 3) if k else []
        if s == 1 and k:
            p = [c - k + i for i in range(k)]                            # all from the end, overlapping
        path[s, :k] = p
        kept.append(k)
        place = lambda x: (table[s, x // page], x % page)  # noqa: E731
        moves += [(place(n - c + a), place(n - c + i)) for i, a in enumerate(p)]
    out = paged.keep(L.caches, _put(np.array(lens, np.int32)), _put(np.array(counts, np.int32)) if min(counts) < T else None, _put(path),
                     _put(np.array(kept, np.int32)))
    device.synchronize()
    fattn.device_errors()
    assert list(out.numpy(np.int32)) == [n - c + k for n, c, k in zip(lens, counts, kept)]
    L.check(L.moved(moves))


def test_keep_reports_what_it_cannot_move(gpu):
    """Wrong entries are left out, wrong sequences stay as they are; pages
    outside the pool."""
    from arclight_amd import device, fattn, paged
    from arclight_amd._lib import ArclightError
    _case("keep, wrong operands")
    rng = np.random.default_rng(2)
    page, T = 8, 6
    lens, counts, kept, path = [20, 30], [6, 6], [3, 3], [[0, 2, 5], [0, 3, 4]]
    table, n_pages = _tables(rng, lens, page)

    def run(lens=lens, counts=counts, kept=kept, path=path, table=table, left=(), none=(), text=""):
        L = Layers(rng, 2, n_pages, page, 2, False, table)
        p = np.full((2, T), MARK, np.int32)
        for s in range(2):
            p[s, :len(path[s])] = path[s]
        out = paged.keep(L.caches, *(_put(np.array(x, np.int32)) for x in (lens, counts)), _put(p), _put(np.array(kept, np.int32)))
        device.synchronize()
        if text:
            with pytest.raises(ArclightError, match=text):
                fattn.device_errors()
        fattn.device_errors()
        moves = []
        for s in range(2):
            for i, a in enumerate(path[s] if s not in none else []):
                src, dst = lens[s] - counts[s] + a, lens[s] - counts[s] + i
                if (s, i) not in left:
                    moves.append(((table[s, src // page], src % page), (table[s, dst // page], dst % page)))
        assert list(out.numpy(np.int32)) == [lens[s] if s in none else lens[s] - counts[s] + kept[s] for s in range(2)]
        L.check(L.moved(moves))

    run()
    run(path=[[0, 0, 5], [0, 3, 4]], left=[(0, 1)], text="kept")
    run(path=[[0, 6, 5], [0, 3, 4]], left=[(0, 1)], text="kept")
    run(path=[[-1, 2, 5], [0, 3, 2 ** 31 - 1]], left=[(0, 0), (1, 2)], text="kept")
    run(kept=[7, 3], none=[0], text="path of")
    run(kept=[-1, 3], none=[0], text="path of")
    run(counts=[7, 6], none=[0], text="new tokens")
    run(counts=[-1, 6], none=[0], text="new tokens")
    run(lens=[table.shape[1] * page + 1, 30], none=[0], text="length")
    run(lens=[-1, 30], none=[0], text="length")
    run(lens=[5, 30], none=[0], text="new tokens")
    wrong = table.copy()
    wrong[1, 27 // page] = n_pages                                       # of cells 24 to 29
    run(table=wrong, left=[(1, 0), (1, 1), (1, 2)], text="page")
    run(kept=[0, 0], path=[[], []])


@pytest.mark.parametrize("layers, n_pages, page, Hkv, heads_first", [(1, 3, 8, 1, False), (65, 9, 16, 2, True), (3, 30, 48, 8, False), (2, 9, 256, 5, True)])
@pytest.mark.parametrize("partly", [False, True])
def test_copy_pages(gpu, layers, n_pages, page, Hkv, heads_first, partly):
    """Some source pages twice, pairs that are left out, no cells, a page into itself."""
    from arclight_amd import device, fattn, paged
    _case(f"copy {layers} layers, pages of {page}, partly={partly}")
    rng = np.random.default_rng(page + layers)
    L = Layers(rng, layers, n_pages, page, Hkv, heads_first)
    order = rng.permutation(n_pages)
    n = max(1, n_pages // 3)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    src = np.concatenate([src, src[:1], [-1, order[0], order[-1]]])
    dst = np.concatenate([dst, order[2 * n:2 * n + 1], [order[-1], -4, order[-1]]])
    if n_pages == 3:
        src, dst = src[:2], dst[:2]
    cells = rng.integers(0, page + 1, len(src))
    cells[0], cells[-1] = page, 0
    paged.copy_pages(L.caches, _put(src.astype(np.int32)), _put(dst.astype(np.int32)), _put(cells.astype(np.int32)) if partly else None)
    device.synchronize()
    fattn.device_errors()
    L.check(L.moved([((a, c), (b, c)) for a, b, k in zip(src, dst, cells) if a >= 0 and b >= 0 for c in range(k if partly else page)]))


def test_copy_reports_what_it_cannot_copy(gpu):
    from arclight_amd import device, fattn, paged
    from arclight_amd._lib import ArclightError
    _case("copy, wrong operands")
    rng = np.random.default_rng(3)
    L = Layers(rng, 2, 4, 16, 2)
    for src, dst, cells, text in ((4, 1, 3, "page 4"), (0, 2 ** 31 - 1, 3, "page"), (0, 1, 17, "cells"), (0, 1, -1, "cells")):
        paged.copy_pages(L.caches, *(_put(np.array(x, np.int32)) for x in ([src], [dst], [cells])))
        device.synchronize()
        with pytest.raises(ArclightError, match=text):
            fattn.device_errors()
        L.check(L.host)


def test_pages_past_4_gb(gpu):
    """Pools whose pages lie 2.5 GB apart, for both calls."""
    from arclight_amd import device, fattn, paged
    _case("moves past 4 GB")
    rng = np.random.default_rng(4)
    page, Hkv, n_pages, apart = 16, 2, 3, 5 * 2 ** 29
    host = [rng.integers(0, 2 ** 16, (n_pages, page, Hkv, D), dtype=np.uint16) for _ in range(2)]
    pools = []
    for x in host:
        buf = device.DeviceBuffer(apart * (n_pages - 1) + page * Hkv * D * 2)
        for i in range(n_pages):
            buf.upload(x[i], apart * i)
        pools.append(device.DeviceTensor(buf, abi.AL_TYPE_F16, x.shape, (apart, Hkv * D * 2, D * 2, 2)))
    cache = paged.PagedCache(*pools, _put(np.array([[1, 2]], np.int32)))
    paged.keep([cache], _put(np.array([30], np.int32)), None, _put(np.array([[0, 20, 25] + [0] * 25], np.int32)), _put(np.array([3], np.int32)))
    paged.copy_pages([cache], _put(np.array([2], np.int32)), _put(np.array([0], np.int32)), _put(np.array([9], np.int32)))
    device.synchronize()
    fattn.device_errors()
    for x, t in zip(host, pools):
        want = x.copy()
        want[1, 3], want[1, 4] = x[2, 6], x[2, 11]                       # cells 22 and 27 to 3 and 4 of the sequence's
        want[0, :9] = x[2, :9]
        for i in range(n_pages):
            assert np.array_equal(t.buf.download(np.empty_like(x[i]), apart * i), want[i])
