"""Paged caches and the plain forms of the operators over them, in numpy and
64 bits, shared by the CPU and GPU tests."""
import math

import numpy as np

D = 128
EPS32 = 2.0 ** -24          # half a step of float32


class Pool:
    """Host copies of one layer's pools and tables: kv heads of 128, pages of
    P cells, for sequences of lens[s] cells; pages lie in a shuffled order,
    unused table entries name no page. Every cell that no sequence owns holds
    NaN in both pools."""

    def __init__(self, rng, lens, Hkv, P, heads_first=False, spare=2, max_pages=None):
        self.rng, self.lens, self.Hkv, self.P, self.heads_first = rng, list(lens), Hkv, P, heads_first
        need = [(max(n, 0) + P - 1) // P for n in lens]
        self.n_pages = sum(need) + spare
        self.max_pages = max_pages or max(max(need, default=1), 1)
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.max_pages), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        # as [page][cell][head][128], whatever the device's order
        self.k = np.full((self.n_pages, P, Hkv, D), np.nan, np.float16)
        self.v = np.full_like(self.k, np.nan)
        for s, n in enumerate(lens):
            for c in range(max(n, 0)):
                self.k[self.table[s, c // P], c % P] = rng.standard_normal((Hkv, D))
                self.v[self.table[s, c // P], c % P] = rng.standard_normal((Hkv, D))

    def cells(self, pool, s, n):
        """Cells 0 .. n - 1 of sequence s, (n, Hkv, 128) float64."""
        c = np.arange(n)
        return pool[self.table[s, c // self.P], c % self.P].astype(np.float64)

    def device(self):
        from arclight_amd import device, paged
        put = [np.ascontiguousarray(x.transpose(0, 2, 1, 3) if self.heads_first else x).view(np.uint16) for x in (self.k, self.v)]
        return paged.PagedCache(*(device.DeviceTensor.from_numpy(x) for x in put), device.DeviceTensor.from_numpy(self.table),
                                heads_first=self.heads_first)

    def download(self, cache):
        """The device pools as (page, cell, head, 128) float16."""
        out = [t.numpy(np.uint16).view(np.float16) for t in (cache.k, cache.v)]
        return [x.transpose(0, 2, 1, 3) if self.heads_first else x for x in out]


def attention(pool, q, lens, counts, scale, sinks=None, cap=0.0):
    """(out, bound): the operator's definition in float64 for q (n_seq, T, Hq,
    128), NaN where a row is left alone; bound: the error a float32
    implementation may have, derived as follows. A score is a sum of 128
    products of values that are carried to 2^-22 (two f16), added in two runs
    of 4 matrix products of 32 terms: at most 2 2^-22 + 40 2^-24 of the sum of
    the products' sizes, scaled by a rounded factor; the soft cap's tanh adds
    2^-21 of the cap. e^x of a difference of size d is off by the scores'
    errors and d 2^-23 + 2^-22; probabilities carried to 2^-22 and sums of n
    terms in chains of at most n / 32 + 64 add their shares; the same
    in the denominator."""
    n_seq, T, Hq, _ = q.shape
    G = Hq // pool.Hkv
    out = np.full(q.shape, np.nan)
    bound = np.zeros(q.shape)
    for s in range(n_seq):
        n = max(lens[s], 0)
        k, v = pool.cells(pool.k, s, n), pool.cells(pool.v, s, n)
        for t in range(min(counts[s], T)):
            sees = min(max(n - counts[s] + 1 + t, 0), n)
            for h in range(Hq):
                if sees == 0:
                    out[s, t, h] = 0.0
                    continue
                kk, vv = k[:sees, h // G], v[:sees, h // G]
                x = kk @ q[s, t, h].astype(np.float64) * scale
                dx = np.abs(kk) @ np.abs(q[s, t, h].astype(np.float64)) * abs(scale) * (2 * 2.0 ** -22 + 41 * EPS32)
                if cap:
                    x = cap * np.tanh(x / cap)
                    dx = dx + cap * 2.0 ** -21
                top = x.max() if sinks is None else max(x.max(), sinks[h])
                p = np.exp(x - top)
                total = p.sum() + (0.0 if sinks is None else math.exp(sinks[h] - top))
                out[s, t, h] = p @ vv / total
                dp = dx + dx.max() + (top - x) * 2.0 ** -23 + 2.0 ** -21 + (sees / 32 + 64) * EPS32
                bound[s, t, h] = (p * dp) @ np.abs(vv) / total + (p @ np.abs(vv)) / total * (p @ dp) / total + 1e-30
    return out, bound


def rope_angles(pos, base=1000000.0):
    """The float32 angles of (T,) positions, (T, 64) float64."""
    step = np.float32(np.float64(base) ** (-2.0 / D))
    th, out = np.asarray(pos, np.float32), []
    for _ in range(D // 2):
        out.append(th.astype(np.float64))
        th = (th * step).astype(np.float32)
    return np.stack(out, -1)


def norm_rotate(x, w, pos, eps, mode):
    """Rows (T, H, 128): normalised when eps is given, rotated ("neox",
    "normal" or None), in float64."""
    x = x.astype(np.float64)
    if eps is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            x = x * w.astype(np.float64)
    if mode is None:
        return x
    a = rope_angles(pos)[:, None]
    c, s = np.cos(a), np.sin(a)
    y = np.empty_like(x)
    lo, hi = (slice(0, 64), slice(64, 128)) if mode == "neox" else (slice(0, 128, 2), slice(1, 128, 2))
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., lo] * s + x[..., hi] * c
    return y
