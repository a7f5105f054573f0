"""Plain forms, in numpy and 64 bits, of what drafts and windows need over a
paged cache, shared by the CPU and GPU tests."""
import math

import numpy as np

from tests.paged_cases import D, EPS32


def visible(n, c, T, window=0, first=0, bits=None, pos=None):
    """(c, n) bool: the cells that each of the last c tokens of n cells sees;
    bits (T, words), pos (T,)."""
    b = n - c
    out = np.zeros((min(c, T), max(n, 0)), bool)
    for t in range(out.shape[0]):
        p = b + t if pos is None else int(pos[t])
        for x in range(max(n, 0)):
            if x < b:
                at, sees = x, True
            else:
                u = x - b
                at = x if pos is None else int(pos[u])
                sees = u <= t if bits is None else bool(int(bits[t, u // 32]) >> (u % 32) & 1)
            out[t, x] = sees and (not window or at > p - window or at < first)
    return out


def attention(pool, q, lens, counts, scale, sees, sinks=None, cap=0.0):
    """(out, bound) in float64 for q (n_seq, T, Hq, 128) and sees[s] (counts[s],
    lens[s]), NaN where a row is left alone. The bound is paged_cases.attention's:
    the masks are exact, and leave less to be rounded."""
    n_seq, T, Hq, _ = q.shape
    G = Hq // pool.Hkv
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s in range(n_seq):
        n = max(lens[s], 0)
        at = np.arange(n)
        page = np.clip(pool.table[s, at // pool.P], 0, pool.n_pages - 1)
        k, v = (x[page, at % pool.P].astype(np.float64) for x in (pool.k, pool.v))
        for t in range(min(counts[s], T)):
            m = sees[s][t]
            for h in range(Hq):
                if not m.any():
                    out[s, t, h] = 0.0
                    continue
                kk, vv = k[m, h // G], v[m, h // G]
                x = kk @ q[s, t, h].astype(np.float64) * scale
                dx = np.abs(kk) @ np.abs(q[s, t, h].astype(np.float64)) * abs(scale) * (2 * 2.0 ** -22 + 41 * EPS32)
                if cap:
                    x = cap * np.tanh(x / cap)
                    dx = dx + cap * 2.0 ** -21
                top = x.max() if sinks is None else max(x.max(), sinks[h])
                p = np.exp(x - top)
                total = p.sum() + (0.0 if sinks is None else math.exp(sinks[h] - top))
                out[s, t, h] = p @ vv / total
                dp = dx + dx.max() + (top - x) * 2.0 ** -23 + 2.0 ** -21 + (m.sum() / 32 + 64) * EPS32
                bound[s, t, h] = (p * dp) @ np.abs(vv) / total + (p @ np.abs(vv)) / total * (p @ dp) / total + 1e-30
    return out, bound


def random_tree(rng, T, bushy=0.5):
    """Parents of T nodes, those of node t below t."""
    return np.array([-1] + [t - 1 if rng.random() > bushy else int(rng.integers(0, t)) for t in range(1, T)], np.int32)[:T]


def tree(parents, n, c, words=None):
    """pos, cells, seq (0 or -1), bits of one sequence's T nodes, c of them there."""
    T = len(parents)
    words = words or max(1, (T + 31) // 32)
    pos, cells, seq, bits = np.zeros(T, np.int32), np.zeros(T, np.int32), np.full(T, -1, np.int32), np.zeros((T, words), np.uint32)
    for t in range(c):
        u, depth = t, -1
        while u >= 0:
            bits[t, u // 32] |= np.uint32(1 << (u % 32))
            u, depth = (int(parents[u]) if parents[u] < u else -1), depth + 1
        pos[t], cells[t], seq[t] = n - c + depth, n - c + t, 0
    return pos, cells, seq, bits.view(np.int32)


def verify(target, tokens, accept, sample, parents=None, count=None, draft=None):
    """path, next of one sequence, by the definition."""
    T, V = target.shape
    count = T if count is None else count
    if not 0 <= count <= T or count == 0:
        return [], -1
    parents = np.arange(-1, T - 1) if parents is None else parents
    clean = lambda x: np.where(x > 0, x, 0).astype(np.float64)  # noqa: E731
    v, path = 0, [0]
    while True:
        own = clean(target[v])
        p, left, mass, found = own.copy(), own.copy(), 1.0, -1
        for u in range(v + 1, count):
            x = int(tokens[u])
            if parents[u] != v or not 0 <= x < V:
                continue
            # without a draft p is not normalised: r < p / mass
            q = mass if draft is None else float(clean(draft[v])[x])
            if p[x] > 0 and float(accept[u]) * q < p[x]:
                found = u
                break
            if draft is None:
                mass -= p[x]
                p[x] = left[x] = 0.0
            else:
                left = np.maximum(p - clean(draft[v]), 0)
                total = left.sum()
                p = left / total if 0 < total < np.inf else np.zeros(V)
        if found < 0:
            break
        v = found
        path.append(v)
    w = left if left.sum() > 0 else own
    run = w.cumsum()
    if not 0 < run[-1] < np.inf:
        return path, -1
    past = np.flatnonzero((run > float(sample) * run[-1]) & (w > 0))
    return path, int(past[0]) if len(past) else int(np.flatnonzero(w > 0)[-1])
