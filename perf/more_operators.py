"""The operators of a server that drafts, as cases to be timed: layers that
see a window of the paged cache and its first cells, trees of drafted tokens
over the cache, their verification, and the cells that stay.

  window   attention of each sequence's new tokens to the last `window` cells
           and the `first` ones
  tree     attention of a tree of drafted tokens to all cells before it and
           to their own ancestors in it
  nodes    from the trees' parents: position, cell and sequence of each
           node's row, and the bits of the nodes that it sees
  verify   the accepted path of each tree and the token after it, from the
           target's probabilities and given random numbers
  move     cells moved in all layers: those of the accepted path to the places
           that follow the sequence's cells, or, for forks, those of pages into
           other pages

A case is a dict of plain values:
  op         which of the above
window, tree:
  heads, kv  query heads and KV heads, of 128
  page       cells of a page; order "cells": a page is [cell][head][128],
             "heads": [head][cell][128]
  seqs, ctx  sequences; cells that the longest holds before the pass (the
             others 1/3 to all of it)
  tokens     most new tokens of a sequence (tree: nodes)
  ragged     sequences bring 1 to `tokens` of them (tree: half to all)
  sinks      a sink logit for each head
window:
  window, first
nodes:
  seqs, tokens, ragged
verify:
  seqs, tokens, vocab
  drafted    a chain of tokens drawn from a draft's probabilities, which are
             given; else a tree of tokens chosen from likely ones
move:
  kv, page, order, layers
  how        "keep" (of seqs, ctx, tokens) or "copy" (of pairs)
"""
import math

import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _window(name, seqs, ctx, window, first, tokens=1, heads=32, kv=8, page=16, order="cells", ragged=False, sinks=False):
    return {"name": name, "op": "window", "heads": heads, "kv": kv, "page": page, "order": order, "seqs": seqs, "ctx": ctx,
            "tokens": tokens, "ragged": ragged, "sinks": sinks, "window": window, "first": first}


def _tree(name, seqs, ctx, tokens, heads=32, kv=8, page=16, order="cells", ragged=False, sinks=False):
    return {"name": name, "op": "tree", "heads": heads, "kv": kv, "page": page, "order": order, "seqs": seqs, "ctx": ctx,
            "tokens": tokens, "ragged": ragged, "sinks": sinks}


def _nodes(name, seqs, tokens, ragged=False):
    return {"name": name, "op": "nodes", "seqs": seqs, "tokens": tokens, "ragged": ragged}


def _verify(name, seqs, tokens, vocab, drafted=False):
    return {"name": name, "op": "verify", "seqs": seqs, "tokens": tokens, "vocab": vocab, "drafted": drafted}


def _keep(name, seqs, ctx, tokens, layers, kv=8, page=16, order="cells"):
    return {"name": name, "op": "move", "how": "keep", "kv": kv, "page": page, "order": order, "layers": layers, "seqs": seqs, "ctx": ctx,
            "tokens": tokens}


def _copy(name, pairs, layers, kv=8, page=16, order="cells"):
    return {"name": name, "op": "move", "how": "copy", "kv": kv, "page": page, "order": order, "layers": layers, "pairs": pairs}


def listed():
    return [
        # one user's decode step in a layer with a window: latency
        _window("window-1-3000", 1, 3000, 1024, 4),
        # a server's decode step, long conversations, larger pages and sinks
        _window("window-30-20000", 30, 20000, 4096, 0, page=64, order="heads", sinks=True),
        # two prompts of a few thousand tokens: matrix products
        _window("window-prompts-2", 2, 500, 1000, 64, tokens=4000),
        # one user's tree of 26 nodes: latency
        _tree("tree-1-2000", 1, 2000, 26),
        # a small server's trees of up to 61 nodes, a larger model
        _tree("tree-11-6000", 11, 6000, 61, heads=64, page=32, ragged=True),
        # the tree's tables, once a step: one user's, a server's
        _nodes("nodes-1-26", 1, 26),
        _nodes("nodes-50-200", 50, 200, ragged=True),
        # one user's tree: latency
        _verify("verify-tree-1", 1, 26, 32003),
        # a server's chains of 6 drafts with the draft's probabilities
        _verify("verify-chain-30", 30, 7, 128000, drafted=True),
        # a server's trees
        _verify("verify-tree-20", 20, 40, 152000),
        # a server's accepted paths, 36 layers
        _keep("keep-40", 40, 600, 33, 36),
        # twenty forks of running requests, 64 layers
        _copy("copy-20", 20, 64, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# bytes and operations of a drawn case: the largest listed's
_MOST = {"window": (5.0e8, 1.3e11), "tree": (2.1e8, 6.5e10), "nodes": (4.4e5, 1e9), "verify": (3.0e7, 1e9), "keep": (2.9e7, 1e9),
         "copy": (3.1e8, 1e9)}


def draw(rng):
    op = rng.choice(["window", "window", "window", "tree", "tree", "nodes", "verify", "verify", "keep", "copy"])
    heads, kv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (8, 8)])
    page, order = rng.choice([16, 16, 32, 48, 64, 256]), rng.choice(["cells", "cells", "heads"])
    if op == "window":
        tokens = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 4000)])
        c = _window("", _log(rng, 1, 100), _log(rng, 1, 30000), _log(rng, 16, 8000), rng.choice([0, 4, 4, _log(rng, 1, 500)]),
                    tokens, heads, kv, page, order, ragged=rng.random() < 0.5, sinks=rng.random() < 0.3)
    elif op == "tree":
        c = _tree("", _log(rng, 1, 60), _log(rng, 1, 20000), _log(rng, 2, 128), heads, kv, page, order, ragged=rng.random() < 0.5,
                  sinks=rng.random() < 0.3)
    elif op == "nodes":
        c = _nodes("", _log(rng, 1, 100), _log(rng, 1, 500), ragged=rng.random() < 0.5)
    elif op == "verify":
        c = _verify("", _log(rng, 1, 48), _log(rng, 2, 64), rng.choice([32000, 32003, 50257, 128000, _log(rng, 1000, 160000)]),
                    drafted=rng.random() < 0.4)
    elif op == "keep":
        c = _keep("", _log(rng, 1, 64), _log(rng, 1, 1000), _log(rng, 2, 64), rng.choice([1, 28, 36, 64]), kv, page, order)
    else:
        c = _copy("", _log(rng, 1, 64), rng.choice([1, 28, 36, 64]), kv, page, order)
    while True:
        w = work(c)
        if w["bytes"] <= _MOST[op][0] and w["flops"] <= _MOST[op][1] and _held(c) <= 1.2e9:
            break
        for k, least in (("seqs", 1), ("ctx", 0), ("pairs", 1), ("tokens", 2), ("layers", 1)):
            if k in c and c[k] > least and (k != "tokens" or c[k] > 8):
                c[k] = max(least, c[k] * 4 // 5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# sizes: what a case's sequences and tokens are
# ---------------------------------------------------------------------------

def _counts(case):
    """New tokens of each sequence."""
    n, t = case["seqs"], case["tokens"]
    if not case.get("ragged"):
        return [t] * n
    least = (t + 1) // 2 if case["op"] in ("tree", "nodes") else 1
    return [least + (5 * s + 3) % (t - least + 1) for s in range(n)]


def _lengths(case):
    """Cells of each sequence, its new tokens among them."""
    n, ctx = case["seqs"], case["ctx"]
    old = [ctx] if n == 1 else [ctx * (n + 2 * ((7 * s) % n)) // (3 * n - 2) for s in range(n)]
    return [o + c for o, c in zip(old, _counts(case))]


def _parents(case, s):
    """The tree of sequence s, level by level: nodes have 4, 3, 2, 1, 3, ...
    children, those near the root first; case["drafted"]: a chain."""
    t = case["tokens"]
    if case.get("drafted"):
        return list(range(-1, t - 1))
    out, v = [-1], 0
    while len(out) < t:
        out += [v] * min((4, 3, 2, 1, 3)[(v + s) % 5], t - len(out))
        v += 1
    return out


def _kept(case):
    """Nodes of each accepted path to be kept, the root among them: half of
    the tree's at most."""
    return [1 + (3 * s + 1) % min(6, max(1, case["tokens"] // 2)) for s in range(case["seqs"])]


def _stay(i, kept):
    """Nodes of sequence i's path that are in their places already."""
    return 1 if i % 3 else min(kept, 2)


def _filled(case):
    """Cells that each pair of a copy case copies."""
    return [1 + (11 * i + 5) % case["page"] for i in range(case["pairs"])]


def _pairs(case):
    """Pairs of a token and a cell that it sees."""
    def ramp(m, most):                          # sum of min(x, most) for x of 1 to m
        m, over = max(m, 0), max(m - most, 0)
        return m * (m + 1) // 2 - over * (over + 1) // 2

    total = 0
    for i, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        if case["op"] == "tree":
            depth = []
            for p in _parents(case, i)[:c]:
                depth.append(depth[p] + 1 if p >= 0 else 1)
            total += c * (n - c) + sum(depth)
        else:
            w, f = case["window"], case["first"]
            total += ramp(n, w) - ramp(n - c, w) + ramp(n - w, f) - ramp(n - c - w, f)
    return total


def _visible(case):
    """Cells of each sequence that some token sees."""
    if case["op"] == "tree":
        return _lengths(case)
    w, f = case["window"], case["first"]
    return [n - max(0, n - c + 1 - w - f) for n, c in zip(_lengths(case), _counts(case))]


def _held(case):
    """Bytes of the state that are not work."""
    if case["op"] == "verify":
        return case["seqs"] * case["tokens"] * case["vocab"] * (8 if case["drafted"] else 4)
    if case.get("how") == "keep":
        return (case["ctx"] + case["seqs"] * (case["tokens"] + 2 * case["page"])) * case["kv"] * 512 * case["layers"]
    return 0


def work(case):
    """window, tree: the cells that a sequence's tokens see, once, the queries
    and the outputs; the products of the visible pairs. nodes: a parent read, a
    position, a cell, a sequence and the bits written for each. verify: one row
    of probabilities a sequence (a row of the draft's beside it). move: each
    cell that moves, read and written."""
    op = case.get("how", case["op"])
    if op in ("window", "tree"):
        h, tokens = case["heads"], sum(_counts(case))
        return {"bytes": sum(_visible(case)) * case["kv"] * D * 4 + tokens * h * D * 8, "flops": 4 * D * h * _pairs(case)}
    if op == "nodes":
        t = case["tokens"]
        return {"bytes": case["seqs"] * t * (16 + 4 * ((t + 31) // 32)), "flops": case["seqs"] * t}
    if op == "verify":
        rows = 2 if case["drafted"] else 1
        return {"bytes": case["seqs"] * (rows * 4 * case["vocab"] + 16 * case["tokens"]), "flops": case["seqs"] * case["vocab"] * rows}
    if op == "keep":
        return {"bytes": sum(k - _stay(i, k) for i, k in enumerate(_kept(case))) * case["kv"] * D * 8 * case["layers"] + case["seqs"] * 8, "flops": 0}
    return {"bytes": sum(_filled(case)) * case["kv"] * D * 8 * case["layers"], "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _State:
    pass


def _pool(case, n_pages):
    heads = case["order"] == "heads"
    return (n_pages, case["kv"], case["page"], D) if heads else (n_pages, case["page"], case["kv"], D)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(s, case, g):
    """The sequences' lengths and page tables: pages in no order, none for
    cells that nothing sees any more (a window's server has freed them)."""
    page, lens, counts = case["page"], _lengths(case), _counts(case)
    s.max_pages = (max(lens) + page - 1) // page
    at, where = 0, torch.full((case["seqs"], s.max_pages), -1, dtype=torch.int64)
    for i, (n, c) in enumerate(zip(lens, counts)):
        have = torch.arange((n + page - 1) // page)
        if case["op"] == "window":
            from_page = max(0, n - c + 1 - case["window"]) // page
            have = have[(have >= from_page) | (have * page < case["first"])]
        where[i, have] = torch.arange(at, at + len(have))
        at += len(have)
    s.n_pages = at + 2
    order = torch.randperm(s.n_pages, device="cuda", generator=g).int()
    where = where.cuda()
    s.table = torch.where(where >= 0, order[where.clamp(min=0)], torch.full_like(where, -1).int())
    s.lens, s.counts = _ints(lens), _ints(counts)


def _bits(case):
    """(seqs, tokens, words): node u's bit in the words of node t where u is t
    or an ancestor of it."""
    t = case["tokens"]
    words = torch.zeros((case["seqs"], t, (t + 31) // 32), dtype=torch.int64)
    for i, c in enumerate(_counts(case)):
        for u, p in enumerate(_parents(case, i)[:c]):
            if p >= 0:
                words[i, u] = words[i, p]
            words[i, u, u // 32] |= 1 << (u % 32)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int().cuda()


def prepare(case, seed):
    s = _State()
    s.case, s.call = case, None
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, dtype=dtype, device="cuda", generator=g)

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    op = case.get("how", case["op"])
    if op in ("window", "tree"):
        _tables(s, case, g)
        n, t, h = case["seqs"], case["tokens"], case["heads"]
        # a spread of the scores of about 2.5
        s.q = randn(n, t, h, D) * 2.5
        s.kc, s.vc = (randn(*_pool(case, s.n_pages), dtype=torch.float16) for _ in range(2))
        s.sinks = randn(h) * 2 + 4 if case["sinks"] else None
        s.bits = _bits(case) if op == "tree" else None
        s.out = torch.zeros((n, t, h, D), device="cuda")
    elif op == "nodes":
        n, t = case["seqs"], case["tokens"]
        turn = torch.randint(0, 1000, (1,), device="cuda", generator=g).item()
        s.parents = _ints([_parents(case, i + turn) for i in range(n)])
        s.counts = _ints(_counts(case))
        s.lens = s.counts + torch.randint(0, 5000, (n,), device="cuda", generator=g).int()
        s.pos, s.cells, s.seq = (torch.zeros((n, t), dtype=torch.int32, device="cuda") for _ in range(3))
        s.bits = torch.zeros((n, t, (t + 31) // 32), dtype=torch.int32, device="cuda")
    elif op == "verify":
        n, t, V = case["seqs"], case["tokens"], case["vocab"]
        # a few likely tokens in each row and a long tail
        likely = torch.randint(0, V, (n, t, 8), device="cuda", generator=g)
        logits = randn(n, t, V) * 1.5
        logits.scatter_(2, likely, math.log(V) + 2 - 0.8 * torch.arange(8.0, device="cuda") + randn(n, t, 8))
        s.target = torch.softmax(logits, -1)
        s.parents = _ints([_parents(case, i) for i in range(n)])
        up = s.parents.long().clamp(min=0)
        if case["drafted"]:
            logits = logits + 0.6 * randn(n, t, V)
            s.draft = torch.softmax(logits, -1)
            drawn = torch.argmax(logits - torch.log(-torch.log(rand(n, t, V).clamp(1e-9, 1 - 1e-7))), -1)
            tokens = drawn.gather(1, up)
        else:
            # a node's children: its likely tokens in turn
            s.draft = None
            at = torch.arange(t, device="cuda")
            rank = ((up[:, :, None] == up[:, None, :]) & (at[None, :] < at[:, None])).sum(-1).clamp(max=7)
            tokens = likely.gather(1, up[:, :, None].expand(-1, -1, 8)).gather(2, rank[:, :, None])[..., 0]
        s.tokens, s.counts = tokens.int().contiguous(), _ints([t] * n)
        s.accept, s.sample = rand(n, t), rand(n)
        s.path = torch.zeros((n, t), dtype=torch.int32, device="cuda")
        s.kept, s.next = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    elif op == "keep":
        # the sequences share the pages of a common beginning
        page, n, t, ctx = case["page"], case["seqs"], case["tokens"], case["ctx"]
        shared = ctx // page
        old = [shared * page + (7 * i) % page for i in range(n)]
        own_pages = (page - 1 + t + page - 1) // page
        s.n_pages = shared + n * own_pages
        order = torch.randperm(s.n_pages, device="cuda", generator=g).int()
        s.table = torch.cat([order[:shared].expand(n, -1), order[shared:].view(n, own_pages)], 1).contiguous()
        s.lens, s.counts = _ints([o + t for o in old]), _ints([t] * n)
        path, kept = torch.full((n, t), -1, dtype=torch.int32), _kept(case)
        for i, k in enumerate(kept):
            # nodes behind the kept ones' places, but for the first that stay
            stay, room = _stay(i, k), t - k
            for j in range(k):
                path[i, j] = j if j < stay else k + (j - stay) * room // k + i % (room // k)
        s.path, s.kept = path.cuda(), _ints(kept)
        s.kc, s.vc = (randn(case["layers"], *_pool(case, s.n_pages), dtype=torch.float16) for _ in range(2))
        s.lens_out = torch.zeros_like(s.lens)
    else:
        n = case["pairs"]
        s.n_pages = 2 * n + 3
        order = torch.randperm(s.n_pages, device="cuda", generator=g).int()
        s.src, s.dst, s.filled = order[:n].contiguous(), order[n:2 * n].contiguous(), _ints(_filled(case))
        s.kc, s.vc = (randn(case["layers"], *_pool(case, s.n_pages), dtype=torch.float16) for _ in range(2))
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _plain_attn(s, case):
    n, t, h, hk, page = case["seqs"], case["tokens"], case["heads"], case["kv"], case["page"]
    at = torch.arange(t, device="cuda")
    begin = (s.lens - s.counts).long()                                # cells before the new ones
    L = s.max_pages * page
    if case["op"] == "window":
        w, f = case["window"], case["first"]
        # the first cells, then those from the first token's window on
        span = min(L, w + t - 1)
        low = (begin + 1 - w).clamp(min=0)[:, None]
        cell = torch.cat([torch.arange(f, device="cuda").expand(n, -1), low + torch.arange(span, device="cuda")], 1)
        again = (torch.arange(f + span, device="cuda") < f) & (cell >= low)
        p = (begin[:, None] + at)[..., None]
        x = cell[:, None]
        seen = (x <= p) & ((x > p - w) | (x < f)) & ~again[:, None]
    else:
        cell = torch.arange(L, device="cuda").expand(n, -1)
        node = (cell - begin[:, None]).clamp(0, t - 1)
        word = s.bits.long().gather(2, (node // 32)[:, None].expand(-1, t, -1))
        seen = (cell < begin[:, None])[:, None] | (((word >> (node % 32)[:, None]) & 1 == 1) &
                                                  ((cell >= begin[:, None]) & (cell < s.lens[:, None]))[:, None])
    m = cell.shape[1]
    place = cell.clamp(max=L - 1)
    pages = s.table.long().gather(1, place // page).clamp(min=0)

    def cells(pool):                            # (n, hk, m, D)
        x = pool[pages, :, place % page] if case["order"] == "heads" else pool[pages, place % page]
        return x.float().permute(0, 2, 1, 3).contiguous()

    q = s.q.view(n, t, hk, h // hk, D).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, D)
    score = torch.matmul(q, cells(s.kc).transpose(2, 3)) * SCALE
    score = score.view(n, hk, t, h // hk, m).masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if case["sinks"]:
        sink = s.sinks.view(1, hk, 1, h // hk, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    o = torch.matmul(p.view(n, hk, -1, m), cells(s.vc)).view(n, hk, t, h // hk, D)
    o = (o / torch.where(total > 0, total, torch.ones_like(total))).permute(0, 2, 1, 3, 4).reshape(n, t, h, D)
    return {"out": torch.where((at < s.counts[:, None])[..., None, None], o, s.out)}


def _ancestors(parents):
    """(n, t, t): u is t or an ancestor of it."""
    t = parents.shape[1]
    at = torch.arange(t, device="cuda")
    up = ((parents[:, :, None] == at) | (at[:, None] == at)).float()
    for _ in range(max(1, (t - 1).bit_length())):
        up = (torch.matmul(up, up) > 0).float()
    return up > 0


def _plain_nodes(s, case):
    n, t = case["seqs"], case["tokens"]
    at = torch.arange(t, device="cuda")
    real = at < s.counts[:, None]
    up = _ancestors(s.parents) & real[:, :, None]
    begin = (s.lens - s.counts)[:, None]
    zero = torch.zeros((n, t), dtype=torch.int32, device="cuda")
    w = (t + 31) // 32
    full = torch.cat([up, up.new_zeros((n, t, w * 32 - t))], 2).view(n, t, w, 32).long()
    word = (full << torch.arange(32, device="cuda")).sum(-1)
    return {"pos": torch.where(real, (begin + up.sum(-1) - 1).int(), zero),
            "cells": torch.where(real, (begin + at).int(), zero),
            "seq": torch.where(real, torch.arange(n, device="cuda", dtype=torch.int32)[:, None], zero - 1),
            "bits": torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()}


def _plain_verify(s, case):
    n, t, V = case["seqs"], case["tokens"], case["vocab"]
    at = torch.arange(t, device="cuda")
    up, tok = s.parents.long().clamp(min=0), s.tokens.long()
    child = s.parents >= 0
    row = torch.arange(n, device="cuda")[:, None]
    p, r = s.target[row, up, tok].double(), s.accept.double()
    before = (s.parents[:, :, None] == s.parents[:, None]) & (at < at[:, None])      # earlier children of the same node
    if s.draft is None:
        # what the children that were rejected before this one leave
        left = 1 - (before * p[:, None]).sum(-1)
        twice = (before & (tok[:, :, None] == tok[:, None])).any(-1)
        passes = child & ~twice & (p > 0) & (r * left < p)
    else:
        passes = child & (r * s.draft[row, up, tok].double() < p)
    chosen = (passes & ~(before & passes[:, None]).any(-1)) | (at == 0)
    on = (~_ancestors(s.parents) | chosen[:, None]).all(-1)                             # the node and all above it
    kept = on.sum(-1)
    last = torch.where(on, at, -1).amax(-1)
    w = s.target[row[:, 0], last].double()
    under = child & (s.parents == last[:, None])
    if s.draft is None:
        gone = torch.zeros((n, V), device="cuda").scatter_add_(1, tok, under.float())
        left = torch.where(gone > 0, torch.zeros_like(w), w)
    else:
        left = torch.where(under.any(-1)[:, None], w - s.draft[row[:, 0], last].double(), w).clamp(min=0)
    w = torch.where((left.sum(-1) > 0)[:, None], left, w)
    run = w.cumsum(-1)
    nxt = (run <= (s.sample.double() * run[:, -1])[:, None]).sum(-1).clamp(max=V - 1)
    order = torch.where(on, at, t).sort(-1).values
    return {"path": torch.where(order < t, order, -1).int(), "kept": kept.int(), "next": nxt.int()}


def _plain_keep(s, case):
    n, t, page = case["seqs"], case["tokens"], case["page"]
    begin = (s.lens - s.counts).long()[:, None]
    to = torch.arange(t, device="cuda").expand(n, -1)
    mine = to < s.kept[:, None]
    src, dst = (begin + s.path.clamp(min=0))[mine], (begin + to)[mine]
    i = torch.arange(n, device="cuda")[:, None].expand(-1, t)[mine]
    sp, dp = s.table[i, src // page].long(), s.table[i, dst // page].long()
    for x in (s.kc, s.vc):
        if case["order"] == "heads":
            x[:, dp, :, dst % page] = x[:, sp, :, src % page]
        else:
            x[:, dp, dst % page] = x[:, sp, src % page]
    return {"k": s.kc, "v": s.vc, "lens": s.lens - s.counts + s.kept}


def _plain_copy(s, case):
    mine = torch.arange(case["page"], device="cuda") < s.filled[:, None]
    mine = mine[:, None, :, None] if case["order"] == "heads" else mine[:, :, None, None]
    src, dst = s.src.long(), s.dst.long()
    for x in (s.kc, s.vc):
        x[:, dst] = torch.where(mine, x[:, src], x[:, dst])
    return {"k": s.kc, "v": s.vc}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

class _Memory:
    """Device memory of a torch tensor, as the buffer of a DeviceTensor."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _dev(t):
    from arclight_amd import abi, device
    types = {torch.float32: abi.AL_TYPE_F32, torch.float16: abi.AL_TYPE_F16, torch.int32: abi.AL_TYPE_I32}
    return device.DeviceTensor(_Memory(t), types[t.dtype], tuple(t.shape))


def _bind(s, case):
    """The pass's call with its argument structure, filled in once, as a
    program holds it."""
    from arclight_amd import draft, paged
    op, heads_first = case.get("how", case["op"]), case.get("order") == "heads"
    if op in ("window", "tree"):
        cache = paged.PagedCache(_dev(s.kc), _dev(s.vc), _dev(s.table), heads_first=heads_first)
        sees = {"window": case["window"], "first": case["first"]} if op == "window" else {"bits": _dev(s.bits)}
        return paged.AttentionCall(cache, _dev(s.q), _dev(s.lens), _dev(s.out), counts=_dev(s.counts),
                                   sinks=None if s.sinks is None else _dev(s.sinks), scale=SCALE, **sees)
    if op == "nodes":
        return draft.TreeCall(_dev(s.parents), _dev(s.lens), _dev(s.counts), _dev(s.pos), _dev(s.cells), _dev(s.seq), _dev(s.bits))
    if op == "verify":
        return draft.VerifyCall(_dev(s.target), _dev(s.tokens), _dev(s.accept), _dev(s.sample), _dev(s.path), _dev(s.kept),
                                _dev(s.next), parents=None if case["drafted"] else _dev(s.parents), counts=_dev(s.counts),
                                draft=None if s.draft is None else _dev(s.draft))
    layers = [paged.PagedCache(_dev(k), _dev(v), _dev(s.table) if op == "keep" else None, heads_first=heads_first)
              for k, v in zip(s.kc, s.vc)]
    if op == "keep":
        return paged.KeepCall(layers, _dev(s.lens), _dev(s.counts), _dev(s.path), _dev(s.kept), _dev(s.lens_out))
    return paged.CopyCall(layers, _dev(s.src), _dev(s.dst), _dev(s.filled))


def run(s):
    case = s.case
    op = case.get("how", case["op"])
    if not own:
        return {"nodes": _plain_nodes, "verify": _plain_verify, "keep": _plain_keep, "copy": _plain_copy}.get(op, _plain_attn)(s, case)
    if s.call is None:
        s.call = _bind(s, case)
    s.call.run()
    if op in ("window", "tree"):
        return {"out": s.out}
    if op == "nodes":
        return {"pos": s.pos, "cells": s.cells, "seq": s.seq, "bits": s.bits}
    if op == "verify":
        return {"path": s.path, "kept": s.kept, "next": s.next}
    return {"k": s.kc, "v": s.vc, "lens": s.lens_out} if op == "keep" else {"k": s.kc, "v": s.vc}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_attn(s, case):
    n, t, h, hk, page = case["seqs"], case["tokens"], case["heads"], case["kv"], case["page"]
    G = h // hk
    out = torch.zeros((n, t, h, D), dtype=torch.float64, device="cuda")
    for i, (c, m) in enumerate(zip(_counts(case), _lengths(case))):
        old = m - c
        if case["op"] == "tree":
            mine = torch.arange(m)
            hidden = torch.ones((c, m), dtype=torch.bool)
            hidden[:, :old] = False
            up = _parents(case, i)
            for u in range(c):
                v = u
                while v >= 0:
                    hidden[u, old + v] = False
                    v = up[v]
            hidden = hidden.cuda()
        else:
            mine = torch.tensor([x for x in range(m) if x < case["first"] or x > old - case["window"]])
            p, x = torch.arange(old, m, device="cuda")[:, None], mine.cuda()[None]
            hidden = (x > p) | ((x + case["window"] <= p) & (x >= case["first"]))
        mine = mine.cuda()
        pages, at = s.table[i].long()[mine // page], mine % page
        for j in range(hk):
            k, v = ((x[pages, j, at] if case["order"] == "heads" else x[pages, at, j]).double() for x in (s.kc, s.vc))
            for c0 in range(0, c, 512):
                q = s.q[i, c0:min(c, c0 + 512), j * G:(j + 1) * G].double()
                x = (q.reshape(-1, D) @ k.T / math.sqrt(D)).view(q.shape[0], G, -1)
                x.masked_fill_(hidden[c0:c0 + 512, None], -math.inf)
                if case["sinks"]:
                    x = torch.cat([x, s.sinks[j * G:(j + 1) * G].double()[None, :, None].expand(x.shape[0], -1, 1)], -1)
                a = torch.softmax(x, -1)[..., :len(mine)]
                out[i, c0:c0 + q.shape[0], j * G:(j + 1) * G] = (a.reshape(-1, len(mine)) @ v).view(q.shape[0], G, D)
    return {"out": out}


def _exact_nodes(s, case):
    n, t = case["seqs"], case["tokens"]
    pos, cells, seq = [[0] * t for _ in range(n)], [[0] * t for _ in range(n)], [[-1] * t for _ in range(n)]
    bits = [[[0] * ((t + 31) // 32) for _ in range(t)] for _ in range(n)]
    parents, lens = s.parents.tolist(), s.lens.tolist()
    for i, c in enumerate(_counts(case)):
        for u in range(c):
            v, depth = u, -1
            while v >= 0:
                bits[i][u][v // 32] |= 1 << (v % 32)
                v, depth = parents[i][v], depth + 1
            pos[i][u], cells[i][u], seq[i][u] = lens[i] - c + depth, lens[i] - c + u, i
        bits[i] = [[w - 2 ** 32 if w >= 2 ** 31 else w for w in node] for node in bits[i]]
    return {"pos": _ints(pos), "cells": _ints(cells), "seq": _ints(seq), "bits": _ints(bits)}


def _exact_verify(s, case):
    n, t = case["seqs"], case["tokens"]
    parents, tokens, accept, sample = s.parents.tolist(), s.tokens.tolist(), s.accept.tolist(), s.sample.tolist()
    paths, kept, nxt = [], [], []
    for i in range(n):
        v, path = 0, [0]
        while True:
            # p: what is left of v's probabilities, mass: its sum, as given
            p, mass, found = s.target[i, v].double(), 1.0, -1
            for u in [u for u in range(t) if parents[i][u] == v]:
                x = tokens[i][u]
                px = float(p[x])
                if px > 0 and accept[i][u] * (mass if s.draft is None else float(s.draft[i, v, x])) < px:
                    found = u
                    break
                if s.draft is None:
                    mass -= px
                    p[x] = 0
                else:
                    p = (p - s.draft[i, v].double()).clamp(min=0)
                    p /= p.sum()
            if found < 0:
                break
            v = found
            path.append(v)
        total = p.cumsum(0)
        nxt.append(int((total > sample[i] * total[-1]).nonzero()[0]))
        kept.append(len(path))
        paths.append(path + [-1] * (t - len(path)))
    return {"path": _ints(paths), "kept": _ints(kept), "next": _ints(nxt)}


def _exact_keep(s, case):
    k, v = s.kc.clone(), s.vc.clone()
    page, table, path = case["page"], s.table.tolist(), s.path.tolist()
    lens = []
    for i, (m, c, kept) in enumerate(zip(s.lens.tolist(), s.counts.tolist(), _kept(case))):
        lens.append(m - c + kept)
        for j in range(kept):
            src, dst = m - c + path[i][j], m - c + j
            a, b = (table[i][src // page], src % page), (table[i][dst // page], dst % page)
            for new, old in ((k, s.kc), (v, s.vc)):
                if case["order"] == "heads":
                    new[:, b[0], :, b[1]] = old[:, a[0], :, a[1]]
                else:
                    new[:, b[0], b[1]] = old[:, a[0], a[1]]
    return {"k": k, "v": v, "lens": _ints(lens)}


def _exact_copy(s, case):
    k, v = s.kc.clone(), s.vc.clone()
    for a, b, m in zip(s.src.tolist(), s.dst.tolist(), s.filled.tolist()):
        for x in (k, v):
            if case["order"] == "heads":
                x[:, b, :, :m] = x[:, a, :, :m]
            else:
                x[:, b, :m] = x[:, a, :m]
    return {"k": k, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    return {"nodes": _exact_nodes, "verify": _exact_verify, "keep": _exact_keep, "copy": _exact_copy}.get(case.get("how", case["op"]), _exact_attn)(s, case)
