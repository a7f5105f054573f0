"""The operators of a served batch, as cases to be timed: a decode step (or a
prompt) of many requests over one paged key-value cache.

  append   Q and K normalised (or not) and rotated, K and V appended to the
           pages of each token's sequence
  attn     attention of each sequence's new tokens over its pages
  wo       the Q4_0 output projection with each request's low-rank adapter
           beside it
  lora     low-rank adapters of many requests beside any other projection

A case is a dict of plain values:
  op       which of the above
append, attn:
  heads, kv    query heads and KV heads, of 128
  page, order  cells of a page; "cells": a page is [cell][head][128], as the
               ring keeps a layer, "heads": [head][cell][128]
  seqs, ctx    sequences; cells that the longest holds before the pass (the
               others 1/3 to all of it)
  tokens       most new tokens of a sequence
  ragged       sequences bring 1 to `tokens` of them (else all `tokens`)
append:
  pad          rows behind the last token that belong to no sequence
  norm, rope   RMSNorm with weights before the rotation; "neox" or "normal"
attn:
  idle         every eighth slot of the batch holds no sequence
  sinks, cap   a sink logit for each head; the logits' soft cap (0: none)
wo, lora:
  K, N         columns and rows of the projection
  tokens       rows of activations
  adapters     resident adapters, of rank `rank` or (mixed) a quarter of it
               to all of it
  runs         tokens come request by request (prompts), else each token is
               another request's (a decode batch); some have no adapter
"""
import math

import numpy as np
import torch

own = False

D, EPS = 128, 1e-6
SCALE = 1.0 / math.sqrt(D)
FREQ_BASE = 1000000.0


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _append(name, seqs, ctx, tokens, heads=32, kv=8, page=16, order="cells", ragged=False, pad=0, norm=True,
            rope="neox"):
    return {"name": name, "op": "append", "heads": heads, "kv": kv, "page": page, "order": order, "seqs": seqs,
            "ctx": ctx, "tokens": tokens, "ragged": ragged, "pad": pad, "norm": norm, "rope": rope}


def _attn(name, seqs, ctx, tokens=1, heads=32, kv=8, page=16, order="cells", ragged=False, idle=False, sinks=False,
          cap=0.0):
    return {"name": name, "op": "attn", "heads": heads, "kv": kv, "page": page, "order": order, "seqs": seqs,
            "ctx": ctx, "tokens": tokens, "ragged": ragged, "idle": idle, "sinks": sinks, "cap": cap}


def _lora(name, op, K, N, tokens, adapters, rank, mixed=False, runs=False):
    return {"name": name, "op": op, "K": K, "N": N, "tokens": tokens, "adapters": adapters, "rank": rank,
            "mixed": mixed, "runs": runs}


def listed():
    return [
        # one decode step of a server's batch, its last slots empty: latency
        _append("append-decode-40", 40, 5000, 1, pad=8),
        # a dozen requests' turns at once, of a model without Q/K norms that
        # rotates neighbouring dims, over head-major pages
        _append("append-turns-12", 12, 9000, 61, page=64, order="heads", ragged=True, norm=False, rope="normal"),
        # prompts of a larger model: bandwidth
        _append("append-prompts-4", 4, 0, 2048, heads=64, page=256),
        # one user, a short conversation: latency
        _attn("attn-1-700", 1, 700),
        # a small server's decode step
        _attn("attn-24-4000", 24, 4000, idle=True),
        # one user, a long document, a larger model: one axis to split
        _attn("attn-1-100k", 1, 100000, heads=64, page=64),
        # a full server's decode step: bandwidth
        _attn("attn-96-9000", 96, 9000, page=256, order="heads"),
        # speculative verify of 2 to 6 drafts each, with sinks
        _attn("attn-verify-10", 10, 6000, tokens=6, page=32, ragged=True, sinks=True),
        # the projection of one token with its adapter: latency
        _lora("wo-8b-1", "wo", 4096, 4096, 1, 8, 16),
        # the projection of a decode batch, larger model, adapters of
        # several ranks
        _lora("wo-32b-48", "wo", 8192, 5120, 48, 20, 32, mixed=True),
        # turns of nine requests through the Q projection
        _lora("lora-turns-300", "lora", 2560, 4096, 300, 9, 64, mixed=True, runs=True),
        # prompts of five requests: bandwidth
        _lora("lora-prompts-8000", "lora", 4096, 4096, 8000, 6, 16, runs=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST = {"append": 6.3e8, "attn": 2.3e9, "wo": 3.0e7, "lora": 3.9e8}   # bytes of a drawn case: the largest listed's


def draw(rng):
    op = rng.choice(["append", "append", "attn", "attn", "attn", "wo", "lora", "lora"])
    if op in ("append", "attn"):
        heads, kv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (8, 8)])
        page = rng.choice([16, 16, 32, 48, 64, 256])
        order = rng.choice(["cells", "cells", "heads"])
    if op == "append":
        tokens = rng.choice([1, 1, _log(rng, 2, 3000)])
        c = _append("", _log(rng, 1, 64), rng.choice([0, _log(rng, 1, 9000)]), tokens, heads, kv, page, order,
                    ragged=rng.random() < 0.5, pad=rng.choice([0, 0, 5]), norm=rng.random() < 0.6,
                    rope=rng.choice(["neox", "neox", "normal"]))
    elif op == "attn":
        tokens = rng.choice([1, 1, 1, rng.randint(2, 8)])
        c = _attn("", _log(rng, 1, 128), _log(rng, 1, 90000), tokens, heads, kv, page, order,
                  ragged=rng.random() < 0.5, idle=rng.random() < 0.3, sinks=rng.random() < 0.3,
                  cap=rng.choice([0.0, 0.0, 30.0]))
    elif op == "wo":
        K, N = rng.choice([(4096, 2560), (4096, 4096), (8192, 5120)])
        c = _lora("", "wo", K, N, _log(rng, 1, 64), _log(rng, 1, 48), rng.choice([8, 16, 32, 64]),
                  mixed=rng.random() < 0.5, runs=rng.random() < 0.3)
    else:
        K, N = rng.choice([(2560, 4096), (2560, 1024), (4096, 2560), (4096, 4096), (5120, 8192)])
        c = _lora("", "lora", K, N, _log(rng, 1, 8000), _log(rng, 1, 32), rng.choice([8, 16, 32, 64]),
                  mixed=rng.random() < 0.5, runs=rng.random() < 0.7)
    while work(c)["bytes"] > _MOST[op]:
        if op == "append":
            c["tokens"] = max(1, c["tokens"] * 2 // 3)
            c["seqs"] = max(1, c["seqs"] * 5 // 6)
        elif op == "attn":
            c["seqs"] = max(1, c["seqs"] * 5 // 6)
            c["ctx"] = c["ctx"] * 5 // 6
        else:
            c["tokens"] = max(1, c["tokens"] * 2 // 3)
            c["adapters"] = max(1, c["adapters"] * 5 // 6)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# sizes: what a case's sequences and tokens are
# ---------------------------------------------------------------------------

def _counts(case):
    """New tokens of each sequence."""
    n, t = case["seqs"], case["tokens"]
    c = [1 + (5 * s + 3) % t if case["ragged"] else t for s in range(n)]
    return [0 if case.get("idle") and s % 8 == 5 else c[s] for s in range(n)]


def _lengths(case):
    """Cells of each sequence, its new tokens among them."""
    n, ctx = case["seqs"], case["ctx"]
    old = [ctx] if n == 1 else [ctx * (n + 2 * ((7 * s) % n)) // (3 * n - 2) for s in range(n)]
    return [o + c if c else 0 for o, c in zip(old, _counts(case))]


def _ranks(case):
    n, r = case["adapters"], case["rank"]
    return [max(1, r * (1 + (3 * a) % 4) // 4) if case["mixed"] else r for a in range(n)]


def _ids(case):
    """Adapter of each token, -1: none."""
    t, n = case["tokens"], case["adapters"]
    if t == 1:
        return [n - 1]
    if case["runs"]:
        pieces = min(t, n + 1)
        return [(i * pieces // t + n) % (n + 1) - 1 for i in range(t)]
    return [(5 * i + i // 7) % (n + 1) - 1 for i in range(t)]


def work(case):
    """append: every new row read and written once. attn: the cells that a
    sequence's tokens see, once, the queries and the outputs; the products of
    the visible pairs. wo, lora: the projection's weights, those of the
    adapters that a token has, the activations and the outputs."""
    if case["op"] == "append":
        t, h, k = sum(_counts(case)), case["heads"], case["kv"]
        return {"bytes": t * D * (8 * h + 12 * k), "flops": t * D * (h + k) * (6 if not case["norm"] else 10)}
    if case["op"] == "attn":
        h, k, counts, lens = case["heads"], case["kv"], _counts(case), _lengths(case)
        pairs = sum(c * n - c * (c - 1) // 2 for c, n in zip(counts, lens))
        return {"bytes": sum(lens) * k * D * 4 + sum(counts) * h * D * 8, "flops": 4 * D * h * pairs}
    K, N, t, ranks, ids = case["K"], case["N"], case["tokens"], _ranks(case), _ids(case)
    low = sum(ranks[a] for a in ids if a >= 0)
    byts = sum(ranks[a] for a in set(ids) if a >= 0) * (K + N) * 2 + t * (K + N) * 4
    if case["op"] == "wo":
        return {"bytes": byts + N * K // 32 * 18, "flops": 2 * t * K * N + 2 * low * (K + N)}
    return {"bytes": byts + t * N * 4, "flops": 2 * low * (K + N)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _State:
    pass


def _pool(case, n_pages):
    heads = case["order"] == "heads"
    return (n_pages, case["kv"], case["page"], D) if heads else (n_pages, case["page"], case["kv"], D)


def _paged(s, case, g):
    """The sequences' lengths and page tables; pages come in no order, the
    tables' unused entries name none."""
    lens, page = _lengths(case), case["page"]
    need = [(n + page - 1) // page for n in lens]
    s.n_pages, s.max_pages = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(s.n_pages, device="cuda", generator=g).int()
    table = torch.full((case["seqs"], s.max_pages), -1, dtype=torch.int32)
    at = 0
    where = torch.full((case["seqs"], s.max_pages), -1, dtype=torch.int64)
    for i, n in enumerate(need):
        where[i, :n] = torch.arange(at, at + n)
        at += n
    where = where.cuda()
    s.table = torch.where(where >= 0, order[where.clamp(min=0)], table.cuda())
    s.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s.counts = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")


def _angles(positions):
    """The float32 angles the operator is defined by, of positions 0 to
    `positions` - 1: pair i's is the position multiplied i times by
    base^(-2/128)."""
    scale = np.float32(np.float64(FREQ_BASE) ** (-2.0 / D))
    th, out = np.arange(positions, dtype=np.float32), np.empty((D // 2, positions), np.float32)
    for i in range(D // 2):
        out[i] = th
        th = th * scale
    return torch.from_numpy(out.T.copy())


def prepare(case, seed):
    s = _State()
    s.case, s.call = case, None
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, dtype=dtype, device="cuda", generator=g)

    if case["op"] == "append":
        _paged(s, case, g)
        counts, lens = _counts(case), _lengths(case)
        seq = [i for i, c in enumerate(counts) for _ in range(c)]
        pos = [p for c, n in zip(counts, lens) for p in range(n - c, n)]
        s.n = len(seq)
        T = s.n + case["pad"]
        s.seq = torch.tensor(seq + [-1] * case["pad"], dtype=torch.int32, device="cuda")
        s.pos = torch.tensor(pos + [0] * case["pad"], dtype=torch.int32, device="cuda")
        s.q, s.k, s.v = randn(T, case["heads"], D) * 2, randn(T, case["kv"], D) * 2, randn(T, case["kv"], D)
        s.qw, s.kw = 1.6 + 0.3 * randn(D), 1.6 + 0.3 * randn(D)
        s.angles = _angles(max(pos) + 1).cuda()
        s.q_out = torch.zeros((T, case["heads"], D), device="cuda")
        s.kc, s.vc = (torch.zeros(_pool(case, s.n_pages), dtype=torch.float16, device="cuda") for _ in range(2))
    elif case["op"] == "attn":
        _paged(s, case, g)
        n, t, h = case["seqs"], case["tokens"], case["heads"]
        # a spread of the scores of about 2.5
        s.q = randn(n, t, h, D) * 2.5
        s.kc, s.vc = (randn(*_pool(case, s.n_pages), dtype=torch.float16) for _ in range(2))
        s.sinks = randn(h) * 2 + 4 if case["sinks"] else None
        s.out = torch.zeros((n, t, h, D), device="cuda")
    else:
        K, N, T, A, R = case["K"], case["N"], case["tokens"], case["adapters"], case["rank"]
        s.x = randn(T, K) * (torch.rand((T, 1), device="cuda", generator=g) + 0.05)
        # slots of the largest rank; what lies behind a smaller one is stale
        s.a = (randn(A, R, K) / math.sqrt(K)).half()
        s.b = (randn(A, N, R) / math.sqrt(R)).half()
        s.ranks = torch.tensor(_ranks(case), dtype=torch.int32, device="cuda")
        s.scales = torch.rand(A, device="cuda", generator=g) * 1.5 + 0.5
        s.ids = torch.tensor(_ids(case), dtype=torch.int32, device="cuda")
        s.y = torch.zeros((T, N), device="cuda")
        if case["op"] == "wo":
            # Q4_0 blocks: an f16 scale, then the nibbles of 32 weights
            s.w = torch.randint(0, 256, (N, K // 32, 18), dtype=torch.uint8, device="cuda", generator=g)
            d = (torch.rand((N, K // 32, 1), device="cuda", generator=g) * 0.01 + 0.002).half()
            s.w[:, :, :2] = d.view(torch.uint8)
        else:
            s.base = randn(T, N)
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _norm_rotate(x, w, s, case):
    if case["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a = s.angles[s.pos[:s.n].long()][:, None]
    c, n = a.cos(), a.sin()
    if case["rope"] == "neox":
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([lo * c - hi * n, lo * n + hi * c], -1)
    lo, hi = x[..., 0::2], x[..., 1::2]
    return torch.stack([lo * c - hi * n, lo * n + hi * c], -1).flatten(-2)


def _plain_append(s, case):
    n, page = s.n, case["page"]
    pos, seq = s.pos[:n].long(), s.seq[:n].long()
    pages, off = s.table[seq, pos // page].long(), pos % page
    s.q_out[:n] = _norm_rotate(s.q[:n], s.qw, s, case)
    k, v = _norm_rotate(s.k[:n], s.kw, s, case).half(), s.v[:n].half()
    if case["order"] == "heads":
        s.kc[pages, :, off], s.vc[pages, :, off] = k, v
    else:
        s.kc[pages, off], s.vc[pages, off] = k, v
    return {"q": s.q_out, "k": s.kc, "v": s.vc}


def _plain_attn(s, case):
    n, t, h, hk, page = case["seqs"], case["tokens"], case["heads"], case["kv"], case["page"]
    L = s.max_pages * page
    pages = s.table.long().clamp(min=0)

    def cells(pool):                            # (n, hk, L, D)
        x = pool[pages].float()
        return x.permute(0, 2, 1, 3, 4).reshape(n, hk, L, D) if case["order"] == "heads" else \
            x.reshape(n, L, hk, D).permute(0, 2, 1, 3).contiguous()

    q = s.q.view(n, t, hk, h // hk, D).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, D)
    score = torch.matmul(q, cells(s.kc).transpose(2, 3)) * SCALE
    score = score.view(n, hk, t, h // hk, L)
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    at = torch.arange(t, device="cuda")
    sees = s.lens[:, None] - s.counts[:, None] + 1 + at               # cells that token t sees
    seen = torch.arange(L, device="cuda") < sees[..., None]
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if case["sinks"]:
        sink = s.sinks.view(1, hk, 1, h // hk, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    o = torch.matmul(p.view(n, hk, -1, L), cells(s.vc)).view(n, hk, t, h // hk, D)
    o = (o / torch.where(total > 0, total, torch.ones_like(total))).permute(0, 2, 1, 3, 4).reshape(n, t, h, D)
    return {"out": torch.where((at < s.counts[:, None])[..., None, None], o, s.out)}


def _plain_lora(s, case):
    K, N, A, R = case["K"], case["N"], case["adapters"], case["rank"]
    if case["op"] == "wo":
        xb = s.x.view(-1, K // 32, 32)
        d = xb.abs().amax(-1, keepdim=True) / 127.0
        xq = torch.round(xb * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))) * d.half().float()
        dw = s.w[:, :, :2].contiguous().view(torch.float16).float()
        nib = s.w[:, :, 2:]
        w = (torch.cat([nib & 15, nib >> 4], -1).float() - 8.0) * dw
        base = xq.view(-1, K) @ w.view(N, K).T
    else:
        base = s.base
    # every adapter's product with every token, what is not a token's own
    # left out
    low = (s.x @ s.a.float().view(A * R, K).T).view(-1, A, R)
    mine = (s.ids[:, None, None] == torch.arange(A, device="cuda")[:, None]) & \
           (torch.arange(R, device="cuda") < s.ranks[:, None])
    low = torch.where(mine, low * s.scales[:, None], torch.zeros_like(low))
    return {"y": base + low.view(-1, A * R) @ s.b.float().permute(0, 2, 1).reshape(A * R, N)}


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
    from arclight_amd import abi, lora, matmul, paged
    if case["op"] in ("append", "attn"):
        cache = paged.PagedCache(_dev(s.kc), _dev(s.vc), _dev(s.table), heads_first=case["order"] == "heads")
    if case["op"] == "append":
        rope = abi.qwen3_rope()
        rope.mode = abi.AL_ROPE_NEOX if case["rope"] == "neox" else abi.AL_ROPE_NORMAL
        return paged.AppendCall(cache, _dev(s.q), _dev(s.k), _dev(s.v), _dev(s.pos), _dev(s.seq), _dev(s.q_out),
                                q_w=_dev(s.qw), k_w=_dev(s.kw), eps=EPS, norm=case["norm"], rope=rope)
    if case["op"] == "attn":
        return paged.AttentionCall(cache, _dev(s.q), _dev(s.lens), _dev(s.out), counts=_dev(s.counts),
                                   sinks=None if s.sinks is None else _dev(s.sinks), scale=SCALE,
                                   logit_softcap=case["cap"])
    ad = lora.Adapters(_dev(s.a), _dev(s.b), _dev(s.scales), ranks=_dev(s.ranks))
    if case["op"] == "wo":
        w = matmul.Q4_0View(s.w.data_ptr(), case["K"], case["N"])
        return lora.ProjectCall(ad, w, _dev(s.x), _dev(s.ids), _dev(s.y))
    return lora.ApplyCall(ad, _dev(s.x), _dev(s.ids), _dev(s.base), _dev(s.y))


def run(s):
    case = s.case
    if not own:
        return {"append": _plain_append, "attn": _plain_attn}.get(case["op"], _plain_lora)(s, case)
    if s.call is None:
        s.call = _bind(s, case)
    s.call.run()
    if case["op"] == "append":
        return {"q": s.q_out, "k": s.kc, "v": s.vc}
    return {"out": s.out} if case["op"] == "attn" else {"y": s.y}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_append(s, case):
    page = case["page"]
    q = torch.zeros_like(s.q_out, dtype=torch.float64)
    k = torch.zeros(s.kc.shape, dtype=torch.float64, device="cuda")
    v = torch.zeros_like(k)
    seq, pos, table = s.seq.tolist(), s.pos.tolist(), s.table.cpu().numpy()
    cell = torch.tensor([int(table[i, p // page]) * page + p % page for i, p in zip(seq[:s.n], pos[:s.n])],
                        device="cuda")
    theta = np.asarray(pos[:s.n], np.float32)
    step = np.float32(np.float64(FREQ_BASE) ** (-2.0 / D))
    cols = []
    for _ in range(D // 2):
        cols.append(theta.astype(np.float64))
        theta = (theta * step).astype(np.float32)
    turn = torch.from_numpy(np.stack(cols, 1)).cuda()
    turn = torch.polar(torch.ones_like(turn), turn)[:, None, :]
    for x, w, out in ((s.q, s.qw, q), (s.k, s.kw, None)):
        x = x[:s.n].double()
        if case["norm"]:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
        pair = x.unflatten(-1, (2, D // 2)).transpose(-1, -2) if case["rope"] == "neox" else x.unflatten(-1, (D // 2, 2))
        r = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        r = (r.transpose(-1, -2) if case["rope"] == "neox" else r).flatten(-2)
        if out is not None:
            out[:s.n] = r
        else:
            rows = r
    for pool, new in ((k, rows), (v, s.v[:s.n].double())):
        flat = torch.zeros((s.n_pages * page, case["kv"], D), dtype=torch.float64, device="cuda")
        flat[cell] = new
        flat = flat.view(s.n_pages, page, case["kv"], D)
        pool.copy_(flat.transpose(1, 2) if case["order"] == "heads" else flat)
    return {"q": q, "k": k, "v": v}


def _exact_attn(s, case):
    n, t, h, hk, page = case["seqs"], case["tokens"], case["heads"], case["kv"], case["page"]
    out = torch.zeros((n, t, h, D), dtype=torch.float64, device="cuda")
    for i, (c, m) in enumerate(zip(_counts(case), _lengths(case))):
        if c == 0:
            continue
        pages = s.table[i, :(m + page - 1) // page].long()
        for j in range(hk):
            kv = []
            for pool in (s.kc, s.vc):
                x = pool[pages, j] if case["order"] == "heads" else pool[pages, :, j]
                kv.append(x.reshape(-1, D)[:m].double())
            q = s.q[i, :c, j * (h // hk):(j + 1) * (h // hk)].double()
            x = q.reshape(-1, D) @ kv[0].T / math.sqrt(D)
            x = x.view(c, h // hk, m)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            hidden = torch.arange(m, device="cuda")[None] > torch.arange(m - c, m, device="cuda")[:, None]
            x.masked_fill_(hidden[:, None], -math.inf)
            if case["sinks"]:
                sink = s.sinks[j * (h // hk):(j + 1) * (h // hk)].double()
                x = torch.cat([x, sink[None, :, None].expand(c, -1, 1)], -1)
            w = torch.softmax(x, -1)[..., :m]
            out[i, :c, j * (h // hk):(j + 1) * (h // hk)] = (w.reshape(-1, m) @ kv[1]).view(c, h // hk, D)
    return {"out": out}


def _exact_lora(s, case):
    K, N = case["K"], case["N"]
    x = s.x.double()
    if case["op"] == "wo":
        # the activations' 8-bit blocks are the operator's own definition,
        # in float32
        blocks = s.x.reshape(-1, 32)
        d = blocks.abs().max(-1, keepdim=True).values / 127.0
        inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
        eight = (torch.round(blocks * inv).double() * d.half().double()).view(-1, K)
        y = torch.empty((x.shape[0], N), dtype=torch.float64, device="cuda")
        for n0 in range(0, N, 1024):
            w = s.w[n0:n0 + 1024]
            half = w[..., :2].contiguous().view(torch.float16).double()
            low, high = (w[..., 2:] % 16).double() - 8, torch.div(w[..., 2:], 16, rounding_mode="floor").double() - 8
            y[:, n0:n0 + 1024] = eight @ (torch.cat([low, high], -1) * half).reshape(-1, K).T
    else:
        y = s.base.double()
    for a, r in enumerate(_ranks(case)):
        mine = torch.tensor([i for i, who in enumerate(_ids(case)) if who == a], dtype=torch.int64, device="cuda")
        if len(mine):
            y[mine] += s.scales[a].double() * ((x[mine] @ s.a[a, :r].double().T) @ s.b[a, :, :r].double().T)
    return {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn}.get(case["op"], _exact_lora)(s, case)
