"""The paged cache, its attention and the projection with adapters as a
server's layer runs them: one after another on a stream, eager and captured,
prompts and decode steps, each stage against the plain forms in 64 bits."""
import math

import numpy as np
import pytest

from arclight_amd import abi
from oracle import oracle as O
from tests import paged_cases as P
from tests.test_gpu_lora import EPS32, _adapters, _ref
from tests.test_gpu_paged import MARK, _check, _put
from tests.test_oracle_q4 import abs_bound, dequant_q4_0, dequant_q8_0

pytestmark = pytest.mark.gpu
D = 128


def _case(name):
    print(f"\n[case] {name}", flush=True)


class Layer:
    """Host and device sides of one layer: a cache for n sequences, the output
    projection and its adapters."""

    def __init__(self, rng, n, Hq, Hkv, page, max_pages, pages, N, R, n_adapters):
        self.n, self.Hq, self.Hkv, self.page = n, Hq, Hkv, page
        self.pool = P.Pool(rng, [0] * n, Hkv, page, spare=pages, max_pages=max_pages)
        self.free = list(rng.permutation(pages))
        self.lens = [0] * n
        self.cache = self.pool.device()
        self.norms = [rng.standard_normal(D).astype(np.float32) for _ in range(2)]
        self.d_norms = [_put(w) for w in self.norms]
        K = Hq * D
        self.w = O.random_q4_0(rng, N, K)
        self.ranks = rng.integers(1, R + 1, n_adapters)
        self.a, self.b = _adapters(rng, n_adapters, R, K, N, self.ranks)
        self.scales = (rng.random(n_adapters) * 2).astype(np.float32)

    def device_side(self):
        from arclight_amd import lora, matmul
        self.ad = lora.Adapters(_put(self.a.view(np.uint16)), _put(self.b.view(np.uint16)), _put(self.scales),
                                _put(self.ranks.astype(np.int32)))
        self.wd = matmul.Q4_0Matrix(self.w.view(np.uint8), self.Hq * D, self.w.shape[0])

    def grow(self, s, by):
        for i in range((self.lens[s] + self.page - 1) // self.page, (self.lens[s] + by + self.page - 1) // self.page):
            self.pool.table[s, i] = self.free.pop()
        self.lens[s] += by

    def appended(self, k, v, pos, seq, what):
        """The device's pools against the host's with the new rows; the host's
        keys are then the device's."""
        kr = P.norm_rotate(k, self.norms[1], np.where(seq >= 0, pos, 0), 1e-6, "neox")
        pool, page = self.pool, self.page
        for t in np.flatnonzero(seq >= 0):
            at = pool.table[seq[t], pos[t] // page], pos[t] % page
            pool.k[at], pool.v[at] = kr[t].astype(np.float16), v[t].astype(np.float16)
        got_k, got_v = pool.download(self.cache)
        seen = ~np.isnan(pool.k)
        assert np.array_equal(got_v.view(np.uint16), pool.v.view(np.uint16)), what
        assert np.array_equal(seen, ~np.isnan(got_k)), what
        # one float16 step, and 3e-5 of the producers' float32
        assert np.all(np.abs(got_k[seen].astype(np.float64) - pool.k[seen]) <= np.abs(pool.k[seen].astype(np.float64)) * 2.0 ** -10 + 3e-5), what
        pool.k = np.where(seen, got_k, pool.k)

    def projected(self, x, ids, y, what):
        base = O.mul_mat_q4_0(self.w, x)
        ref, bound = _ref(x, self.a, self.b, self.scales, self.ranks, ids, base)
        bound += (x.shape[1] // 32 + 16) * 2 * EPS32 * abs_bound(dequant_q4_0(self.w), dequant_q8_0(O.quantize_q8_0(x)))
        err = np.abs(y.astype(np.float64) - ref)
        print(f"{what}: projection, worst error {float((err / bound).max()):.3f} of the bound", flush=True)
        assert np.all(err <= bound), what


@pytest.mark.parametrize("replayed", [False, True])
def test_layers_decode_steps(gpu, replayed):
    """Append, attention, projection with adapters for a batch with an empty
    slot (whose row names no adapter, and whose attention row is what it was),
    sequences and adapters changing between the steps."""
    from arclight_amd import device, fattn, lora, paged
    _case(f"decode steps of a layer, replayed={replayed}")
    rng = np.random.default_rng(31)
    n, Hq, Hkv, N, A = 5, 32, 8, 320, 4
    L = Layer(rng, n, Hq, Hkv, 16, 12, 50, N, 16, A)
    for s, m in enumerate((17, 0, 150, 31, 64)):
        L.grow(s, m)
        for c in range(m):
            at = L.pool.table[s, c // 16], c % 16
            L.pool.k[at], L.pool.v[at] = rng.standard_normal((2, Hkv, D))
    L.cache = L.pool.device()
    L.device_side()
    st = device.Stream()
    buf = {k: device.DeviceTensor.from_numpy(np.zeros(s, t)) for k, s, t in (
        ("q", (n, Hq, D), np.float32), ("k", (n, Hkv, D), np.float32), ("v", (n, Hkv, D), np.float32), ("pos", (n,), np.int32),
        ("seq", (n,), np.int32), ("lens", (n,), np.int32), ("counts", (n,), np.int32), ("out", (n, 1, Hq, D), np.float32),
        ("ids", (n,), np.int32), ("y", (n, N), np.float32))}
    # the queries are rotated where they are
    app = paged.AppendCall(L.cache, buf["q"], buf["k"], buf["v"], buf["pos"], buf["seq"], buf["q"], q_w=L.d_norms[0],
                           k_w=L.d_norms[1], eps=1e-6, rope=abi.qwen3_rope(), stream=st)
    att = paged.AttentionCall(L.cache, device.DeviceTensor(buf["q"].buf, abi.AL_TYPE_F32, (n, 1, Hq, D)), buf["lens"], buf["out"],
                              counts=buf["counts"], scale=1 / math.sqrt(D), stream=st)
    pro = lora.ProjectCall(L.ad, L.wd, device.DeviceTensor(buf["out"].buf, abi.AL_TYPE_F32, (n, Hq * D)), buf["ids"], buf["y"], st)

    def step():
        app.run()
        att.run()
        pro.run()

    graph = None
    for i in range(6):
        idle = i % 3
        host = {k: rng.standard_normal(buf[k].shape).astype(np.float32) for k in ("q", "k", "v")}
        host["seq"] = np.array([-1 if s == idle else s for s in range(n)], np.int32)
        host["pos"] = np.array(L.lens, np.int32)
        for s in range(n):
            if s != idle:
                L.grow(s, 1)
        host["lens"], host["counts"] = np.array(L.lens, np.int32), (host["seq"] >= 0).astype(np.int32)
        host["out"] = np.full(buf["out"].shape, 0.5, np.float32)
        host["ids"] = np.where(host["seq"] >= 0, rng.integers(-1, A, n), -1).astype(np.int32)
        for k, x in host.items():
            buf[k].buf.upload(x)
        L.cache.table.buf.upload(L.pool.table)
        device.synchronize()
        if replayed and i == 1:
            graph = device.Graph(st, step)
        graph.launch(st) if graph else step()
        device.synchronize()
        fattn.device_errors()
        L.appended(host["k"], host["v"], host["pos"], host["seq"], f"step {i}")
        q = buf["q"].numpy(np.float32)
        mine = host["seq"] >= 0
        ref_q = P.norm_rotate(host["q"], L.norms[0], np.where(mine, host["pos"], 0), 1e-6, "neox")
        assert np.all(np.abs(q[mine] - ref_q[mine]) <= 3e-5 + 1e-6 * np.abs(ref_q[mine]))
        assert np.array_equal(q[~mine], host["q"][~mine])
        out = buf["out"].numpy(np.float32)
        assert np.all(out[~mine] == 0.5)
        ref, bound = P.attention(L.pool, q[:, None], L.lens, host["counts"].tolist(), 1 / math.sqrt(D))
        _check(np.where(np.isnan(ref), np.float32(MARK), out), (ref, bound), f"step {i}")
        L.projected(out.reshape(n, -1), host["ids"], buf["y"].numpy(np.float32), f"step {i}")
    if graph:
        graph.destroy()
    st.destroy()


def test_layers_prompts_then_decode(gpu):
    """Two prompts of different lengths in one append, their attention with a
    count each, the adapters beside a projection that is already there
    (apply), and then a token more for each."""
    from arclight_amd import device, fattn, lora, paged
    _case("prompts of a layer, then a token")
    rng = np.random.default_rng(32)
    n, Hq, Hkv, N, A = 2, 8, 2, 130, 3
    L = Layer(rng, n, Hq, Hkv, 32, 20, 30, N, 24, A)
    L.device_side()
    for counts in ([500, 170], [1, 1]):
        T = max(counts)
        for s in range(n):
            L.grow(s, counts[s])
        L.cache.table.buf.upload(L.pool.table)
        # rows as the attention takes them, T for each sequence, padded
        seq = np.array([[s if t < counts[s] else -1 for t in range(T)] for s in range(n)], np.int32).reshape(-1)
        pos = np.array([[L.lens[s] - counts[s] + t for t in range(T)] for s in range(n)], np.int32).reshape(-1)
        q, k, v = (rng.standard_normal((n * T, H, D)).astype(np.float32) for H in (Hq, Hkv, Hkv))
        ids = np.where(seq >= 0, rng.integers(0, A, n).repeat(T), -1).astype(np.int32)
        qd = _put(q)
        paged.append(L.cache, qd, _put(k), _put(v), _put(pos), _put(seq), qd, q_w=L.d_norms[0], k_w=L.d_norms[1], eps=1e-6,
                     rope=abi.qwen3_rope())
        out = _put(np.full((n, T, Hq, D), MARK, np.float32))
        paged.attention(L.cache, device.DeviceTensor(qd.buf, abi.AL_TYPE_F32, (n, T, Hq, D)), _put(np.array(L.lens, np.int32)), out,
                        counts=_put(np.array(counts, np.int32)), scale=1 / math.sqrt(D))
        y0 = rng.standard_normal((n * T, N)).astype(np.float32)
        y = lora.apply(L.ad, device.DeviceTensor(out.buf, abi.AL_TYPE_F32, (n * T, Hq * D)), _put(ids), _put(y0))
        device.synchronize()
        fattn.device_errors()
        L.appended(k, v, pos, seq, f"{counts}")
        qr = qd.numpy(np.float32).reshape(n, T, Hq, D)
        got = out.numpy(np.float32)
        _check(got, P.attention(L.pool, qr, L.lens, counts, 1 / math.sqrt(D)), f"{counts}")
        ref, bound = _ref(got.reshape(n * T, -1), L.a, L.b, L.scales, L.ranks, ids, y0)
        err = np.abs(y.numpy(np.float32).astype(np.float64) - ref)
        print(f"{counts}: adapters, worst error {float((err / bound).max()):.3f} of the bound", flush=True)
        assert np.all(err <= bound)


@pytest.mark.parametrize("T", [1, 5, 90])
def test_pages_in_order_are_a_ring(gpu, T):
    """A sequence whose pages follow one another, seen by al_fattn_f16 as a
    ring: the two attentions agree to the roundings of al_fattn_f16, which
    carries queries and probabilities in f16 (2^-11 of each, the largest
    score's and the sum's taken whole)."""
    from arclight_amd import device, fattn, paged
    _case(f"pages as a ring, T={T}")
    rng = np.random.default_rng(33)
    n, Hq, Hkv, page, pages = 333, 16, 4, 16, 24
    pool = P.Pool(rng, [n], Hkv, page, spare=0, max_pages=pages)
    first = 2
    pool.n_pages = pages
    k, v = (rng.standard_normal((pages, page, Hkv, D)).astype(np.float16) for _ in range(2))
    pool.k, pool.v = k, v
    pool.table = (first + np.arange(pages, dtype=np.int32))[None]
    cache = pool.device()
    q = rng.standard_normal((1, T, Hq, D)).astype(np.float32)
    qd = _put(q)
    out = paged.attention(cache, qd, _put(np.array([n], np.int32)), scale=1 / math.sqrt(D))
    cells = (pages - first) * page
    row = Hkv * D * 2
    ring = [device.DeviceTensor(t.buf, abi.AL_TYPE_F16, (1, cells, Hkv, D), (cells * row, row, D * 2, 2), first * page * row, abi.KV_AXES)
            for t in (cache.k, cache.v)]
    r = fattn.flash_attn_ext(fattn.upload_q(q), *ring, scale=1 / math.sqrt(D), kv_len=n, causal_pos0=n - T)
    device.synchronize()
    fattn.device_errors()
    ref, bound = P.attention(pool, q, [n], [T], 1 / math.sqrt(D))
    got = out.numpy(np.float32)
    _check(got, (ref, bound), f"T={T}")
    # a score of q rounded to f16: sum |q| |k| scale 2^-11; a probability, and
    # the sum that divides them: 2^-11 each; their sizes taken whole
    size = np.einsum("thd,chd->thc", np.abs(q[0]).astype(np.float64), np.abs(pool.cells(pool.k, 0, n)).repeat(Hq // Hkv, 1)).max(-1) / math.sqrt(D)
    tol = (2 * size + 2) * 2.0 ** -11 * np.abs(pool.cells(pool.v, 0, n)).max() + 1e-4
    assert np.all(np.abs(r.numpy(np.float32)[0] - got[0]) <= tol[..., None])
