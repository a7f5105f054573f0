"""Verification where many of a node's children, drawn from a draft's row, are
rejected one after another: the accepted path and the token after it by the
definition, in time that grows with the children and not with their square."""
import time

import numpy as np
import pytest

from arclight_amd import abi
from tests import tree_cases as C
from tests.test_gpu_draft import _same, _verify
from tests.test_gpu_paged import _case, _put

pytestmark = pytest.mark.gpu


def _rows(rng, n, T, V):
    """Probabilities of the target and of the draft, and tokens that the draft is
    more likely to draw by half at least: once one is rejected, nothing of any is left."""
    target = rng.random((n, T, V)) ** 3
    target = (target / target.sum(-1, keepdims=True)).astype(np.float32)
    draft = target * np.exp(rng.standard_normal(target.shape) * 0.7)
    draft = (draft / draft.sum(-1, keepdims=True)).astype(np.float32)
    return target, draft, lambda s, v, k: rng.choice(np.flatnonzero(draft[s, v] > 1.5 * target[s, v]), k)


@pytest.mark.parametrize("V", [300, 2048, 2049, 20003])
def test_siblings_at_several_nodes(gpu, V):
    """Root, its third child and a child of that with children of their own; trees
    that end at each of them."""
    _case(f"siblings of a draft, V={V}")
    rng = np.random.default_rng(V)
    n, T = 6, 40
    target, draft, pick = _rows(rng, n, T, V)
    parents = np.tile(np.array([-1] + [0] * 12 + [3] * 13 + [20] * 14, np.int32), (n, 1))
    tokens, accept = np.zeros((n, T), int), np.full((n, T), 0.99)
    for s in range(n):
        for v in (0, 3, 20):
            u = np.flatnonzero(parents[s] == v)
            tokens[s, u] = pick(s, v, len(u))
    for s in range(n):                                               # nodes 3 and 20 are accepted, as the paths go on
        if s % 3 > 0:
            tokens[s, 3] = np.argmax(target[s, 0] / draft[s, 0])
            accept[s, 3] = 0.0
        if s % 3 > 1:
            tokens[s, 20] = np.argmax(target[s, 3] / draft[s, 3])
            accept[s, 20] = 0.0
    sample = rng.random(n)
    counts = np.array([T, T, T, 13, 26, 21])
    got = _verify(target, tokens, accept, sample, parents, counts, draft)
    assert list(got[1]) == [1, 2, 3, 1, 2, 3]
    _same(got, target, tokens, accept, sample, parents, counts, draft)


def test_a_thousand_siblings(gpu):
    """1023 children of the root, all rejected, and 511 of them: each is a pass
    over the rows of some 30 us (50000 tokens by 256 threads), 0.03 s in all. Were
    each to begin from the rows again with a division for every rejection before it,
    a thread's 196 tokens times 1023^2 / 2 divisions of 0.05 us would take 5 s."""
    from arclight_amd import device
    from arclight_amd import draft as calls
    _case("1023 siblings of a draft")
    rng = np.random.default_rng(1)
    n, T, V = 2, 1024, 50000
    target, draft = (np.lib.stride_tricks.as_strided(np.ascontiguousarray(x), (n, T, V), (0, 0, 4)) for x in _rows(rng, 1, 1, V)[:2])
    parents = np.tile(np.array([-1] + [0] * (T - 1), np.int32), (n, 1))
    tokens = np.stack([rng.choice(np.flatnonzero(draft[0, 0] > 1.5 * target[0, 0]), T) for _ in range(n)])
    accept, sample, counts = np.full((n, T), 0.99), rng.random(n), np.array([T, 512])
    want = [C.verify(target[s], tokens[s], accept[s], sample[s], parents[s], counts[s], draft[s]) for s in range(n)]
    rows = [device.DeviceTensor(_put(np.ascontiguousarray(x[0, 0])).buf, abi.AL_TYPE_F32, (n, T, V), (0, 0, 4)) for x in (target, draft)]
    args = [rows[0], _put(tokens.astype(np.int32)), _put(accept.astype(np.float32)), _put(sample.astype(np.float32))]
    kw = dict(parents=_put(parents), counts=_put(counts.astype(np.int32)), draft=rows[1])
    calls.verify(*args, **kw)                                        # (allocates the workspace)
    device.synchronize()
    start = time.perf_counter()
    got = [x.numpy(np.int32) for x in calls.verify(*args, **kw)]
    took = time.perf_counter() - start
    for s, (path, follow) in enumerate(want):
        assert path == [0] and got[1][s] == 1 and list(got[0][s, :2]) == [0, -1] and got[2][s] == follow
    print(f"{took * 1e3:.1f} ms", flush=True)
    assert took < 1.0
