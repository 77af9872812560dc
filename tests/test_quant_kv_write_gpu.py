"""quant/kv_write of many rows: of rows that name one slot the last is kept whatever their number, and the time of a write is in
proportion to its rows."""

import numpy as np
import pytest

import tessel_amd as T
from tests import quant_refs as R
from tests.test_quant_gpu import _say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _open(gpu):
    yield


def _case(rng, slot, g, d, p, pages):
    t = len(slot)
    kn, vn, ks, vs = R.cached(rng, pages, g, p, d)
    qkv = rng.standard_normal((t, 2 * g * d)).astype(np.float16)
    one, zero = np.ones((1, d // 2), np.float32), np.zeros((1, d // 2), np.float32)
    # (position 0: not turned)
    return [qkv, np.zeros(t, np.int32), slot.astype(np.int32), one, zero, R.pack_k(kn), R.pack_v(vn), ks, vs,
            np.full((t, g, d), 7, np.float16), np.full((t, g, d), 7, np.float16)], (kn, vn)


def _want(case, codes):
    qkv, slot, (pages, _, p, _), (t, g, d) = case[0], case[2], case[5].shape, case[9].shape
    x = qkv.reshape(t, 2, g, d)
    last = {s: i for i, s in enumerate(slot.tolist()) if 0 <= s < pages * p}
    at, row = np.array(list(last), np.int64), np.array(list(last.values()), np.int64)
    kv = []
    for j in (0, 1):
        n, pair = codes[j].copy(), case[7 + j].copy()
        if len(at):
            n[at // p, :, at % p], pair[at // p, :, at % p] = R.heads4(x[row, j])
        kv.append((n, pair))
    return [R.pack_k(kv[0][0]), R.pack_v(kv[1][0]), kv[0][1], kv[1][1], x[:, 0], x[:, 1]]


def _check(got, want):
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)


def _slots(rng, kind, t, room):
    if kind == "all":  # each its own, in any order
        return rng.permutation(room)[:t]
    if kind == "one":
        return np.full(t, room - 1)
    if kind == "none":
        return rng.choice([-1, -2 ** 31, room, 2 ** 31 - 1], t)
    if kind == "steps":  # one slot of every page, over and over
        return np.arange(t) * 32 % room
    s = rng.integers(-3, room + 3, t)
    s[rng.integers(0, t, t // 3)] = rng.integers(0, 5, t // 3)
    return s


@pytest.mark.parametrize("kind", ["all", "one", "none", "steps", "mixed"])
@pytest.mark.parametrize("t,g,d,p", [(6144, 2, 32, 16), (6145, 1, 16, 32), (7001, 3, 64, 16), (20011, 1, 16, 64)])
def test_many_rows(kind, t, g, d, p):
    _say("kv_write", kind, t, g, d, p)
    rng = np.random.default_rng(t + len(kind))
    pages = (t + p - 1) // p + 1
    case, codes = _case(rng, _slots(rng, kind, t, pages * p), g, d, p, pages)
    _check(list(T.run("quant", "kv_write", case, outputs=range(5, 11)).values()), _want(case, codes))


def test_many_rows_in_a_graph():
    # Two writes of one handle into two caches, replayed with other slots and with products between that use the same scratch.
    _say("kv_write graph")
    rng = np.random.default_rng(5)
    t, g, d, p, pages = 6500, 1, 32, 16, 410
    cases = [_case(rng, _slots(rng, "mixed", t, pages * p), g, d, p, pages) for _ in range(2)]
    bufs = [[T.tensor(x) for x in c] for c, _ in cases]
    kern = T.kernel("quant", "kv_write", [x.shape for x in cases[0][0]])
    m, n, k = 1500, 2100, 2001
    prod = T.kernel("quant", "linear", [(m, k), (m,), (n, k), (n,), (m, n)])
    pb = [T.alloc(b) for b in (m * k, 4 * m, n * k, 4 * n, 2 * m * n)]
    T.write(pb[0], 0, np.full(m * k, 0x55, np.uint8))
    T.capture_begin()
    for b in bufs:
        T.launch(kern, b)
        T.launch(prod, pb)
    graph = T.capture_end()
    assert T.graph_nodes(graph)["memset"] == 0 and T.graph_nodes(graph)["memcpy"] == 0
    for rep in range(4):
        for (c, codes), b in zip(cases, bufs):
            c[2][:] = _slots(rng, ("mixed", "all", "one", "mixed")[rep], t, pages * p)
            for i in (2, 5, 6, 7, 8):
                T.write(b[i], 0, c[i])
        T.launch(prod, pb)
        T.replay(graph)
        for (c, codes), b in zip(cases, bufs):
            _check([T.read_array(b[i], c[i].dtype, c[i].shape) for i in range(5, 11)], _want(c, codes))
    for b in (*bufs[0], *bufs[1], *pb):
        T.free(b)


def test_time_in_proportion_to_the_rows():
    # 8 times the rows: 8 times the time where each looks at its own slot, 64 times where each looks at all the others'.
    _say("kv_write times")
    g, d, p, us = 1, 16, 16, []
    for t in (32768, 262144):
        shapes = [(t, 2 * g * d), (t,), (t,), (1, d // 2), (1, d // 2), (t // p, g, p, d // 2), (t // p, g, p // 16, d // 2, 16),
                  (t // p, g, p, 2), (t // p, g, p, 2), (t, g, d), (t, g, d)]
        kern = T.kernel("quant", "kv_write", shapes)
        bufs = [T.alloc(4 * int(np.prod(s))) for s in shapes]
        T.write(bufs[2], 0, np.random.default_rng(0).permutation(t).astype(np.int32))
        T.time_launches(kern, bufs, 3)
        us.append(min(T.time_launches(kern, bufs, 5) for _ in range(5)) / 5 * 1e3)
        for b in bufs:
            T.free(b)
    print("[times]", us, flush=True)
    assert us[1] < 24 * us[0], us
