"""The quant kernels on the GPU against plain 64-bit forms (tests/quant_refs.py):
8-bit rows and products by their bits, 4-bit cache writes by their bits,
decode attention over the 4-bit cache within tolerances derived from its
roundings, and the whole as a decode step uses it."""

import numpy as np
import pytest

import tessel_amd as T
from tests import quant_refs as R

pytestmark = pytest.mark.gpu

H = 2.0 ** -11  # half a step of f16, relative
F = 2.0 ** -24  # of f32


@pytest.fixture(autouse=True)
def _open(gpu):
    yield


def _say(*a):
    print("[case]", *a, flush=True)


def run(name, arrays, scalars=(), outputs=()):
    return T.run("quant", name, arrays, scalars, outputs=list(outputs))


# ---------------------------------------------------------------- 8-bit rows

def _quantize(x):
    m, k = x.shape
    # A guard behind the codes: rows of any length end where they end.
    q = np.full((m, k), 99, np.int8)
    out = run("quantize", [x, q, np.zeros(m, np.float32)], outputs=[1, 2])
    return out[1], out[2]


@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (1, 8), (5, 15), (2, 64), (9, 511), (4, 512), (3, 513), (7, 1023),
                                 (6, 1024), (2, 1025), (5, 2048), (3, 2049), (2, 4097), (3, 5632), (2, 8193),
                                 (2, 11008), (1, 16384), (2, 16385), (1, 40001), (300, 96)])
def test_quantize_rows(m, k):
    _say("quantize", m, k)
    rng = np.random.default_rng(m * 100003 + k)
    x = (rng.standard_normal((m, k)) * rng.choice([1e-6, 1.0, 100.0], (m, 1))).astype(np.float16)
    x[0, k // 2] = 0
    if m > 2:
        x[1] = 0
    q, s = _quantize(x)
    wq, ws = R.rows8(x)
    np.testing.assert_array_equal(q, wq)
    np.testing.assert_allclose(s, ws, rtol=2 * F)  # (one division, rounded)


def test_quantize_ties_and_special_values():
    _say("quantize ties")
    # Largest 254 / 2^j: every whole number is a tie or a code; and one either side by an f16 step.
    k = 508
    ties = np.concatenate([np.arange(-254, 255)[:k - 1], [254]]).astype(np.float16)
    near = np.nextafter(ties, np.float16(1000)).astype(np.float16)
    below = np.nextafter(ties, np.float16(-1000)).astype(np.float16)
    near[0] = below[0] = 254
    x = np.stack([ties, near, below, ties / 128, ties / np.float16(2.0 ** 15), -ties])
    x = np.minimum(x, np.float16(254))
    q, _ = _quantize(x)
    np.testing.assert_array_equal(q, R.rows8(x)[0])
    # Rows that hold a NaN or an infinity: a NaN step, codes 0; the rows beside them are untouched.
    y = np.random.default_rng(0).standard_normal((6, 700)).astype(np.float16)
    y[1, 3], y[3, 699], y[4, 0] = np.nan, np.inf, -np.inf
    q, s = _quantize(y)
    wq, ws = R.rows8(y)
    np.testing.assert_array_equal(q, wq)
    np.testing.assert_array_equal(np.isnan(s), [False, True, False, True, True, False])
    # The largest and the smallest magnitudes.
    z = np.zeros((3, 16), np.float16)
    z[0, 5], z[1, 5], z[2] = 65504, np.float16(6e-8), np.float16(6e-8)
    z[0, 6] = -32752
    np.testing.assert_array_equal(_quantize(z)[0], R.rows8(z)[0])


def _norm(x, r, w, eps):
    m, k = r.shape
    q, s = np.full((m, k), 99, np.int8), np.zeros(m, np.float32)
    if x is None:
        out = run("rmsnorm", [r, w, q, s], [T.F32(eps)], [0, 2, 3])
        return out[0], out[2], out[3]
    out = run("add_rmsnorm", [x, r, w, q, s], [T.F32(eps)], [1, 3, 4])
    return out[1], out[3], out[4]


def _check_norm(x, r, w, eps=1e-5):
    got_r, q, s = _norm(x, r, w, eps)
    want_r = r if x is None else r + x.astype(np.float32)
    np.testing.assert_array_equal(got_r, want_r)
    y = want_r.astype(np.float64) * w.astype(np.float64)
    wq, ws = R.rows8(y)
    rms = np.sqrt((want_r.astype(np.float64) ** 2).mean(axis=1) + float(np.float32(eps)))
    np.testing.assert_array_equal(q, wq)
    np.testing.assert_allclose(s, ws / rms, rtol=1.01 * F)  # (f64 throughout, rounded once)


@pytest.mark.parametrize("add", [True, False])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 64), (9, 511), (4, 1000), (7, 1024), (32, 2048), (3, 2049), (5, 4096),
                                 (2, 4099), (2, 8192), (3, 10001), (1, 16390)])
def test_rmsnorm_rows(m, k, add):
    _say("rmsnorm", m, k, add)
    rng = np.random.default_rng(m * 7919 + k)
    r = (rng.standard_normal((m, k)) * rng.choice([1e-3, 1.0, 300.0], (m, 1))).astype(np.float32)
    x = rng.standard_normal((m, k)).astype(np.float16) if add else None
    w = (1 + 0.2 * rng.standard_normal(k)).astype(np.float16)
    if m > 2:
        r[1] = 0
        if add:
            x[1] = 0
    _check_norm(x, r, w)


def test_rmsnorm_ties_and_special_values():
    _say("rmsnorm ties")
    k = 509
    r = np.stack([np.arange(-254, 255), np.arange(-254, 255) * 3.0, np.arange(-254, 255) / 1024]).astype(np.float32)
    _check_norm(None, r, np.ones(k, np.float16))
    _check_norm(np.full((3, k), 0.5, np.float16), r - np.float32(0.5), np.full(k, 3, np.float16))
    # Squares past f32's range: the sums are f64.
    big = np.random.default_rng(5).standard_normal((2, k)).astype(np.float32) * np.float32(1e25)
    _check_norm(None, big, np.ones(k, np.float16))
    r = np.random.default_rng(1).standard_normal((5, 777)).astype(np.float32)
    x = np.zeros((5, 777), np.float16)
    r[0, 3], r[2, 776], x[3, 5] = np.nan, np.inf, -np.inf
    w = np.ones(777, np.float16)
    got_r, q, s = _norm(x, r, w, 1e-5)
    np.testing.assert_array_equal(got_r, r + x)
    np.testing.assert_array_equal(np.isnan(s), [True, False, True, True, False])
    assert not q[[0, 2, 3]].any()
    np.testing.assert_array_equal(q[[1, 4]], R.rows8(r[[1, 4]])[0])
    # A weight that is NaN spoils every row.
    w[7] = np.nan
    assert np.isnan(_norm(None, r[[1, 4]], w, 1e-5)[2]).all()


# ---------------------------------------------------------------- 8-bit products

def _rows(rng, m, k):
    x = rng.integers(-128, 128, (m, k)).astype(np.int8)
    return x, rng.uniform(0.2, 2.0, m).astype(np.float32) / 1000


PRODUCTS = [(1, 1, 1), (1, 16, 8), (3, 5, 7), (2, 96, 64), (1, 2560, 2048), (5, 100, 130), (16, 64, 128), (17, 200, 144),
            (32, 2048, 5632), (33, 130, 2048), (64, 520, 1024), (65, 70, 96), (100, 90, 70), (128, 256, 256),
            (130, 333, 1000), (200, 1376, 1001), (256, 2048, 2048), (300, 257, 2000), (513, 640, 128),
            (777, 1155, 1001), (1024, 1024, 80), (1100, 2100, 272), (2048, 4096, 192), (63, 64, 11008), (4, 40, 16400)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear_bits(m, n, k):
    # The sums are whole numbers, so Y's bits follow from three roundings.
    _say("linear", m, n, k)
    rng = np.random.default_rng(m * 31 + n * 17 + k)
    (x, sx), (w, sw) = _rows(rng, m, k), _rows(rng, n, k)
    y = run("linear", [x, sx, w, sw, np.full((m, n), 7, np.float16)], outputs=[4])[4]
    np.testing.assert_array_equal(y.view(np.uint16), R.product(x, sx, w, sw).astype(np.float16).view(np.uint16))


def _check_gate_up(rng, m, f, k):
    (x, sx), (wg, sg), (wu, su) = _rows(rng, m, k), _rows(rng, f, k), _rows(rng, f, k)
    sx = sx * np.float32(400 / np.sqrt(k))
    y = run("gate_up", [x, sx, wg, sg, wu, su, np.full((m, f), 7, np.float16)], outputs=[6])[6].astype(np.float64)
    g, u = (R.product(x, sx, ww, ss).astype(np.float64) for ww, ss in ((wg, sg), (wu, su)))
    want = g / (1 + np.exp(-g)) * u
    # f16's half step, and g, u, exp2 of a product rounded once (|g| log2(e) half-steps), reciprocal and products in f32.
    tol = H * np.abs(want) + (16 + 4 * np.abs(g)) * F * np.abs(want) + 2.0 ** -25
    assert (np.abs(y - want) <= tol).all(), np.abs(y - want).max()


@pytest.mark.parametrize("m,f,k", [(1, 1, 1), (1, 128, 64), (3, 5, 7), (1, 5632, 2048), (7, 333, 256), (16, 48, 128),
                                   (32, 5632, 2048), (33, 72, 1040), (64, 4000, 1024), (65, 70, 96), (100, 90, 70),
                                   (213, 704, 2048), (300, 257, 2001), (512, 1408, 512), (1024, 2048, 64), (63, 24, 11008)])
def test_gate_up(m, f, k):
    _say("gate_up", m, f, k)
    _check_gate_up(np.random.default_rng(m + f + k), m, f, k)


def test_products_of_extreme_rows():
    _say("products, extreme rows")
    # The longest rows, every product 2^14: the sum reaches 2^31 - 2^14.
    k = 131071
    x = np.full((3, k), -128, np.int8)
    w = np.full((17, k), -128, np.int8)
    one = np.float32(2.0 ** -20)
    y = run("linear", [x, np.full(3, one), w, np.ones(17, np.float32), np.zeros((3, 17), np.float16)], outputs=[4])[4]
    np.testing.assert_array_equal(y, np.full((3, 17), k * 2.0 ** -6, np.float64).astype(np.float16))
    # No columns: sums of nothing. A NaN step spoils its row or channel alone; an overflow is an infinity.
    y = run("linear", [np.zeros((3, 0), np.int8), np.ones(3, np.float32), np.zeros((5, 0), np.int8), np.ones(5, np.float32),
                       np.full((3, 5), 9, np.float16)], outputs=[4])[4]
    np.testing.assert_array_equal(y, np.zeros((3, 5)))
    rng = np.random.default_rng(3)
    for m in (5, 130):
        (x, sx), (w, sw) = _rows(rng, m, 128), _rows(rng, 70, 128)
        x[1] = w[4] = 0
        sx[1], sw[4], sw[6] = np.nan, np.nan, 1e30
        y = run("linear", [x, sx, w, sw, np.zeros((m, 70), np.float16)], outputs=[4])[4]
        with np.errstate(over="ignore"):
            want = R.product(x, sx, w, sw).astype(np.float16)
        assert np.isnan(y[1]).all() and np.isnan(y[:, 4]).all()
        np.testing.assert_array_equal(y, want)


@pytest.mark.parametrize("m,n,k", [(70, 2300, 1000), (300, 1600, 4095), (5, 48, 2001)])
def test_linear_at_any_alignment(m, n, k):
    # Operands that begin at odd addresses, and Y at an odd f16: the bits are those of aligned ones.
    _say("linear unaligned", m, n, k)
    rng = np.random.default_rng(m + n + k)
    (x, sx), (w, sw) = _rows(rng, m, k), _rows(rng, n, k)
    want = R.product(x, sx, w, sw).astype(np.float16)
    kern = T.kernel("quant", "linear", [x.shape, sx.shape, w.shape, sw.shape, (m, n)])
    for off in (1, 4, 16):
        bx, bw, by = T.alloc(x.nbytes + 32), T.alloc(w.nbytes + 32), T.alloc(2 * m * n + 64)
        bsx, bsw = T.tensor(sx), T.tensor(sw)
        T.write(bx, off, x)
        T.write(bw, off, w)
        T.launch(kern, [T.Buf(bx.ptr + off, x.nbytes), bsx, T.Buf(bw.ptr + off, w.nbytes), bsw, T.Buf(by.ptr + 2, 2 * m * n)])
        got = T.read(by, 0, 2 * m * n + 64).view(np.float16)
        np.testing.assert_array_equal(got[1:1 + m * n].reshape(m, n).view(np.uint16), want.view(np.uint16))
        assert not got[0] and not got[1 + m * n:].any()  # nothing beside Y
        for b in (bx, bw, by, bsx, bsw):
            T.free(b)


@pytest.mark.parametrize("m,f,k,launches", [(70, 300, 1001, 1), (9, 40, 2048, 1), (1000, 1155, 1001, 2), (40, 33, 13, 1)])
def test_gate_up_at_any_alignment(m, f, k, launches):
    # Operands that begin at odd addresses, each at another, give the bits of aligned ones; with one column of Wu spoilt by
    # its step, and a graph that says whether rows are copied first.
    _say("gate_up unaligned", m, f, k)
    rng = np.random.default_rng(m + f + k)
    _check_gate_up(rng, m, f, k)
    (x, sx), (wg, sg), (wu, su) = _rows(rng, m, k), _rows(rng, f, k), _rows(rng, f, k)
    su[f // 2] = np.nan
    want = run("gate_up", [x, sx, wg, sg, wu, su, np.full((m, f), 7, np.float16)], outputs=[6])[6]
    assert np.isnan(want[:, f // 2]).all() and np.isnan(want).sum() == m
    kern = T.kernel("quant", "gate_up", [x.shape, sx.shape, wg.shape, sg.shape, wu.shape, su.shape, (m, f)])
    for offs in ((1, 2, 3), (15, 0, 8)):
        bufs = [T.alloc(v.nbytes + 32) for v in (x, wg, wu)]
        bsx, bsg, bsu, by = T.tensor(sx), T.tensor(sg), T.tensor(su), T.alloc(2 * m * f + 64)
        for b, v, o in zip(bufs, (x, wg, wu), offs):
            T.write(b, o, v)
        bx, bg, bu = (T.Buf(b.ptr + o, v.nbytes) for b, v, o in zip(bufs, (x, wg, wu), offs))
        T.capture_begin()
        T.launch(kern, [bx, bsx, bg, bsg, bu, bsu, T.Buf(by.ptr + 2, 2 * m * f)])
        graph = T.capture_end()
        assert T.graph_nodes(graph)["kernel"] == launches
        for _ in range(2):
            T.replay(graph)
            got = T.read(by, 0, 2 * m * f + 64).view(np.float16)
            np.testing.assert_array_equal(got[1:1 + m * f].reshape(m, f).view(np.uint16), want.view(np.uint16))
            assert not got[0] and not got[1 + m * f:].any()
        for b in (*bufs, bsx, bsg, bsu, by):
            T.free(b)


def test_empty_sizes_launch_and_write_nothing():
    _say("empty sizes")
    pool = [(2, 2, 16, 32), (2, 2, 1, 32, 16), (2, 2, 16, 2), (2, 2, 16, 2)]
    cases = [("quantize", [(0, 64), (0, 64), (0,)], 0), ("rmsnorm", [(0, 64), (64,), (0, 64), (0,)], 1),
             ("add_rmsnorm", [(0, 64), (0, 64), (64,), (0, 64), (0,)], 1), ("linear", [(0, 64), (0,), (5, 64), (5,), (0, 5)], 0),
             ("linear", [(5, 64), (5,), (0, 64), (0,), (5, 0)], 0), ("linear", [(0, 7), (0,), (5, 7), (5,), (0, 5)], 0),
             ("gate_up", [(0, 64), (0,), (5, 64), (5,), (5, 64), (5,), (0, 5)], 0),
             ("gate_up", [(3, 64), (3,), (0, 64), (0,), (0, 64), (0,), (3, 0)], 0),
             ("kv_write", [(0, 256), (0,), (0,), (9, 32), (9, 32), *pool, (0, 2, 64), (0, 2, 64)], 0),
             ("decode_attention", [(0, 4, 64), *pool, (0, 3), (0,), (0, 4, 64)], 1)]
    for name, shapes, scalars in cases:
        bufs = [T.alloc(4 * max(1, int(np.prod(s)))) for s in shapes]
        for b in bufs:
            T.write(b, 0, np.full(b.bytes, 0x5a, np.uint8))
        T.launch(T.kernel("quant", name, shapes), bufs + [T.F32(1.0)] * scalars)
        for b in bufs:
            assert (T.read(b, 0, b.bytes) == 0x5a).all(), name
            T.free(b)
    # Rows of no columns have the step 0; tables of no pages, and a pool that none reads, give NaN.
    out = run("quantize", [np.zeros((3, 0), np.float16), np.zeros((3, 0), np.int8), np.ones(3, np.float32)], outputs=[2])
    assert not out[2].any()
    for d in (16, 64):
        case = _attention_case(np.random.default_rng(d), 2, 4, 2, d, 16, [20, 3])
        case[5] = np.zeros((2, 0), np.int32)
        assert np.isnan(_attend(*case)).all()


@pytest.mark.parametrize("m", [3, 200])
def test_linear_of_weights_past_4_gib(m):
    # 40000 rows of 131056: the last rows' offsets pass 32 bits. Zeros but for three rows.
    _say("linear past 4 GiB", m)
    n, k = 40000, 131056
    rng = np.random.default_rng(m)
    (x, sx), (rows, srows) = _rows(rng, m, k), _rows(rng, 3, k)
    at, sw = np.array([0, 32800, n - 1]), np.ones(n, np.float32)
    sw[at] = srows
    bw, by = T.alloc(n * k), T.alloc(2 * m * n)
    for i, r in zip(at, rows):
        T.write(bw, int(i) * k, r)
    bx, bsx, bsw = T.tensor(x), T.tensor(sx), T.tensor(sw)
    T.launch(T.kernel("quant", "linear", [x.shape, sx.shape, (n, k), sw.shape, (m, n)]), [bx, bsx, bw, bsw, by])
    y = T.read_array(by, np.float16, (m, n))
    np.testing.assert_array_equal(y[:, at].view(np.uint16), R.product(x, sx, rows, srows).astype(np.float16).view(np.uint16))
    y[:, at] = 0
    assert not y.any()
    for b in (bw, by, bx, bsx, bsw):
        T.free(b)


@pytest.mark.parametrize("m,n,k,launches", [(400, 2100, 1001, 1), (1500, 2100, 2001, 2)])
def test_products_share_a_handle_in_a_graph(m, n, k, launches):
    # Two products of one handle in a graph, replayed with eager launches of other operands between; the second size's
    # rows are copied first, into the handle's scratch.
    _say("linear twice in a graph", m, n, k)
    rng = np.random.default_rng(4)
    kern, sets = T.kernel("quant", "linear", [(m, k), (m,), (n, k), (n,), (m, n)]), []
    for _ in range(3):
        (x, sx), (w, sw) = _rows(rng, m, k), _rows(rng, n, k)
        sets.append(([T.tensor(v) for v in (x, sx, w, sw)] + [T.alloc(2 * m * n)], R.product(x, sx, w, sw).astype(np.float16)))
    T.capture_begin()
    for args, _ in sets[:2]:
        T.launch(kern, args)
    graph = T.capture_end()
    assert T.graph_nodes(graph) == {"kernel": 2 * launches, "memset": 0, "memcpy": 0, "other": 0}
    for _ in range(3):
        for args, _ in sets:
            T.fill_nan(args[4])
        T.launch(kern, sets[2][0])
        T.replay(graph)
        T.launch(kern, sets[2][0])
        for args, want in sets:
            np.testing.assert_array_equal(T.read_array(args[4], np.float16, (m, n)).view(np.uint16), want.view(np.uint16))
    for args, _ in sets:
        for b in args:
            T.free(b)


@pytest.mark.parametrize("name", ["quantize", "rmsnorm"])
def test_rows_end_where_they_end(name):
    # Codes at odd addresses, bytes before and after untouched; rows of every tail length.
    _say("row guards", name)
    rng = np.random.default_rng(8)
    for m, k in ((3, 9), (2, 63), (5, 517), (2, 1031), (2, 2055), (1, 4101), (2, 6150), (1, 9001), (1, 16391), (1, 33001)):
        x = rng.standard_normal((m, k)).astype(np.float16)
        q, s = T.tensor(np.full(m * k + 64, 99, np.int8)), T.tensor(np.full(m + 2, 7, np.float32))
        out, sc = T.Buf(q.ptr + 33, m * k), T.Buf(s.ptr + 4, 4 * m)
        if name == "quantize":
            bufs = [T.tensor(x)]
            T.launch(T.kernel("quant", name, [(m, k), (m, k), (m,)]), bufs + [out, sc])
        else:
            bufs = [T.tensor(x.astype(np.float32)), T.tensor(np.ones(k, np.float16))]
            T.launch(T.kernel("quant", name, [(m, k), (k,), (m, k), (m,)]), bufs + [out, sc, T.F32(1e-5)])
        got, gs = T.read(q, 0, m * k + 64).view(np.int8), T.read_array(s, np.float32, (m + 2,))
        np.testing.assert_array_equal(got[33:33 + m * k].reshape(m, k), R.rows8(x)[0])
        assert (got[:33] == 99).all() and (got[33 + m * k:] == 99).all() and gs[0] == 7 and gs[-1] == 7
        for b in bufs + [q, s]:
            T.free(b)


# ---------------------------------------------------------------- the 4-bit cache

def _write_case(rng, t, h, g, d, p, pages, w_extra=0):
    w = (h + 2 * g) * d + w_extra
    qkv = rng.standard_normal((t, w)).astype(np.float16)
    pos = rng.integers(0, 300, t).astype(np.int32)
    slot = rng.permutation(pages * p)[:t].astype(np.int32)
    a = rng.uniform(0, 6.28, (300, d // 2))
    kn, vn, ks, vs = R.cached(rng, pages, g, p, d)
    return [qkv, pos, slot, np.cos(a).astype(np.float32), np.sin(a).astype(np.float32), R.pack_k(kn), R.pack_v(vn), ks, vs,
            np.full((t, g, d), 7, np.float16), np.full((t, g, d), 7, np.float16)], (kn, vn)


def _check_write(case, codes):
    """K is the rotation with its three roundings (and so within a step of llm/kv_write's), V the values' bits; the
    cache holds their 4-bit forms, and elsewhere what it held."""
    qkv, pos, slot, cos, sin, kc, vc, ks, vs, k, v = case
    kn, vn = (c.copy() for c in codes)
    t, g, d = k.shape
    pages, _, p, _ = kc.shape
    got = run("kv_write", case, outputs=range(5, 11))
    kv = qkv[:, qkv.shape[1] - 2 * g * d:].reshape(t, 2, g, d)
    there = ((pos >= 0) & (pos < len(cos)))[:, None, None]
    c, s = (np.where(there, x[np.clip(pos, 0, len(cos) - 1)][:, None].astype(np.float64), 0.0) for x in (cos, sin))
    x1, x2 = kv[:, 0, :, :d // 2].astype(np.float64), kv[:, 0, :, d // 2:].astype(np.float64)
    with np.errstate(invalid="ignore"):
        p2, p1 = ((x * s).astype(np.float32).astype(np.float64) for x in (x2, x1))
        want_k = np.concatenate([x1 * c - p2, x2 * c + p1], -1).astype(np.float32).astype(np.float16)
    np.testing.assert_array_equal(got[9], want_k)
    np.testing.assert_array_equal(got[10].view(np.uint16), kv[:, 1].view(np.uint16))
    wide = np.zeros((pages * p, g, d), np.float16)
    ref = T.run("llm", "kv_write", [qkv, pos, slot, cos, sin, wide, wide, k, v], outputs=[7, 8])
    # (llm/kv_write may round the multiply-add to f16 at once: a step apart where f32 rounds it onto a tie)
    np.testing.assert_allclose(ref[7].astype(np.float64), want_k.astype(np.float64), rtol=2 * H, atol=2.0 ** -24)
    np.testing.assert_array_equal(got[10].view(np.uint16), ref[8].view(np.uint16))
    ks, vs = ks.copy(), vs.copy()
    for x, n, pair in ((got[9], kn, ks), (got[10], vn, vs)):
        cn, cp = R.heads4(x)
        for i in range(t):  # (in order: of rows with one slot the last is kept)
            if 0 <= slot[i] < pages * p:
                n[slot[i] // p, :, slot[i] % p], pair[slot[i] // p, :, slot[i] % p] = cn[i], cp[i]
    np.testing.assert_array_equal(got[5], R.pack_k(kn))
    np.testing.assert_array_equal(got[6], R.pack_v(vn))
    np.testing.assert_array_equal(got[7], ks)
    np.testing.assert_array_equal(got[8], vs)


@pytest.mark.parametrize("t,h,g,d,p", [(1, 4, 2, 16, 16), (5, 8, 4, 32, 16), (64, 32, 4, 64, 32), (37, 32, 8, 128, 16),
                                       (3, 16, 16, 64, 64), (300, 8, 2, 64, 16), (9, 20, 20, 128, 32), (2, 1, 1, 128, 16),
                                       (70, 3, 3, 32, 128), (11, 5, 5, 16, 32)])
def test_kv_write(t, h, g, d, p):
    _say("kv_write", t, h, g, d, p)
    rng = np.random.default_rng(t + 10 * g + d + p)
    case, codes = _write_case(rng, t, h, g, d, p, (t + p - 1) // p + 2)
    _check_write(case, codes)


@pytest.mark.parametrize("g,d", [(2, 16), (4, 64), (8, 128)])
def test_kv_write_special_rows(g, d):
    _say("kv_write special", g, d)
    rng = np.random.default_rng(d)
    t, p = 40, 16
    case, codes = _write_case(rng, t, 2 * g, g, d, p, 4, w_extra=2)
    qkv, pos, slot = case[0], case[1], case[2]
    lo = qkv.shape[1] - g * d  # the values' first column
    slot[3], slot[7], slot[8] = -1, 4 * p, 2 ** 31 - 1        # dropped
    slot[10] = slot[20] = slot[39] = slot[0]                   # one slot four times: the last row's
    pos[5], pos[6] = -1, 300                                   # outside the tables: keys 0
    qkv[11, lo:lo + d] = 3.25                                  # a constant head: step 0
    qkv[12, lo:lo + d] = 0
    qkv[13, lo + 1], qkv[14, lo + d - 1] = np.nan, np.inf      # spoilt heads
    qkv[15, lo:lo + d] = np.where(np.arange(d) % 2, 65504, -65504)
    qkv[16, lo:lo + d] = np.arange(d) % 16 * 0.5               # codes without a rounding
    qkv[17, lo:lo + d] = np.arange(d) % 31                     # whole and half codes: ties
    qkv[18, lo:lo + d] = np.float16(6e-8) * (np.arange(d) % 3)  # subnormal
    _check_write(case, codes)


def _attend(q, kn, vn, ks, vs, table, lens, scale):
    arrays = [q, R.pack_k(kn), R.pack_v(vn), ks, vs, table, lens, np.full_like(q, 7)]
    return run("decode_attention", arrays, [T.F32(scale)], [7])[7].astype(np.float64)


def _close(got, q, kn, vn, ks, vs, table, lens, scale):
    want, mag, top = R.attention(q, kn, vn, ks, vs, table, lens, scale)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    # The output's half step; a probability's times its step, rounded to f16; f32 sums: a score's error is at
    # most (D + 8) half-steps of sum |q| (|low| + |k|), which moves a probability by as much of itself, and the sums
    # over tokens add theirs (their terms' square root; bounded by 64 here).
    d = q.shape[2]
    tol = H * np.abs(want) + mag * (H + F * (2 * (d + 8) * top + 64))
    ok = np.isnan(want) | (np.abs(got - want) <= tol + 2.0 ** -25)
    assert ok.all(), (np.abs(got - want)[~ok].max(), np.argwhere(~ok)[:5])


def _attention_case(rng, b, h, g, d, p, lens, spread=1.0, spare=3):
    lens = np.asarray(lens, np.int32)
    need = (np.maximum(lens, 0) + p - 1) // p
    mp = max(1, int(need.max()))
    pages = int(need.sum()) + spare
    perm = rng.permutation(pages).astype(np.int32)
    table, o = np.zeros((b, mp), np.int32), 0
    for i in range(b):
        table[i, :need[i]] = perm[o:o + need[i]]
        o += need[i]
    q = rng.standard_normal((b, h, d)).astype(np.float16)
    return [q, *R.cached(rng, pages, g, p, d, spread), table, lens, float(np.float32(d ** -0.5))]


ATTENTION = [(1, 4, 2, 16, 16, [1]), (2, 8, 4, 32, 16, [15, 17]), (3, 32, 4, 64, 16, [1, 16, 333]),
             (2, 32, 8, 128, 16, [63, 64]), (4, 16, 16, 64, 32, [65, 0, 31, 200]), (1, 16, 1, 128, 16, [1000]),
             (5, 8, 2, 64, 64, [5, 64, 129, 700, 2]), (1, 32, 4, 64, 16, [5000]), (2, 16, 2, 128, 32, [2111, 3]),
             (7, 4, 4, 128, 16, [1, 2, 3, 4, 255, 256, 257]), (2, 16, 1, 16, 16, [300, 40]), (1, 2, 1, 32, 128, [1500]),
             (40, 8, 8, 128, 16, list(range(1, 400, 10))), (1, 8, 1, 64, 16, [4097]), (3, 4, 2, 16, 16, [1500, 0, 300]),
             (2, 4, 1, 128, 512, [2000, 700]), (2, 8, 4, 64, 2048, [2049, 5000]), (1, 8, 8, 32, 256, [1025]),
             (300, 4, 4, 64, 16, [1100] + [5, 0, 64] * 99 + [1023, 33]), (2, 32, 2, 64, 1024, [0, 3000])]


@pytest.mark.parametrize("b,h,g,d,p,lens", ATTENTION)
def test_decode_attention(b, h, g, d, p, lens):
    _say("decode_attention", b, h, g, d, p, lens[:4])
    case = _attention_case(np.random.default_rng(b + h + d + p), b, h, g, d, p, lens)
    _close(_attend(*case), *case)


@pytest.mark.parametrize("b,h,g,d,p,most", [(70, 8, 4, 32, 16, 1100), (33, 8, 8, 64, 64, 3000), (130, 2, 2, 32, 16, 1040),
                                            (300, 1, 1, 64, 16, 1025), (512, 1, 1, 32, 32, 1100), (64, 8, 8, 32, 1024, 2048),
                                            (17, 16, 16, 32, 16, 5000)])
def test_decode_attention_of_many_ragged_sequences(b, h, g, d, p, most):
    # Batches of one to two workgroups a CU: ties, empty and negative lengths, lengths past the table; then all equal.
    _say("decode_attention ragged", b, g)
    rng = np.random.default_rng(b + g)
    lens = rng.integers(0, 60, b)
    lens[rng.integers(0, b, b // 3)] = 17
    lens[[0, b // 2, b - 1]] = most, 0, most - 1
    case = _attention_case(rng, b, h, g, d, p, lens)
    case[6][[3, 5, 8]] = -9, 2 ** 31 - 1, -2 ** 31
    _close(_attend(*case), *case)
    case[6][:] = 33
    case[5][:] = case[5][:, :1]
    _close(_attend(*case), *case)
    case[6][:] = 0
    assert np.isnan(_attend(*case)).all()


@pytest.mark.parametrize("d,h,g", [(16, 4, 2), (64, 32, 4), (128, 16, 2)])
def test_decode_attention_odd_tables(d, h, g):
    _say("decode_attention odd tables", d)
    rng = np.random.default_rng(d + 1)
    case = _attention_case(rng, 6, h, g, d, 16, [100, 0, -5, 40, 333, 90])
    q, kn, vn, ks, vs, table, lens, scale = case
    npg = len(kn)
    table[0, 2], table[3, 0], table[5, 1] = -1, npg, 2 ** 31 - 1   # pages outside the pool: zeros
    table[1:3] = -7                                                # (empty sequences read none)
    # A spoilt token past a sequence's end is not read; one inside spoils its kv head's rows.
    kn[table[0, 6], :, 4:], ks[table[0, 6], :, 4:], vs[table[0, 6], :, 4:] = 15, np.nan, np.nan
    got = _attend(*case)
    _close(got, *case)
    lens[4] = 2 ** 31 - 1                                          # past the table: its MP P tokens
    _close(_attend(*case), *case)
    vs[table[4, 1], 0, 3] = np.nan
    got = _attend(*case)
    assert np.isnan(got[4, :h // g]).all() and not np.isnan(got[4, h // g:]).any()


@pytest.mark.parametrize("d,h,g", [(64, 16, 4), (128, 8, 1), (32, 4, 2)])
def test_decode_attention_far_scores(d, h, g):
    # Scores of +-100s: the running maximum moves by much, early probabilities vanish; a far first token.
    _say("decode_attention far scores", d)
    rng = np.random.default_rng(d + 2)
    case = _attention_case(rng, 3, h, g, d, 16, [1300, 70, 513], spread=12.0)
    _close(_attend(*case), *case)
    case[0] *= np.float16(1e-3)   # and near-uniform ones, of small q
    _close(_attend(*case), *case)
    case[0][0] = 0
    _close(_attend(*case), *case)


@pytest.mark.parametrize("d,h,g", [(16, 4, 2), (32, 8, 8), (64, 16, 1), (128, 8, 1)])
def test_decode_attention_scales_and_spoilt_queries(d, h, g):
    # A negative scale turns the order over; 0 makes a mean of the values. A query that holds an infinity or a NaN
    # spoils its own head, one of the largest and smallest f16 magnitudes none.
    _say("decode_attention scales", d)
    rng = np.random.default_rng(d + 3)
    case = _attention_case(rng, 3, h, g, d, 16, [70, 1100, 9])
    for scale in (-0.25, 0.0, 1e-30):
        case[7] = float(np.float32(scale))
        _close(_attend(*case), *case)
    case[7] = 2.0 ** -20
    q = case[0]
    q[1, 1, 2] = 65504
    q[1, 1, 3:6] = np.float16(6e-8)
    _close(_attend(*case), *case)
    q[0, 0, 1], q[1, 2, d - 1], q[2, h - 1, 0] = np.inf, np.nan, -np.inf
    got = _attend(*case)
    want = np.zeros((3, h), bool)
    want[0, 0] = want[1, 2] = want[2, h - 1] = True
    np.testing.assert_array_equal(np.isnan(got), np.broadcast_to(want[:, :, None], got.shape))
    q[0, 0, 1] = q[1, 2, d - 1] = q[2, h - 1, 0] = 0
    clean = _attend(*case)
    np.testing.assert_array_equal(got[~want], clean[~want])


def test_decode_attention_refuses_a_pool_off_its_alignment():
    kern = T.kernel("quant", "decode_attention", [[1, 4, 64], [2, 2, 16, 32], [2, 2, 1, 32, 16], [2, 2, 16, 2], [2, 2, 16, 2],
                                                  [1, 2], [1], [1, 4, 64]])
    bufs = [T.alloc(n + 64) for n in (512, 2048, 2048, 256, 256, 8, 4, 512)]
    for i in (1, 2, 3, 4):
        at = [T.Buf(b.ptr + (8 if j == i else 0), b.bytes - 64) for j, b in enumerate(bufs)]
        with pytest.raises(T.TesselError, match="16-byte aligned"):
            T.launch(kern, at + [T.F32(0.125)])
    for b in bufs:
        T.free(b)


@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_decode_attention_of_a_scale_that_is_no_number(d):
    _say("decode_attention NaN scale", d)
    for lens in ([70, 9], [1100, 20]):
        case = _attention_case(np.random.default_rng(d), 2, 8, 2, d, 16, lens)
        case[7] = float("nan")
        assert np.isnan(_attend(*case)).all()


@pytest.mark.parametrize("d,h,g", [(16, 4, 2), (32, 16, 1), (64, 8, 4), (128, 8, 1)])
def test_decode_attention_small_and_large_values(d, h, g):
    # Values of 1e-5 to 6e4, alone and on neighbouring pages: probabilities keep their bits beside any step.
    _say("decode_attention values", d)
    rng = np.random.default_rng(d + 4)
    for factor in (2e-5, 1e-3, 1000.0, None):
        case = _attention_case(rng, 3, h, g, d, 16, [1300, 70, 400])
        vs = case[4].astype(np.float64)
        vs *= factor if factor else rng.choice([1e-4, 1.0, 3000.0], (len(vs), 1, 1, 1))
        case[4] = vs.astype(np.float16)
        _close(_attend(*case), *case)
    case[4][:] = np.array([-65504, 8736], np.float16)  # the widest head
    case[2] = np.minimum(case[2], 14)
    _close(_attend(*case), *case)
    case[4][:] = np.array([6e-8, 0], np.float16)       # equal values
    _close(_attend(*case), *case)


def test_a_cache_past_4_gib():
    # 600000 pages of 8 heads of 128: codes of 4.9 GB each. Tokens written to its last pages and read from there.
    _say("cache past 4 GiB")
    rng = np.random.default_rng(12)
    h, g, d, p, pages, t = 16, 8, 128, 16, 600000, 40
    kc, vc, ks, vs = (T.alloc(pages * g * p * n) for n in (d // 2, d // 2, 4, 4))
    qkv = rng.standard_normal((t, 2 * g * d)).astype(np.float16)
    where = np.array([pages - 1, 3, pages - 2], np.int32)  # tokens 0 .. 15, 16 .. 31, 32 .. 39
    slot = (where[np.arange(t) // p] * p + np.arange(t) % p).astype(np.int32)
    one, zero = np.ones((1, d // 2), np.float32), np.zeros((1, d // 2), np.float32)
    k, v, q, o = T.alloc(2 * t * g * d), T.alloc(2 * t * g * d), rng.standard_normal((1, h, d)).astype(np.float16), T.alloc(2 * h * d)
    cache = [(pages, g, p, d // 2), (pages, g, 1, d // 2, 16), (pages, g, p, 2), (pages, g, p, 2)]
    ins = [T.tensor(x) for x in (qkv, np.zeros(t, np.int32), slot, one, zero, q, where[None], np.array([t], np.int32))]
    T.launch(T.kernel("quant", "kv_write", [qkv.shape, (t,), (t,), one.shape, zero.shape, *cache, (t, g, d), (t, g, d)]),
             ins[:5] + [kc, vc, ks, vs, k, v])
    T.launch(T.kernel("quant", "decode_attention", [q.shape, *cache, (1, 3), (1,), q.shape]),
             [ins[5], kc, vc, ks, vs, ins[6], ins[7], o, T.F32(0.09)])
    x = qkv.reshape(t, 2, g, d)  # (not turned: position 0)
    kn, kp = R.heads4(x[:, 0])
    vn, vp = R.heads4(x[:, 1])
    small = [np.zeros((3, g, p, *a.shape[2:]), a.dtype) for a in (kn, vn, kp, vp)]
    for a, b in zip(small, (kn, vn, kp, vp)):
        for i in range(t):
            a[i // p, :, i % p] = b[i]
    _close(T.read_array(o, np.float16, q.shape).astype(np.float64), q, *small[:2], small[2], small[3], np.array([[0, 1, 2]]),
           np.array([t]), 0.09)
    at = ((pages - 2) * g + 5) * p * (d // 2)
    np.testing.assert_array_equal(T.read(kc, at, p * d // 2).reshape(p, -1), R.pack_k(small[0])[2, 5])
    for b in (kc, vc, ks, vs, k, v, o, *ins):
        T.free(b)


def test_decode_attention_repeats_and_replays_its_bits():
    _say("decode_attention repeat, replay")
    rng = np.random.default_rng(9)
    a, b = (_attention_case(rng, 4, 32, 8, 128, 16, lens) for lens in ([900, 3, 77, 2000], [5, 1999, 900, 1]))
    pool = [max(len(a[1]), len(b[1]))]
    # Both cases' tables over one shape, through one handle and its scratch.
    mp = max(a[5].shape[1], b[5].shape[1])
    bufs = []
    for c in (a, b):
        c[5] = np.pad(c[5], ((0, 0), (0, mp - c[5].shape[1])))
        for i in range(1, 5):
            c[i] = np.concatenate([c[i], c[i][:pool[0] - len(c[i])]])
        arrays = [c[0], R.pack_k(c[1]), R.pack_v(c[2]), c[3], c[4], c[5], c[6], np.full_like(c[0], 7)]
        bufs.append([T.tensor(x) for x in arrays])
        k = T.kernel("quant", "decode_attention", [x.shape for x in arrays])
    launches = [(k, bb + [T.F32(a[7])]) for bb in bufs]
    first = []
    for kk, args in launches:
        T.launch(kk, args)
        first.append(T.read_array(args[7], np.float16, a[0].shape))
    for c, f in zip((a, b), first):
        _close(f.astype(np.float64), *c)
    T.capture_begin()
    for kk, args in launches:
        T.launch(kk, args)
    graph = T.capture_end()
    assert T.graph_nodes(graph)["memset"] == 0 and T.graph_nodes(graph)["memcpy"] == 0
    for _ in range(4):
        for args in (launches[0][1], launches[1][1]):
            T.fill_nan(args[7])
        T.replay(graph)
        T.launch(*launches[0])
        for (kk, args), f in zip(launches, first):
            np.testing.assert_array_equal(T.read_array(args[7], np.float16, a[0].shape).view(np.uint16), f.view(np.uint16))
    for bb in bufs:
        for x in bb:
            T.free(x)


# ---------------------------------------------------------------- together

def test_a_decode_step_in_8_and_4_bits():
    """A decoder layer for a batch of single tokens, as a program runs it: weights quantised on the GPU, the
    norm's codes into QKV, the cache written and read, the output and MLP projections, captured and replayed."""
    _say("decode step")
    rng = np.random.default_rng(11)
    t, h, g, d, dm, f, p, pages = 5, 8, 2, 64, 512, 704, 16, 24
    w = (h + 2 * g) * d
    lens = np.array([1, 17, 40, 64, 33], np.int32)
    perm, table, o = rng.permutation(pages).astype(np.int32), np.zeros((t, 5), np.int32), 0
    for i, n in enumerate((lens + p - 1) // p):
        table[i, :n] = perm[o:o + n]
        o += n
    slot = np.array([table[i, (n - 1) // p] * p + (n - 1) % p for i, n in enumerate(lens)], np.int32)
    weights = {n: (rng.standard_normal(s) / np.sqrt(s[1])).astype(np.float16)
               for n, s in (("qkv", (w, dm)), ("o", (dm, h * d)), ("g", (f, dm)), ("u", (f, dm)), ("d", (dm, f)))}
    wn = (1 + 0.1 * rng.standard_normal(dm)).astype(np.float16)
    r0, x0 = rng.standard_normal((t, dm)).astype(np.float32), rng.standard_normal((t, dm)).astype(np.float16)
    pos = (lens - 1).astype(np.int32)
    a = np.arange(80)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    kn, vn, ks, vs = R.cached(rng, pages, g, p, d)
    scale = float(np.float32(d ** -0.5))

    buf, shape, dt = {}, {}, {}

    def put(name, x):
        buf[name], shape[name], dt[name] = T.tensor(x), x.shape, x.dtype

    def get(name):
        return T.read_array(buf[name], dt[name], shape[name])

    def call(file, name, names, scalars=()):
        k = T.kernel(file, name, [shape[n] for n in names])
        return k, [buf[n] for n in names] + [T.F32(s) for s in scalars]

    for n, x in weights.items():
        put("w_" + n, x)
        put("q_" + n, np.zeros(x.shape, np.int8))
        put("s_" + n, np.zeros(len(x), np.float32))
        T.launch(*call("quant", "quantize", ["w_" + n, "q_" + n, "s_" + n]))
    for n, x in (("x", x0), ("r", r0), ("wn", wn), ("hq", np.zeros((t, dm), np.int8)), ("hs", np.zeros(t, np.float32)),
                 ("qkv", np.zeros((t, w), np.float16)), ("pos", pos), ("slot", slot), ("c", np.cos(a).astype(np.float32)),
                 ("s", np.sin(a).astype(np.float32)), ("kc", R.pack_k(kn)), ("vc", R.pack_v(vn)), ("ks", ks), ("vs", vs),
                 ("q", np.zeros((t, h, d), np.float16)), ("k", np.zeros((t, g, d), np.float16)),
                 ("v", np.zeros((t, g, d), np.float16)), ("table", table), ("lens", lens),
                 ("att", np.zeros((t, h, d), np.float16)), ("aq", np.zeros((t, h * d), np.int8)),
                 ("as", np.zeros(t, np.float32)), ("ox", np.zeros((t, dm), np.float16)), ("mlp", np.zeros((t, f), np.float16)),
                 ("mq", np.zeros((t, f), np.int8)), ("ms", np.zeros(t, np.float32)), ("dx", np.zeros((t, dm), np.float16))):
        put(n, x)
    buf["att2"], shape["att2"], dt["att2"] = buf["att"], (t, h * d), np.dtype(np.float16)
    step = [call("quant", "add_rmsnorm", ["x", "r", "wn", "hq", "hs"], [1e-5]),
            call("quant", "linear", ["hq", "hs", "q_qkv", "s_qkv", "qkv"]),
            call("llm", "rope_q", ["qkv", "pos", "c", "s", "q"]),
            call("quant", "kv_write", ["qkv", "pos", "slot", "c", "s", "kc", "vc", "ks", "vs", "k", "v"]),
            call("quant", "decode_attention", ["q", "kc", "vc", "ks", "vs", "table", "lens", "att"], [scale]),
            call("quant", "quantize", ["att2", "aq", "as"]),
            call("quant", "linear", ["aq", "as", "q_o", "s_o", "ox"]),
            call("quant", "add_rmsnorm", ["ox", "r", "wn", "hq", "hs"], [1e-5]),
            call("quant", "gate_up", ["hq", "hs", "q_g", "s_g", "q_u", "s_u", "mlp"]),
            call("quant", "quantize", ["mlp", "mq", "ms"]),
            call("quant", "linear", ["mq", "ms", "q_d", "s_d", "dx"])]
    for s in step:
        T.launch(*s)
    names = ("r", "hq", "hs", "qkv", "q", "k", "v", "kc", "vc", "ks", "vs", "att", "aq", "ox", "mlp", "mq", "dx")
    got = {n: get(n) for n in names}

    # Each stage against its plain form on what the stage before it wrote.
    qw = {n: R.rows8(x) for n, x in weights.items()}
    for n, (codes, _) in qw.items():
        np.testing.assert_array_equal(get("q_" + n), codes)
    r1 = r0 + x0.astype(np.float32)
    hq, _ = R.rows8(r1.astype(np.float64) * wn)
    hs = (np.abs(r1.astype(np.float64) * wn).max(1) / 127 / np.sqrt((r1.astype(np.float64) ** 2).mean(1) + float(np.float32(1e-5))))
    qkv = R.product(hq, hs.astype(np.float32), qw["qkv"][0], get("s_qkv")).astype(np.float16)
    # (the step's last bit is its own: within two f16 steps)
    np.testing.assert_allclose(got["qkv"].astype(np.float64), qkv.astype(np.float64), rtol=4 * H, atol=1e-7)
    for x, n, pair, codes_at, pairs_at in ((got["k"], kn, ks, "kc", "ks"), (got["v"], vn, vs, "vc", "vs")):
        cn, cp = R.heads4(x)
        for i in range(t):
            n[slot[i] // p, :, slot[i] % p], pair[slot[i] // p, :, slot[i] % p] = cn[i], cp[i]
        np.testing.assert_array_equal(got[codes_at], R.pack_k(n) if codes_at == "kc" else R.pack_v(n))
        np.testing.assert_array_equal(got[pairs_at], pair)
    _close(got["att"].astype(np.float64), got["q"], kn, vn, ks, vs, table, lens, scale)
    aq, as_ = R.rows8(got["att"].reshape(t, -1))
    np.testing.assert_array_equal(got["aq"], aq)
    np.testing.assert_array_equal(got["ox"], R.product(aq, get("as"), qw["o"][0], get("s_o")).astype(np.float16))
    r2 = r1 + got["ox"].astype(np.float32)
    np.testing.assert_array_equal(got["r"], r2)
    np.testing.assert_array_equal(got["hq"], R.rows8(r2.astype(np.float64) * wn)[0])
    np.testing.assert_array_equal(got["mq"], R.rows8(got["mlp"])[0])
    np.testing.assert_array_equal(got["dx"], R.product(got["mq"], get("ms"), qw["d"][0], get("s_d")).astype(np.float16))
    T.capture_begin()
    for s in step:
        T.launch(*s)
    graph = T.capture_end()
    assert T.graph_nodes(graph)["memset"] == 0
    for _ in range(3):
        T.write(buf["r"], 0, r0)
        for n in ("att", "dx", "mlp", "qkv"):
            T.fill_nan(buf[n])
        T.replay(graph)
        for n in names:
            np.testing.assert_array_equal(get(n), got[n])
        T.write(buf["r"], 0, r0)
        for s in step:
            T.launch(*s)
        np.testing.assert_array_equal(get("dx"), got["dx"])
    for b in set(buf.values()):
        T.free(b)
