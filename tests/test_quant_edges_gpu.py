"""Calls of the quant kernels that their documents allow: operands that begin at any element, more rows than one launch holds
workgroups for, products of very many rows or columns."""

import numpy as np
import pytest

import tessel_amd as T
from tests import quant_refs as R
from tests.test_quant_gpu import F, _attention_case, _rows, _say, _write_case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _open(gpu):
    yield


def _place(x, elements):
    """x on the device, `elements` of its own past a multiple of 16 bytes, 0x5a around it."""
    off = elements * x.itemsize
    b = T.alloc(x.nbytes + off + 64)
    T.write(b, 0, np.full(b.bytes, 0x5a, np.uint8))
    T.write(b, off, np.ascontiguousarray(x))
    return T.Buf(b.ptr + off, x.nbytes), b, off


def _run(name, arrays, elements, scalars=()):
    """Launches with array i `elements[i]` elements off; the arrays read back, after a look at what lies around them."""
    k = T.kernel("quant", name, [x.shape for x in arrays])
    placed = [_place(x, e) for x, e in zip(arrays, elements)]
    T.launch(k, [p[0] for p in placed] + [T.F32(s) for s in scalars])
    out = []
    for x, (_, b, off) in zip(arrays, placed):
        raw = T.read(b, 0, b.bytes)
        assert (raw[:off] == 0x5a).all() and (raw[off + x.nbytes:] == 0x5a).all()
        out.append(raw[off:off + x.nbytes].view(x.dtype).reshape(x.shape))
        T.free(b)
    return out


@pytest.mark.parametrize("h,g,d,p,lens", [(8, 2, 64, 16, [333, 20]), (4, 4, 128, 32, [1500, 2]), (4, 1, 32, 16, [70, 64]),
                                          (4, 2, 16, 16, [300, 5])])
def test_attention_of_queries_and_tables_at_any_element(h, g, d, p, lens):
    _say("attention at any element", h, g, d)
    q, kn, vn, ks, vs, table, lens, scale = _attention_case(np.random.default_rng(d), 2, h, g, d, p, lens)
    arrays = [q, R.pack_k(kn), R.pack_v(vn), ks, vs, table, lens, np.full_like(q, 7)]
    outs = [_run("decode_attention", arrays, [e, 0, 0, 0, 0, e, e, e], [scale])[7].view(np.uint16) for e in (0, 1, 3)]
    np.testing.assert_array_equal(outs[0], outs[1])
    np.testing.assert_array_equal(outs[0], outs[2])


@pytest.mark.parametrize("t,h,g,d,p,extra", [(37, 4, 2, 16, 16, 1), (20, 4, 4, 64, 32, 3), (5, 8, 8, 128, 16, 0), (9, 2, 1, 32, 16, 1)])
def test_cache_writes_at_any_element(t, h, g, d, p, extra):
    _say("kv_write at any element", t, g, d)
    case, _ = _write_case(np.random.default_rng(d + t), t, h, g, d, p, (t + p - 1) // p + 2, extra)
    ref = _run("kv_write", case, [0] * 11)
    for e in (1, 3):
        for a, b in zip(ref, _run("kv_write", case, [e] * 11)):
            np.testing.assert_array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("k", [7, 64, 1001, 2100, 5000])
def test_norms_at_any_element(k):
    _say("norms at any element", k)
    rng = np.random.default_rng(k)
    x, r = rng.standard_normal((3, k)).astype(np.float16), rng.standard_normal((3, k)).astype(np.float32)
    w, q, s = (1 + 0.1 * rng.standard_normal(k)).astype(np.float16), np.zeros((3, k), np.int8), np.zeros(3, np.float32)
    ref = _run("add_rmsnorm", [x, r, w, q, s], [0] * 5, [1e-5])
    np.testing.assert_array_equal(ref[3], R.rows8((r + x).astype(np.float64) * w)[0])
    for e in ([1, 1, 1, 1, 1], [3, 2, 5, 7, 3]):
        for a, b in zip(ref, _run("add_rmsnorm", [x, r, w, q, s], e, [1e-5])):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("m,k", [(4_300_001, 9), (1_100_003, 1100)])
def test_more_rows_than_workgroups(m, k):
    # (2^20 workgroups of four rows, and of one.)
    _say("rows past the grid", m, k)
    x = np.random.default_rng(k).standard_normal((min(m, 65521), k)).astype(np.float16)
    x = np.resize(x, (m, k))
    out = T.run("quant", "quantize", [x, np.zeros((m, k), np.int8), np.zeros(m, np.float32)], outputs=[1, 2])
    wq, ws = R.rows8(x[:65521])
    for i in range(0, m, 65521):
        n = min(65521, m - i)
        np.testing.assert_array_equal(out[1][i:i + n], wq[:n])
        np.testing.assert_allclose(out[2][i:i + n], ws[:n], rtol=2 * F)


def test_more_norms_than_workgroups():
    _say("norms past the grid")
    m, k, n = 4_200_007, 16, 65521
    r = np.resize(np.random.default_rng(1).standard_normal((n, k)).astype(np.float32), (m, k))
    w = np.ones(k, np.float16)
    out = T.run("quant", "rmsnorm", [r, w, np.zeros((m, k), np.int8), np.zeros(m, np.float32)], [T.F32(1e-5)], outputs=[2, 3])
    wq, _ = R.rows8(r[:n])
    for i in range(0, m, n):
        np.testing.assert_array_equal(out[2][i:i + n], wq[:min(n, m - i)])
    np.testing.assert_array_equal(out[3], np.resize(out[3][:n], m))


@pytest.mark.parametrize("m,n,k", [(1_000_003, 5, 16), (3, 1_000_003, 16), (70, 400_001, 33), (1_000_003, 3, 7)])
def test_products_of_many_rows_or_columns(m, n, k):
    _say("linear", m, n, k)
    rng = np.random.default_rng(n)
    (x, sx), (w, sw) = _rows(rng, m, k), _rows(rng, n, k)
    y = T.run("quant", "linear", [x, sx, w, sw, np.full((m, n), 7, np.float16)], outputs=[4])[4]
    np.testing.assert_array_equal(y.view(np.uint16), R.product(x, sx, w, sw).astype(np.float16).view(np.uint16))
