"""Every form of the 8-bit products (T.product_form names the one a launch takes, so that a rule that moves cannot leave one
without a test): sums by their bits, with rows, columns and steps that end inside a tile."""

import numpy as np
import pytest

import tessel_amd as T
from tests import quant_refs as R
from tests.test_quant_gpu import F, H, _rows, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _open(gpu):
    yield


LINEAR = [
    (1, 2560, 2048, 0, "skinny 16"), (20, 300, 256, 0, "skinny 32"), (33, 2000, 640, 0, "skinny 48"), (50, 301, 272, 0, "skinny 64"),
    (70, 1155, 1040, 0, "64x64"), (700, 2401, 1040, 0, "64x128"), (1024, 4096, 1024, 0, "128x128"), (1001, 4001, 1040, 0, "128x128"),
    (2500, 3001, 2064, 0, "256x128"),
    # One step of K, two, three, and more than the stages of the ring.
    (16383, 8191, 128, 0, "256x256"), (8191, 8190, 256, 0, "256x256"), (4095, 8190, 384, 0, "256x256"), (1501, 5629, 1024, 0, "256x256"),
    (777, 1155, 1001, 0, "any 4"), (1025, 1155, 201, 0, "any 2"), (1025, 1155, 7, 0, "any 2"), (300, 2000, 256, 1, "any 4"),
    (1025, 1155, 256, 3, "any 2"), (4001, 4001, 1001, 0, "copied 256x256"), (1500, 2100, 2001, 0, "copied 128x128")]
GATE_UP = [
    (7, 333, 256, 0, "skinny 16"), (20, 72, 1040, 0, "skinny 32"), (33, 2000, 640, 0, "skinny 48"), (60, 201, 640, 0, "skinny 64"),
    (65, 70, 96, 0, "64x64"), (700, 1401, 1040, 0, "64x128"), (600, 2003, 2064, 0, "128x128"), (500, 5601, 2048, 0, "256x128"),
    (8191, 8190, 128, 0, "256x256"), (4095, 8190, 256, 0, "256x256"), (4000, 4001, 384, 0, "256x256"), (511, 11001, 1024, 0, "256x256"),
    (300, 257, 201, 0, "any 4"), (1025, 601, 201, 0, "any 2"), (200, 500, 256, 1, "any 4"), (1025, 601, 128, 2, "any 2"),
    (2000, 4001, 1001, 0, "copied 256x256")]
FORMS = {"any 4", "any 2", "64x64", "64x128", "128x128", "256x128", "256x256", "skinny 16", "skinny 32", "skinny 48", "skinny 64"}


def test_the_lists_reach_every_form():
    for cases in (LINEAR, GATE_UP):
        assert {c[4] for c in cases} >= FORMS


def _at(x, off):
    """x on the device `off` bytes past a multiple of 16, and the buffer."""
    b = T.alloc(x.nbytes + 16)
    T.write(b, off, x)
    return T.Buf(b.ptr + off, x.nbytes), b


def _run(name, arrays, n, off, form):
    m = len(arrays[0])
    kern = T.kernel("quant", name, [x.shape for x in arrays] + [(m, n)])
    assert T.product_form(kern, off == 0) == form
    placed = [_at(x, off if x.dtype == np.int8 else 0) for x in arrays]
    y = T.alloc(2 * m * n + 64)
    T.fill_nan(y)
    T.launch(kern, [p for p, _ in placed] + [T.Buf(y.ptr, 2 * m * n)])
    got, behind = T.read_array(y, np.float16, (m, n)), T.read(y, 2 * m * n, 60)
    nans = np.full(16, 0x7fc00000, np.uint32).view(np.uint8)[2 * m * n % 4:][:60]
    np.testing.assert_array_equal(behind, nans)  # (nothing behind Y)
    for b in [b for _, b in placed] + [y]:
        T.free(b)
    return got


def _sums(x, w):
    """i32 sums as floats (f32 holds them exactly up to 1024 columns of 2^14)."""
    t = np.float32 if x.shape[1] <= 1024 else np.float64
    return (x.astype(t) @ w.astype(t).T).astype(np.float32)


@pytest.mark.parametrize("m,n,k,off,form", LINEAR)
def test_linear(m, n, k, off, form):
    _say("linear", m, n, k, off, form)
    rng = np.random.default_rng(m + n + k)
    (x, sx), (w, sw) = _rows(rng, m, k), _rows(rng, n, k)
    y = _run("linear", [x, sx, w, sw], n, off, form)
    for i in range(0, m, 2048):
        want = (_sums(x[i:i + 2048], w) * sx[i:i + 2048, None] * sw).astype(np.float16)
        np.testing.assert_array_equal(y[i:i + 2048].view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("m,f,k,off,form", GATE_UP)
def test_gate_up(m, f, k, off, form):
    _say("gate_up", m, f, k, off, form)
    rng = np.random.default_rng(m + f + k)
    (x, sx), (wg, sg), (wu, su) = _rows(rng, m, k), _rows(rng, f, k), _rows(rng, f, k)
    sx = sx * np.float32(400 / np.sqrt(k))
    y = _run("gate_up", [x, sx, wg, sg, wu, su], f, off, form)
    for i in range(0, m, 1024):
        g, u = ((_sums(x[i:i + 1024], w) * sx[i:i + 1024, None] * s).astype(np.float64) for w, s in ((wg, sg), (wu, su)))
        with np.errstate(over="ignore"):
            want = g / (1 + np.exp(-g)) * u
        # (test_quant_gpu's: f16's half step; exp2 of a product rounded once, reciprocal and products in f32)
        tol = H * np.abs(want) + (16 + 4 * np.abs(g)) * F * np.abs(want) + 2.0 ** -25
        off_by = np.abs(y[i:i + 1024].astype(np.float64) - want)
        assert (off_by <= tol).all(), (i, off_by.max())


def test_other_kernels_have_no_form():
    with pytest.raises(T.TesselError, match="no product of 8-bit rows"):
        T.product_form(T.kernel("quant", "quantize", [(2, 64), (2, 64), (2,)]))
