"""The scratch of the quant kernels' handles: one buffer for all of them, whatever the number of handles, beside graphs
that were captured before it grew, and products without it where there is no memory for it."""

import ctypes

import numpy as np
import pytest

import tessel_amd as T
from tests import quant_refs as R
from tests.test_quant_gpu import _attention_case, _close, _rows, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _open(gpu):
    yield


def _linear(rng, m, n, k):
    """A handle, its buffers and the product."""
    (x, sx), (w, sw) = _rows(rng, m, k), _rows(rng, n, k)
    kern = T.kernel("quant", "linear", [(m, k), (m,), (n, k), (n,), (m, n)])
    return kern, [T.tensor(v) for v in (x, sx, w, sw)] + [T.alloc(2 * m * n)], R.product(x, sx, w, sw).astype(np.float16)


def _check(bufs, want):
    np.testing.assert_array_equal(T.read_array(bufs[4], np.float16, want.shape).view(np.uint16), want.view(np.uint16))


def _memory_free():
    # (of the runtime that the library has loaded)
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    assert ctypes.CDLL("libamdhip64.so.7").hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
    return free.value


def _free(bufs):
    for b in bufs:
        T.free(b)


def _capture(launches):
    T.capture_begin()
    for kern, bufs in launches:
        T.launch(kern, bufs)
    return T.capture_end()


def test_handles_of_many_row_counts_hold_one_copy():
    # A copy of W and X is 27 MB here.
    _say("handles of many row counts")
    n, k = 5000, 4001
    before = None
    for i in range(30):
        m = 1500 + 7 * i
        kern = T.kernel("quant", "linear", [(m, k), (m,), (n, k), (n,), (m, n)])
        if i == 0:
            bufs = [T.alloc(b) for b in (m * k, 4 * m, n * k, 4 * n, 2 * m * n)]
            assert T.graph_nodes(_capture([(kern, bufs)]))["kernel"] == 2  # (rows are copied first)
            _free(bufs)
            before = _memory_free()
    assert before - _memory_free() < 120e6


def test_a_product_without_memory_for_a_copy():
    # 4194240 rows of 131071: a copy would be 550 GB. The handle is made (and launched nowhere: its operands do not fit either).
    _say("no memory for a copy")
    m, n, k = 4000, 2 ** 22 - 64, 131071
    T.kernel("quant", "linear", [(m, k), (m,), (n, k), (n,), (m, n)])
    rng = np.random.default_rng(0)
    kern, bufs, want = _linear(rng, 700, 900, 1001)
    T.launch(kern, bufs)
    _check(bufs, want)
    _free(bufs)


def test_graphs_beside_a_scratch_that_grows():
    # Three products and an attention of several chunks, captured in turn, each after the handle before; then larger ones; every
    # replay and eager launch in changing order gives its own bits.
    _say("graphs and growing scratch")
    rng = np.random.default_rng(1)
    case = _attention_case(rng, 2, 8, 2, 64, 16, [3000, 2100])
    arrays = [case[0], R.pack_k(case[1]), R.pack_v(case[2]), case[3], case[4], case[5], case[6], np.full_like(case[0], 7)]
    att = T.kernel("quant", "decode_attention", [x.shape for x in arrays])
    att_bufs = [T.tensor(x) for x in arrays]
    args = att_bufs + [T.F32(case[7])]
    T.launch(att, args)
    first = T.read_array(att_bufs[7], np.float16, case[0].shape)
    _close(first.astype(np.float64), *case)
    done, graphs = [], []
    for m, n, k in ((1500, 2100, 2001), (1600, 2500, 2001), (1500, 4100, 4001), (2500, 6000, 4001)):
        kern, bufs, want = _linear(rng, m, n, k)
        done.append((kern, bufs, want))
        graphs.append(_capture([(kern, bufs), (att, args), done[0][:2]]))
        assert T.graph_nodes(graphs[-1]) == {"kernel": 6, "memset": 0, "memcpy": 0, "other": 0}
    for rep in range(3):
        for graph, (_, bufs, want) in zip(graphs, done):
            for _, b, _ in done:
                T.fill_nan(b[4])
            T.fill_nan(att_bufs[7])
            other = done[(rep + 2) % len(done)]
            T.launch(*other[:2])
            T.replay(graph)
            _check(bufs, want)
            _check(*done[0][1:])
            np.testing.assert_array_equal(T.read_array(att_bufs[7], np.float16, first.shape).view(np.uint16), first.view(np.uint16))
            T.launch(*other[:2])
            _check(*other[1:])
    for _, bufs, _ in done:
        _free(bufs)
    _free(att_bufs)
