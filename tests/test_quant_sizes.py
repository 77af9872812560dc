"""Sizes of the quant kernels whose products pass 64 bits or whose values pass 32, refused when the handle is made (no GPU)."""

import pytest

import tessel_amd as T
from tests.test_quant import _decode, _write


def _b(shapes, b):
    return [[b] + s[1:] if i in (0, 5, 6, 7) else s for i, s in enumerate(shapes)]


@pytest.mark.parametrize("name,shapes,msg", [
    ("kv_write", _write(p=2 ** 31), "at most 2\\^30 tokens"),
    ("kv_write", _write(p=2 ** 32), "at most 2\\^30 tokens"),
    ("kv_write", _write(p=2 ** 60), "at most 2\\^30 tokens"),
    ("decode_attention", _decode(p=2 ** 32, mp=0), "at most 2\\^30 tokens"),
    ("decode_attention", _decode(p=2 ** 31, mp=0), "at most 2\\^30 tokens"),
    ("decode_attention", _decode(p=2 ** 30, mp=2), "tokens a table"),
    ("decode_attention", _b(_decode(h=2 ** 30, g=2 ** 30), 2 ** 34), "2\\^22"),  # B H and B G are 0 in 64 bits
    ("decode_attention", _b(_decode(), 2 ** 62), "2\\^22"),
])
def test_refusals(name, shapes, msg):
    with pytest.raises(T.TesselError, match=msg):
        T.kernel("quant", name, shapes)


def test_the_largest_pages_are_taken():
    T.kernel("quant", "kv_write", _write(p=2 ** 30))
    T.kernel("quant", "decode_attention", _decode(b=0, p=2 ** 30, mp=1))


def test_a_launch_opens_the_device():
    # (A handle that needs no scratch is made without one; a launch before anything else went to the null stream of whatever
    # device was current, which tsl_sync does not wait for. Rows of none: nothing is launched.)
    k = T.kernel("quant", "quantize", [[0, 64], [0, 64], [0]])

    def says(f):
        try:
            return f()
        except T.TesselError as e:
            return str(e)

    launched = says(lambda: T.launch(k, [T.Buf(0, 0)] * 3))
    assert launched == says(T.open)
