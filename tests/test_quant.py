"""The quant kernels without a GPU: their keys, the sizes they refuse, and the
plain forms that the GPU tests compare with, pinned by their definitions."""

from fractions import Fraction

import numpy as np
import pytest

import tessel_amd as T
from tests import quant_refs as R


def _cache(np_=4, g=2, p=16, d=64, **kw):
    d2, pb, last, two = kw.get("d2", d // 2), kw.get("pb", p // 16), kw.get("last", 16), kw.get("two", 2)
    return [[np_, g, p, d2], [np_, g, pb, d2, last], [np_, g, p, two], [np_, g, p, two]]


def _decode(b=3, h=8, g=2, d=64, p=16, mp=5, **kw):
    kc, vc, ks, vs = _cache(4, g, p, d, **kw)
    return [[b, h, d], kc, vc, ks, vs, [b, mp], [b], [b, h, d]]


def _write(t=3, w=768, g=2, d=64, p=16, **kw):
    kc, vc, ks, vs = _cache(4, g, p, d, **kw)
    return [[t, w], [t], [t], [99, d // 2], [99, d // 2], kc, vc, ks, vs, [t, g, d], [t, g, d]]


@pytest.mark.parametrize("name,shapes,msg", [
    ("linear", [[2, 131072], [2], [3, 131072], [3], [2, 3]], "K = 131072 exceeds 131071"),
    ("linear", [[2, 64], [2], [3, 63], [3], [2, 3]], "dimension K is 64 and 63"),
    ("linear", [[2, 64], [3], [3, 64], [3], [2, 3]], "dimension M is 2 and 3"),
    ("linear", [[2, 64], [2], [3, 64], [3], [2, 4]], "dimension N is 3 and 4"),
    ("linear", [[2 ** 25, 64], [2 ** 25], [3, 64], [3], [2 ** 25, 3]], "at most 2\\^24"),
    ("linear", [[2 ** 18, 64], [2 ** 18], [2 ** 18, 64], [2 ** 18], [2 ** 18, 2 ** 18]], "at most 2\\^34 outputs"),
    ("gate_up", [[2, 131072], [2], [3, 131072], [3], [3, 131072], [3], [2, 3]], "K = 131072 exceeds"),
    ("gate_up", [[2, 64], [2], [3, 64], [3], [4, 64], [4], [2, 3]], "dimension F is 3 and 4"),
    ("quantize", [[2, 64], [2, 64], [3]], "dimension M is 2 and 3"),
    ("quantize", [[2, 2 ** 31], [2, 2 ** 31], [2]], "at most"),
    ("rmsnorm", [[2, 0], [0], [2, 0], [2]], "rows of 0 columns"),
    ("add_rmsnorm", [[2, 0], [2, 0], [0], [2, 0], [2]], "rows of 0 columns"),
    ("add_rmsnorm", [[2, 8], [2, 8], [9], [2, 8], [2]], "dimension Dm is 8 and 9"),
    ("kv_write", _write(p=8, pb=1), "multiple of 16 tokens"),
    ("kv_write", _write(p=48), "powers of two"),
    ("kv_write", _write(p=32, pb=1), "PB must be P / 16"),
    ("kv_write", _write(d=64, d2=64), "dimension D2 is"),
    ("kv_write", _write(d=256, w=4096), "head dimension 256 unsupported"),
    ("kv_write", _write(w=255), "hold no 2 G D"),
    ("kv_write", _write(last=8), "dimension must be 16"),
    ("kv_write", _write(two=1), "dimension must be 2"),
    ("decode_attention", _decode(h=7), "multiple of G"),
    ("decode_attention", _decode(h=6), "H / G must be"),
    ("decode_attention", _decode(d=8), "head dimension 8 unsupported"),
    ("decode_attention", _decode(d2=16), "D2 must be D / 2"),
    ("decode_attention", _decode(p=8, pb=1), "multiple of 16 tokens"),
    ("decode_attention", _decode(mp=2 ** 28), "tokens a table"),
    ("decode_attention", _decode(b=2 ** 23), "2\\^22"),
    ("decode_attention", _decode(b=2 ** 19 + 1), "2\\^22"),
    ("linear", [[2 ** 20 - 63, 64], [2 ** 20 - 63], [2 ** 14 - 31, 64], [2 ** 14 - 31], [2 ** 20 - 63, 2 ** 14 - 31]], "at most 2\\^34"),
    ("kv_write", _write(t=2 ** 23), "below 2\\^23"),
    ("decode_attention", [x[:0] + [0] + x[1:] if len(x) > 2 and x[0] == 4 else x for x in _decode()], "pool of no pages"),
    ("decode_attention", [[3, 8, 64]], "no shape given"),
    ("linear_residual", [], "no kernel linear_residual"),
])
def test_refusals(name, shapes, msg):
    with pytest.raises(T.TesselError, match=msg):
        T.kernel("quant", name, shapes)


def test_arguments_are_counted_and_handles_shared():
    shapes = [[2, 64], [2], [3, 64], [3], [2, 3]]
    k = T.kernel("quant", "linear", shapes)
    assert k.key == "quant/linear [[2, 64], [2], [3, 64], [3], [2, 3]] [] 4"
    assert T.kernel("quant", "linear", shapes).handle == k.handle
    with pytest.raises(T.TesselError, match="2 arguments for 5 parameters"):
        T.launch(k, [T.Buf(0, 4), T.Buf(0, 4)])
    with pytest.raises(T.TesselError, match="no meta constant BM"):
        T.kernel("quant", "linear", shapes, [("BM", 64)])


def test_the_plain_forms_round_as_fractions_do():
    rng = np.random.default_rng(0)
    for _ in range(40):
        y = np.concatenate([rng.integers(-60, 61, 12), [0]]) * 2.0 ** rng.integers(-8, 3)
        q, s = R.rows8(y[None])
        top = max(abs(Fraction(v)) for v in y)
        assert s[0] == float(top) / 127
        assert [int(c) for c in q[0]] == [round(Fraction(v) * 127 / top) if top else 0 for v in y]
        x = y.astype(np.float16)
        n, pair = R.heads4(x)
        lo, hi = (Fraction(float(f(x))) for f in (np.min, np.max))
        assert [int(c) for c in n] == [round((Fraction(float(v)) - lo) * 15 / (hi - lo)) if hi > lo else 0 for v in x]
        assert float(pair[0]) == lo and abs(float(pair[1]) - (hi - lo) / 15) <= (hi - lo) / 15 * Fraction(1, 2048)
        # A code is off by at most half a step, in both forms (and by the step's own rounding, 15 of them at most).
        assert (np.abs(q[0] * s[0] - y) <= s[0] * (0.5 + 1e-12)).all()
        step = float((hi - lo) / 15)
        assert (np.abs(R.values(n, pair) - x) <= step * (0.5 + 15 / 2048) + 1e-12).all()


def test_the_cache_layouts_hold_every_code():
    rng = np.random.default_rng(1)
    n = rng.integers(0, 16, (3, 2, 32, 16)).astype(np.uint8)
    k, v = R.pack_k(n), R.pack_v(n)
    assert k.shape == (3, 2, 32, 8) and v.shape == (3, 2, 2, 8, 16)
    for page, g, t, c in rng.integers(0, (3, 2, 32, 16), (200, 4)):
        shift = 4 * (c % 2)
        assert k[page, g, t, c // 2] >> shift & 15 == n[page, g, t, c]
        assert v[page, g, t // 16, c // 2, t % 16] >> shift & 15 == n[page, g, t, c]


def test_the_attention_form_is_softmax_over_the_held_values():
    rng = np.random.default_rng(2)
    kn, vn, ks, vs = R.cached(rng, 4, 2, 16, 16)
    q = rng.standard_normal((2, 4, 16)).astype(np.float16)
    table, lens = np.array([[3, 1], [2, -1]], np.int32), np.array([20, 30], np.int32)
    out, _, _ = R.attention(q, kn, vn, ks, vs, table, lens, 0.25)
    k, v = R.values(kn, ks), R.values(vn, vs)
    zero = np.zeros((14, 16))
    for i, h in ((0, 0), (0, 3), (1, 1), (1, 2)):
        pages = [(k[p, h // 2], v[p, h // 2]) for p in table[i] if p >= 0]
        kk, vv = (np.concatenate([x[j] for x in pages])[:20] if i == 0 else np.concatenate([pages[0][j], zero]) for j in (0, 1))
        e = np.exp(0.25 * (kk @ q[i, h].astype(np.float64)))
        np.testing.assert_allclose(out[i, h], (e @ vv) / e.sum(), rtol=1e-9, atol=1e-12)
