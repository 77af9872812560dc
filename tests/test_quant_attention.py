"""The tolerance of quant/decode_attention's tests (quant_refs.within_f32), without a GPU: f32 arithmetic passes, a
probability in one f16, a lost token and a chunk joined with another's maximum do not."""

import numpy as np
import pytest

from tests import quant_refs as R


def _case(rng, h, g, d, p, n):
    pages = (n + p - 1) // p + 2
    q = rng.standard_normal((1, h, d)).astype(np.float16)
    table = rng.permutation(pages).astype(np.int32)[None, :pages - 2]
    return [q, *R.cached(rng, pages, g, p, d), table, np.array([n], np.int32), float(np.float32(d ** -0.5))]


def _form(case, split=2, lose=None, bump=0.0):
    """The operator in f32 steps; p step in `split` f16; without token `lose`; its second half scaled by 1 + bump."""
    q, kn, vn, ks, vs, table, lens, scale = case
    (_, h, d), (_, g, p, _), n = q.shape, kn.shape, int(lens[0])
    t, out, f = np.arange(n), np.zeros(q.shape), np.float32
    page = table[0, t // p]
    for hh in range(h):
        (kc, kp), (vc, vp) = ((c[page, hh // (h // g), t % p].astype(f), x[page, hh // (h // g), t % p].astype(f))
                              for c, x in ((kn, ks), (vn, vs)))
        s = (kp[:, 1] * (kc @ q[0, hh].astype(f)) + kp[:, 0] * q[0, hh].astype(f).sum()) * f(scale)
        e = np.exp(s - s.max())
        e[n // 2:] *= f(1 + bump)
        if lose is not None:
            e[lose] = 0
        w = e * vp[:, 1] * f(2.0 ** 13)
        hi = w.astype(np.float16).astype(f)
        w = hi + (w - hi).astype(np.float16).astype(f) if split == 2 else hi
        acc = w @ (vc - 8) * f(2.0 ** -13) + e @ (vp[:, 0] + 8 * vp[:, 1])
        out[0, hh] = (acc / e.sum()).astype(np.float16)
    return out


@pytest.mark.parametrize("h,g,d,p,n", [(8, 2, 128, 16, 4000), (8, 4, 32, 16, 1000), (32, 4, 64, 16, 333), (16, 8, 16, 32, 1500)])
def test_f32_passes_and_what_is_less_does_not(h, g, d, p, n):
    case = _case(np.random.default_rng(n + d), h, g, d, p, n)
    want, rms = R.attention_error(*case)
    np.testing.assert_allclose(want, R.attention(*case)[0], rtol=1e-9, atol=1e-12)

    def passes(x):
        fine, moved, most = R.within_f32(x, want, rms)
        return fine and moved <= most

    assert passes(want.astype(np.float16).astype(np.float64)) and passes(_form(case))
    for broken in (_form(case, split=1), _form(case, lose=n - 1), _form(case, lose=0), _form(case, bump=2.0 ** -12)):
        assert not passes(broken)


def test_steps_of_f16():
    x = np.array([1.0, 0.9999, 2.0 ** -14, 2.0 ** -15, 0.0, 40000.0])
    np.testing.assert_array_equal(R.f16_steps(x), np.array([2.0 ** -10, 2.0 ** -11, 2.0 ** -24, 2.0 ** -24, 2.0 ** -24, 32.0]))
