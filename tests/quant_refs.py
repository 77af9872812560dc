"""Plain 64-bit forms of the quant kernels for the tests: 8-bit rows, 8-bit
products, 4-bit heads and the paged cache that holds them. No code of the
kernels or of the oracle."""

import numpy as np


def round_half_even(num, den):
    """The whole numbers nearest to num / den (den > 0), ties to even; num, den exact in f64."""
    q = np.floor(num / den)
    r = num - q * den  # (exact: small multiples of the inputs)
    q = q + (2 * r > den)
    tie = (2 * r == den) & (np.mod(q, 2) == 1)
    return q + tie


def rows8(y):
    """Codes and step (f64) of 8-bit rows; NaN and 0 where a row holds a NaN or an infinity."""
    y = np.asarray(y, np.float64)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(y).all(axis=1)
    y = np.where(bad[:, None], 0.0, y)
    top = np.abs(y).max(axis=1) if y.shape[1] else np.zeros(len(y))
    den = np.where(top > 0, top, 1.0)
    q = round_half_even(127 * y, den[:, None]) * (top > 0)[:, None]
    return q.astype(np.int8), np.where(bad, np.nan, top / 127)


def product(x, sx, w, sw):
    """f32 values of the 8-bit product's definition, one rounding after another: i32 sums, then SX, then SW."""
    sums = (x.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)  # (exact: below 2^53)
    with np.errstate(all="ignore"):
        return sums * np.asarray(sx, np.float32)[:, None] * np.asarray(sw, np.float32)


def heads4(x):
    """Codes [.., D] and (low, step) f16 pairs of 4-bit heads x [.., D] f16."""
    bad = ~np.isfinite(x.astype(np.float64)).all(axis=-1)
    y = np.where(bad[..., None], 0.0, x.astype(np.float64))
    lo, hi = y.min(axis=-1), y.max(axis=-1)
    rng = hi - lo
    n = round_half_even(15 * (y - lo[..., None]), np.where(rng > 0, rng, 1.0)[..., None])
    pair = np.stack([lo, (rng / 15).astype(np.float32)], -1).astype(np.float16)
    pair[bad] = np.nan
    return n.astype(np.uint8), pair


def pack_k(n):
    """Codes [NP, G, P, D] as the cache's keys hold them."""
    return (n[..., 0::2] | n[..., 1::2] << 4).astype(np.uint8)


def pack_v(n):
    """Codes [NP, G, P, D] as the cache's values hold them: [NP, G, P / 16, D / 2, 16]."""
    np_, g, p, d = n.shape
    b = pack_k(n).reshape(np_, g, p // 16, 16, d // 2)
    return np.ascontiguousarray(b.swapaxes(-1, -2))


def cached(rng, pages, g, p, d, spread=1.0):
    """A random cache: codes [NP, G, P, D] of keys and values, and their pairs."""
    kn, vn = (rng.integers(0, 16, (pages, g, p, d)).astype(np.uint8) for _ in range(2))
    pairs = []
    for _ in range(2):
        step = (spread * rng.uniform(0.1, 0.4, (pages, g, p))).astype(np.float16)
        low = (-step.astype(np.float64) * rng.uniform(4, 11, step.shape)).astype(np.float16)
        pairs.append(np.stack([low, step], -1))
    return kn, vn, pairs[0], pairs[1]


def values(n, pair):
    pair = pair.astype(np.float64)
    return pair[..., :1] + pair[..., 1:] * n


def attention(q, kn, vn, ks, vs, table, lens, scale):
    """softmax(scale q K^T) V over the cache in f64, and two sums that rounding errors scale with: sum p step n
    and sum p |v|, and each row's largest |score|. NaN rows for empty sequences; pages outside the pool are zeros."""
    b, h, d = q.shape
    npg, g, p, _ = kn.shape
    out, mag, top = np.full((b, h, d), np.nan), np.zeros((b, h, d)), np.zeros((b, h, 1))
    for i in range(b):
        n = min(max(int(lens[i]), 0), table.shape[1] * p)
        if n == 0:
            continue
        t = np.arange(n)
        page = table[i, t // p]
        ok = (page >= 0) & (page < npg)
        pg = np.where(ok, page, 0)
        for hh in range(h):
            gg = hh // (h // g)
            k = np.where(ok[:, None], values(kn[pg, gg, t % p], ks[pg, gg, t % p]), 0.0)
            v = np.where(ok[:, None], values(vn[pg, gg, t % p], vs[pg, gg, t % p]), 0.0)
            low = np.where(ok[:, None], np.abs(vs[pg, gg, t % p, :1].astype(np.float64)), 0.0)
            s = k @ q[i, hh].astype(np.float64) * float(scale)
            e = np.exp(s - s.max())
            e /= e.sum()
            out[i, hh] = e @ v
            mag[i, hh] = e @ (np.abs(v) + 2 * low)
            # |q| . (|low| + |step n|): what a score's f32 sums round against.
            kl = np.where(ok[:, None], np.abs(k) + 2 * np.abs(ks[pg, gg, t % p, :1].astype(np.float64)), 0.0)
            top[i, hh] = (kl @ np.abs(q[i, hh].astype(np.float64))).max() * abs(float(scale))
    return out, mag, top


def attention_error(q, kn, vn, ks, vs, table, lens, scale):
    """softmax(scale q K^T) V in f64 (NaN rows for empty sequences), and the root mean square of what f32 arithmetic is off
    by before the output's rounding to f16, element by element.

    Token t's score step (q . n) + low sum(q) is off by one rounding of each term and of the sum, and by those of q . n's
    partial sums (a term's size, |q| 15 step at most): its probability by r_t = 2^-24 (4 + scale (|step q . n| +
    |low sum(q)| + |score| + 15 step max|q|)) of itself, each token's for itself, which moves an output by
    p_t r_t |v_t - out|. The sums over tokens are of centred values, sum p step (n - 8) and sum p (low + 8 step): a chain of N roundings
    of a sum that grows adds to sqrt(N / 3) half-steps, 4 of the sum of magnitudes for N = 48."""
    b, h, d = q.shape
    npg, g, p, _ = kn.shape
    out, rms = np.full((b, h, d), np.nan), np.zeros((b, h, d))
    for i in range(b):
        n = min(max(int(lens[i]), 0), table.shape[1] * p)
        if n == 0:
            continue
        t = np.arange(n)
        page = table[i, t // p]
        ok = ((page >= 0) & (page < npg))[:, None]
        pg = np.where(ok[:, 0], page, 0)
        for gg in range(g):
            (kc, kp), (vc, vp) = ((c[pg, gg, t % p].astype(np.float64), np.where(ok, x[pg, gg, t % p].astype(np.float64), 0.0))
                                  for c, x in ((kn, ks), (vn, vs)))
            v, mag = vp[:, :1] + vp[:, 1:] * vc, np.abs(vp[:, 1:] * (vc - 8)) + np.abs(vp[:, :1] + 8 * vp[:, 1:])
            for hh in range(gg * (h // g), (gg + 1) * (h // g)):
                qq = q[i, hh].astype(np.float64)
                a, c = kp[:, 1] * (kc @ qq), kp[:, 0] * qq.sum()
                e = np.exp((a + c) * float(scale) - ((a + c) * float(scale)).max())
                e /= e.sum()
                r = 4 + abs(float(scale)) * (np.abs(a) + np.abs(c) + np.abs(a + c) + 15 * kp[:, 1] * np.abs(qq).max())
                out[i, hh] = e @ v
                rms[i, hh] = 2.0 ** -24 * np.sqrt(((e * r) ** 2) @ (v - out[i, hh]) ** 2 + (4 * (e @ mag)) ** 2)
    return out, rms


def f16_steps(x):
    """The distance of f16's neighbours at x (f64)."""
    return 2.0 ** (np.where(x == 0, -13, np.maximum(np.frexp(np.abs(x))[1], -13)) - 11.0)


def within_f32(got, want, rms):
    """Whether f16 outputs are the exact ones as f32 arithmetic leaves them (attention_error): none further off than
    half a step of f16 and 8 times `rms`; and how many of them are another f16 than the exact one's, and how many may be: an
    error moves an output over a border between two f16 with the odds error / step, its mean magnitude is `rms` at
    most, and their number varies by its square root."""
    live = ~np.isnan(want)
    near = np.abs(got - want) <= f16_steps(want) / 2 + 8 * rms
    moved = (got != want.astype(np.float16)) & live
    odds = np.where(live, np.minimum(1.0, rms / f16_steps(want)), 0.0)
    most = odds.sum() + 4 * np.sqrt(odds.sum()) + 1
    return bool((np.isnan(got) == np.isnan(want)).all() and (near | ~live).all()), int(moved.sum()), float(most)
