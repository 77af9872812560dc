"""quant/decode_attention on the GPU within what f32 arithmetic leaves of 64 bits (quant_refs.within_f32), and each
token of a sequence where it counts alone: the first and last ones, those at the ends of pages, tiles and chunks."""

import numpy as np
import pytest

from tests import quant_refs as R
from tests.test_quant_gpu import _attend, _attention_case, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _open(gpu):
    yield


def _moved(case):
    """How many outputs are another f16 than the exact one's, and how many f32 arithmetic may move; whether none is too far off."""
    got = _attend(*case)
    fine, moved, most = R.within_f32(got, *R.attention_error(*case))
    print("[moved]", moved, "of", got.size, "at most %.0f" % most, flush=True)
    return fine, moved, most


# Short and long tables, one chunk a sequence and several, batches of one to two workgroups a CU (taken by length).
CASES = [
    (4, 32, 8, 128, 16, [4000, 130, 2777, 1]), (3, 8, 4, 32, 16, [1000, 900, 37]), (2, 8, 1, 64, 16, [4097, 3000]),
    (3, 4, 2, 16, 16, [1500, 700, 20]), (5, 32, 4, 64, 16, [333, 20, 100, 250, 17]), (1, 16, 1, 128, 32, [16000]),
    (2, 4, 4, 128, 64, [2111, 1024]), (40, 8, 8, 128, 16, list(range(1100, 2000, 23))), (2, 4, 2, 64, 512, [3000, 700]),
    (2, 32, 2, 32, 16, [6000, 1025])]


@pytest.mark.parametrize("b,h,g,d,p,lens", CASES)
def test_few_outputs_are_another_f16_than_the_exact_ones(b, h, g, d, p, lens):
    _say("attention, moved outputs", b, h, g, d, p)
    _, moved, most = _moved(_attention_case(np.random.default_rng(b + h + d + p), b, h, g, d, p, lens))
    assert moved <= most


@pytest.mark.parametrize("d,h,g", [(16, 8, 2), (32, 4, 4), (64, 16, 1), (128, 8, 2)])
def test_far_scores_and_equal_ones(d, h, g):
    _say("attention, scores", d)
    case = _attention_case(np.random.default_rng(d), 3, h, g, d, 16, [1300, 70, 513], spread=6.0)
    for q in (case[0], case[0] * np.float16(1e-3)):
        _, moved, most = _moved([q, *case[1:]])
        assert moved <= most


# (300 sequences of 8 heads: a product p step whose two halves are not of one f32 value shows once in some thousand tokens.)
@pytest.mark.parametrize("b,h,g,d,p,lens", CASES + [(300, 8, 2, 32, 16, [40, 17, 3] * 100), (100, 16, 1, 64, 16, [60, 2] * 50)])
def test_no_output_is_further_off_than_f32_arithmetic_leaves_it(b, h, g, d, p, lens):
    _say("attention, error", b, h, g, d, p)
    assert _moved(_attention_case(np.random.default_rng(b + h + d + p), b, h, g, d, p, lens))[0]


@pytest.mark.parametrize("d,h,g", [(16, 8, 2), (32, 4, 4), (64, 16, 1), (128, 8, 2)])
def test_no_output_is_further_off_at_far_scores(d, h, g):
    _say("attention, error at far scores", d)
    assert _moved(_attention_case(np.random.default_rng(d), 3, h, g, d, 16, [1300, 70, 513], spread=6.0))[0]


def _needles(rng, h, g, d, p, n, at):
    """A sequence of n tokens for each of `at`, whose token at that place has nearly all the weight (its key follows the
    signs of the queries); behind each sequence's end lie tokens that would have more."""
    case = _attention_case(rng, len(at), h, g, d, p, [n] * len(at))
    q, kn, vn, ks, vs, table, _, scale = case
    sign = rng.choice([-1, 1], (len(at), g, d))
    q[:] = np.abs(q) * np.repeat(sign, h // g, axis=1)
    for i, t in enumerate(at):
        for x in (t, *range(n, min(n + 5, table.shape[1] * p))):
            page, off = table[i, x // p], x % p
            kn[page, :, off] = np.where(sign[i] > 0, 15, 0)
            ks[page, :, off] = np.array([-7.5, 1.0]) * (0.8 if x == t else 4.0) * 4 / np.sqrt(d) ** 0.5
    return case


@pytest.mark.parametrize("h,g,d,p,n", [(2, 1, 16, 16, 900), (8, 2, 64, 16, 1000), (16, 1, 32, 32, 300), (4, 4, 128, 64, 1000),
                                       (8, 8, 64, 16, 77), (4, 2, 16, 16, 2100)])
def test_every_edge_of_short_tables(h, g, d, p, n):
    _say("needles", h, g, d, p, n)
    at = sorted({0, 1, n - 1, n - 2} | {x + e for x in range(0, n, 64) for e in (-1, 0, 15, 16) if 0 <= x + e < n})
    case = _needles(np.random.default_rng(n + d), h, g, d, p, n, at)
    want, _ = R.attention_error(*case)
    for i, t in enumerate(at):  # the token's own values, nearly (what the tests above could not tell apart otherwise)
        page = case[5][i, t // p]
        own = R.values(case[2][page, :, t % p], case[4][page, :, t % p])
        np.testing.assert_allclose(want[i], np.repeat(own, h // g, axis=0), atol=0.05)
    assert _moved(case)[0]


@pytest.mark.parametrize("h,g,d,p,n", [(4, 1, 64, 16, 5001), (8, 2, 128, 16, 4100), (2, 2, 32, 512, 3000)])
def test_every_edge_of_long_tables(h, g, d, p, n):
    # Chunks are multiples of 256 tokens.
    _say("needles, long", h, g, d, p, n)
    at = sorted({0, n - 1} | {x + e for x in range(256, n, 256) for e in (-1, 0)})
    assert _moved(_needles(np.random.default_rng(n + d), h, g, d, p, n, at))[0]
    assert _moved(_needles(np.random.default_rng(n), h, g, d, p, n, [0, n - 1, 2048]))[0]  # (few sequences: other chunks)


def test_every_edge_of_a_batch_by_length():
    # 64 sequences of 8 kv heads, each of another length, its last or first token the one that counts.
    _say("needles, by length")
    rng = np.random.default_rng(3)
    h, g, d, p, n = 8, 8, 64, 16, 1700
    case = _needles(rng, h, g, d, p, n, [n - 1] * 64)
    lens, table = case[6], case[5]
    lens[:] = rng.permutation(np.arange(1, n, n // 64)[:64])
    lens[5], lens[9] = n, 1025
    for i in range(64):
        t = 0 if i % 2 else lens[i] - 1
        page = table[i, t // p]
        case[1][page, :, t % p] = np.where(case[0][i] > 0, 15, 0)  # (a query head a kv head)
        case[3][page, :, t % p] = np.array([-7.5, 1.0]) * 0.7
    assert _moved(case)[0]


@pytest.mark.parametrize("b,h,g,d,most", [(64, 32, 8, 128, 4096), (40, 8, 8, 64, 1500), (300, 4, 1, 32, 1200), (20, 8, 4, 64, 5000)])
def test_a_sequence_has_its_bits_wherever_it_stands_in_the_batch(b, h, g, d, most):
    # Sequences are taken by length, in order, or in chunks: again, and in another order, each gives the same bits.
    _say("attention, order of the batch", b, g, d)
    rng = np.random.default_rng(b + d)
    lens = rng.integers(1, most + 1, b)
    lens[0] = most
    q, kn, vn, ks, vs, table, lens, scale = _attention_case(rng, b, h, g, d, 16, lens)
    first = _attend(q, kn, vn, ks, vs, table, lens, scale)
    for _ in range(3):
        at = rng.permutation(b)
        np.testing.assert_array_equal(_attend(q[at], kn, vn, ks, vs, table[at], lens[at], scale), first[at])
        np.testing.assert_array_equal(_attend(q, kn, vn, ks, vs, table, lens, scale), first)
