"""quant/decode_attention on the GPU within what f32 arithmetic leaves of 64 bits (quant_refs.within_f32)."""

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
