"""Rows that take the largest logit (rivoli_sample_rows by a temperature of none): whatever its size."""
import numpy as np
import pytest

from tests.test_gpu_sample import sample
from tests.util import bf16_to_f32, f32_to_bf16_rne

pytestmark = pytest.mark.gpu

NONE = [0.0, -1.0, np.nan, 2.0 ** -16, 2.0 ** -17, -0.0]


def taken(x, bf16, t=None):
    x = np.asarray(x, np.float32)
    assert not bf16 or (bf16_to_f32(f32_to_bf16_rne(np.where(np.isnan(x), 0, x))) == np.where(np.isnan(x), 0, x)).all()
    n = len(x)
    return sample(x, [0.0] * n if t is None else t, None, None, None, [0.7] * n, bf16)


def check(got, want, vocab):
    tokens, kept, logprobs, probs = got
    want = np.asarray(want)
    assert tokens.tolist() == want.tolist() and kept.tolist() == (want >= 0).astype(int).tolist()
    assert (logprobs == np.where(want >= 0, 0.0, -np.inf)).all()
    assert (probs == (np.arange(vocab) == want[:, None])).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_large_logits_are_told_apart(bf16):
    """Values past 2^25 that differ, in either order, near each other and chunks of the row apart; infinite ones above them all, the lower index first."""
    vocab = 20011
    a, b = 5.0 * 2 ** 23, 7.0 * 2 ** 24        # 4e7 and 1.2e8, of few bits
    inf = np.inf
    rows, want = [], []
    for at, to in ((3, 5), (2, 9000), (8191, 8192), (10, 20010), (0, 1)):
        for big, small in ((b, a), (a * 2.0 ** 90, b), (inf, a), (inf, 3e38 if not bf16 else 2.0 ** 127), (inf, inf)):
            for order in (0, 1):
                x = np.zeros(vocab)
                x[at], x[to] = (big, small) if order == 0 else (small, big)
                rows.append(x), want.append(at if order == 0 or big == small else to)
    check(taken(rows, bf16), want, vocab)
    # all of a row's are large, and rise: the last; and by every temperature that takes the first
    x = np.tile(2.0 ** 26 * (1 + (np.arange(vocab) // 160) / 128), (len(NONE), 1))
    check(taken(x, bf16, NONE), [vocab // 160 * 160] * len(NONE), vocab)


@pytest.mark.parametrize("bf16", [False, True])
def test_what_is_never_taken(bf16):
    """NaN, what is not above -2^25, and nothing else; rows of nothing but those take none."""
    vocab = 9001
    least = -2.0 ** 25
    above = least * (1 - 2.0 ** -8)
    x = np.full((6, vocab), least)
    x[0, 8500] = above
    x[1] = np.nan
    x[2], x[2, 77] = -np.inf, above
    x[3] = bf16_to_f32(np.array([0xFF7F], np.uint16))[0]       # the lowest number
    x[4], x[4, 8999] = np.nan, -3.0
    x[5, ::2] = -np.inf
    check(taken(x, bf16), [8500, -1, 77, -1, 8999, -1], vocab)
