"""Draws (rivoli_sample_rows) from rows with one token far above the others, whose weights are next to nothing beside its own: what is drawn is a
kept token whatever the random number, and its results are written."""
import numpy as np
import pytest

from tests.draft_cases import F32
from tests.sample_cases import sample_row
from tests.test_gpu_sample import sample
from tests.util import bf16_to_f32, f32_to_bf16_rne

pytestmark = pytest.mark.gpu

VOCAB = 26001                       # three whole chunks of 8 192 tokens and some
# the first and the last number of [0, 1), some next to nothing, and the first past it
US = [0.0, 2.0 ** -140, 2.0 ** -40, 2.0 ** -33, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0]


def rows(rng, kind, gap, t, bf16):
    """A row for each random number: the others `gap` temperatures below the first, all alike or over six temperatures; in front of them, or not, masked tokens."""
    x = np.full((len(US), VOCAB), -gap * t)
    if "spread" in kind:
        x -= t * rng.uniform(0, 6, x.shape)
    if "masked" in kind:
        x[:, :8192 if "chunk" in kind else 1] = -np.inf
    x[:, VOCAB // 2 if "middle" in kind else VOCAB - 1] = 0.0
    x = x.astype(np.float32)
    return np.where(np.isinf(x), x, bf16_to_f32(f32_to_bf16_rne(x))) if bf16 else x


def check(got, x, t, k, m):
    m = float(np.float32(m))
    tokens, kept, logprobs, probs = got
    for r, u in enumerate(US):
        _, count, share = sample_row(x[r], t, k, 1.0, m, u)
        z = ((x[r].astype(np.float64) - x[r].max()) / float(np.float32(t))).astype(np.longdouble)
        order = np.lexsort((np.arange(VOCAB), -x[r]))[:count]
        keep = np.zeros(VOCAB, bool)
        keep[order] = True
        assert kept[r] == count, r
        token = int(tokens[r])
        assert 0 <= token < VOCAB and keep[token], (r, u, token)
        w = np.where(keep, np.exp(z), 0)
        upto = np.cumsum(w)
        want = float(z[token] - np.log(upto[-1]))
        # a share is right to a weight's 2^-29 and, among whole numbers, to half of 2^-42 a token: of a whole of one at least
        assert abs(logprobs[r] - want) <= F32 * abs(want) + 2.0 ** -29 + VOCAB * 2.0 ** -43, (r, u)
        if u == 0.0:
            assert token == np.nonzero(keep)[0][0]
        elif u >= 1.0:
            assert token == np.nonzero(keep)[0][-1]
        else:
            # its own part of the sum, to what weights and sums are right to: 2^-29 of themselves, in bins 2^-23 of those below 2^-11, and a whole number of 2^-42 a token and a chunk
            far = 2.0 ** -29 * upto + 2.0 ** -23 * np.cumsum(np.where(w < 2.0 ** -11, w, 0)) + 2.0 ** -42 * (np.cumsum(keep) + 256)
            target, target_far = u * upto[-1], u * far[-1]
            assert upto[token] + far[token] + target_far >= target, (r, u)
            assert token == 0 or upto[token - 1] - far[token - 1] - target_far <= target, (r, u)
        off = np.abs(probs[r] - share)
        assert (off <= (F32 + VOCAB * 2.0 ** -42) * share + 2.0 ** -149).all() and ((probs[r] > 0) <= (share > 0)).all(), r


@pytest.mark.parametrize("kind", ["alike", "alike masked", "alike masked chunk", "alike middle", "spread", "spread masked chunk", "spread masked middle"])
@pytest.mark.parametrize("k,m", [(0, 0.0), (20000, 0.0), (9000, 0.0), (2500, 0.0), (300, 0.0), (40, 0.0), (0, 1e-20), (15000, 1e-20)])
def test_a_draw_is_of_a_kept_token(kind, k, m):
    rng = np.random.default_rng(len(kind) + k)
    for gap, t, bf16 in ((29.0, 1.0, False), (32.0, 0.2, True), (38.0, 1.0, False), (64.0, 0.7, False), (150.0, 1.0, True), (400.0, 0.3, False)):
        x = rows(rng, kind, gap, t, bf16)
        n = len(US)
        check(sample(x, [t] * n, [k] * n, None, [m] * n, US, bf16), x, t, k, m)


def test_rows_in_front_of_each_other_write_their_own():
    """Rows of either kind in one call, without filters, some of which were never written: none keeps what was there."""
    rng = np.random.default_rng(3)
    for gap in (30.0, 32.0, 36.0, 45.0):
        x = np.concatenate([rows(rng, kind, gap, 1.0, True) for kind in ("alike masked chunk", "alike", "spread masked chunk")])
        u = US * 3
        tokens, kept, logprobs, probs = sample(x, None, None, None, None, u, True)
        assert (kept == (x > -np.inf).sum(1)).all() and np.isfinite(logprobs).all()
        assert (np.abs(probs.sum(1) - 1) <= 2.0 ** -20).all()
        assert np.isfinite(x[np.arange(len(x)), tokens]).all()
        first = [np.nonzero(np.isfinite(r))[0][0] for r in x]
        for r in range(len(x)):
            assert u[r] != 0.0 or tokens[r] == first[r]


@pytest.mark.parametrize("first", [True, False])
def test_the_longest_rows(first):
    """2^21 tokens, each next to nothing, half a millionth together: the last numbers in front of one are theirs where they come last."""
    vocab, gap = 2 ** 21, 29.0
    u = [0.0, 2.0 ** -33, 0.5, 1 - 2.0 ** -22, 1 - 2.0 ** -23, 1 - 2.0 ** -24, 1.0]
    x = np.full((len(u), vocab), -gap, np.float32)
    top = 0 if first else vocab - 1
    x[:, top] = 0.0
    tokens, kept, logprobs, _ = sample(x, None, None, None, None, u, False, probs=False)
    w = np.exp(-np.longdouble(gap))
    whole = 1 + (vocab - 1) * w
    assert (kept == vocab).all()
    for token, number, logprob in zip(tokens, u, logprobs):
        assert abs(logprob - (float(token != top) * -gap - float(np.log(whole)))) <= F32 * gap + 2.0 ** -29
        if number in (0.0, 1.0):
            assert token == (0 if number == 0.0 else vocab - 1)
        else:
            # 2^-42 a chunk, 2^-23 of what lies in bins, in tokens of w; where the first outweighs them, it is drawn
            exact = (np.longdouble(number) * whole - (1 if first else 0)) / w
            far = float((256 * 2.0 ** -42 + 2.0 ** -23 * vocab * w) / w) + 1
            assert token == top if exact < 0 or exact >= vocab else abs(float(token - exact)) <= far
