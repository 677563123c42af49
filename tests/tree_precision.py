"""What tree attention's precision is held to beyond tests/draft_cases.tree_attention's element by element: sums over many elements, in which
roundings average out and a rounding too many does not.

A result is rounded to bf16 once: that error is known, e = bf16(want) - want, and over N elements the norm of another vector's that is as
good as `want` differs from |e| by some 0.9 / (2 sqrt(N)) of it. What comes before the rounding adds to it in squares:
  - a weight's rounding to fp16, at most 2^-11 of it (half a step), and different tokens' independent: 2^-11 of the norm;
  - a score's: 576 additions in f32, each half a step of a partial sum, which is within three standard deviations of a random walk's, 3
    sqrt(sum (q k)^2): 72 2^-24 |scale| max_t sqrt(sum (q k)^2) of a weight;
  - what fp16 cannot hold of the smallest weights: 2^-13 of the largest weight of a work item's first tile, over all of its tokens.
(bf16 weights would add 2^-8 / sqrt(6) or so, as much as the result's own rounding: 2.3e-3 and more in place of 1.7e-3.)"""
import numpy as np

from tests.draft_cases import e4m3_values
from tests.util import bf16_to_f32, f32_to_bf16_rne

HALF = 2.0 ** -11          # fp16's half step
FLOOR = 2.0 ** -13


def bf16_of(x):
    return bf16_to_f32(f32_to_bf16_rne(np.asarray(x, np.float32))).astype(np.float64)


# ---- an early dominant token over a long flat tail ------------------------------------------------------------

SINK_TOKENS, SINK_HEADS, SINK_PAGE = 131072, 64, 64


class Sink:
    """One sequence: a first token that every head attends most, 131 072 others whose weights are equal and, by head, 2^-22 to 2^-34 of it, and whose
    values have a common part. The last of them is the drafted node."""

    def __init__(self):
        rng = np.random.default_rng(77)
        self.pages = SINK_TOKENS // SINK_PAGE + 1
        common = rng.integers(0x60, 0x70, 512).astype(np.uint8) | (rng.integers(0, 2, 512).astype(np.uint8) << 7)   # 32 to 120
        codes = np.zeros((self.pages * SINK_PAGE, 576), np.uint8)
        codes[:, :512] = common
        codes[:, ::7] ^= rng.integers(0, 2, codes[:, ::7].shape, dtype=np.uint8) << 7                               # and a part that is not
        codes[:, 512:] = 0
        codes[0, :512] = rng.permutation(common)
        codes[0, 512:] = 0x70                                                                                         # 128
        self.codes, self.row_scale = codes, np.float32(2.0 ** -7)
        self.pool = np.zeros((self.pages, SINK_PAGE * 580), np.uint8)
        self.pool[:, :SINK_PAGE * 576] = codes.reshape(self.pages, -1)
        self.pool[:, SINK_PAGE * 576:] = np.full((self.pages, SINK_PAGE), self.row_scale).view(np.uint8)
        # a head's score is that of the first token alone: 64 dims of 128 2^-7 = 1 times q
        self.scale = 0.125
        apart = np.linspace(22, 34, SINK_HEADS)
        self.qabs = np.zeros((SINK_HEADS, 512), np.uint16)
        self.qrope = f32_to_bf16_rne(np.repeat((apart * np.log(2) / (64 * self.scale))[:, None], 64, 1).astype(np.float32))

    def exact(self, kept=None, lift=None):
        """[heads][512] in 64 bits, from weights as they are or (`kept`, a type; `lift`, of the first token's in powers of two) rounded for the values."""
        values = e4m3_values()[self.codes[:SINK_TOKENS + 1, :512]] * np.float64(self.row_scale)
        x = bf16_to_f32(self.qrope).astype(np.float64).sum(1) * self.scale
        tail = np.exp(-x)
        if kept is None:
            first, low = np.ones(SINK_HEADS), tail
        else:
            first, low = (np.asarray(kept(w * 2.0 ** lift), np.float64) / 2.0 ** lift for w in (np.ones(SINK_HEADS), tail))
        common = values[1:].sum(0)
        return (first[:, None] * values[0] + low[:, None] * common) / (1 + SINK_TOKENS * tail)[:, None], common / np.linalg.norm(common), np.linalg.norm(common) / SINK_TOKENS

    def check(self, got):
        """By head: the norm, and the error along the tail's common part against the rounded result: there an element that comes out a step (2^-7 of it at
        most) away does so with a likelihood of its error in steps, and six standard deviations of such elements are allowed."""
        want, along, each = self.exact()
        rounded, size = bf16_of(want), np.linalg.norm(want, axis=1)
        off, far = np.linalg.norm(got - want, axis=1), np.linalg.norm(rounded - want, axis=1) * 1.15 + (HALF + FLOOR) * size
        assert (off <= far).all(), (off / size, far / size)
        off = np.abs((got - rounded) @ along)
        far = 6 * np.sqrt(((HALF + FLOOR) * 2.0 ** -7 * want ** 2 * along ** 2).sum(1)) + HALF * np.abs(want @ along) + FLOOR * each
        assert (off <= far).all(), (off / size, far / size)
