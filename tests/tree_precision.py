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

from tests.draft_cases import e4m3_values, rows_of, tree_attention
from tests.util import bf16_to_f32, f32_to_bf16_rne

HALF = 2.0 ** -11          # fp16's half step
FLOOR = 2.0 ** -13


def bf16_of(x):
    return bf16_to_f32(f32_to_bf16_rne(np.asarray(x, np.float32))).astype(np.float64)


def score_error(case):
    """The score's term above, the largest of a case."""
    q = np.concatenate([bf16_to_f32(case.qabs), bf16_to_f32(case.qrope)], 2).astype(np.float64)
    worst = 0.0
    for s in range(len(case.ctx)):
        held = case.cu[s + 1] - case.cu[s]
        if held:
            rows, _ = rows_of(case.pool, case.tables[s], case.page, q.shape[2], case.ctx[s] + held)
            worst = max(worst, float((q[case.cu[s]:case.cu[s + 1]] ** 2 @ (rows ** 2).T).max()))
    return 72 * 2.0 ** -24 * abs(case.scale) * np.sqrt(worst)


def norm_bound(want, scores):
    """Of |got - want| over all elements of `want`."""
    n = want.size
    e, size = np.linalg.norm(bf16_of(want) - want), np.linalg.norm(want)
    return e * (1 + 5 * 0.9 / (2 * np.sqrt(n))) + np.hypot(e, (HALF + scores) * size) - e + FLOOR * size


def check_norm(case, got):
    """got: bf16 as uint16, [n][H][kvl]; of the nodes that there are."""
    want = tree_attention(case.qabs, case.qrope, case.pool, case.tables, case.ctx, case.cu, case.masks, case.page, case.scale)[0][:case.cu[-1]]
    x = bf16_to_f32(got[:case.cu[-1]]).astype(np.float64)
    off, far = np.linalg.norm(x - want), norm_bound(want, score_error(case))
    assert off <= far, (off / np.linalg.norm(want), far / np.linalg.norm(want))


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


# ---- rows that attend one token each --------------------------------------------------------------------------

def single_out(case, growth, seed=0, apart=1):
    """Gives every row (node and head) of a case a token of its own, all of a sequence's cached ones in turn (or every `apart`-th) and then the node itself, that outweighs
    nearly always all others: q along that token's latent codes, long enough for a score of 80, where a token whose scale is `growth` times the row's own (up to 4) has
    scores of 80 growth / sqrt(kvl) deviation, 14 or 20. Returns [n][H] tokens."""
    n, H, kvl = case.qabs.shape
    width = kvl + case.qrope.shape[2]
    scales = case.pool[:, case.page * width:].view(np.float32)
    scales[:] = 1 / 300
    for s in range(len(case.ctx)):
        for b, page in enumerate(case.tables[s]):
            scales[page] *= np.float32(dict(flat=1.0, grow=1.0 + 3.0 * b / max(1, case.tables.shape[1] - 1), swing=(1.0, 4.0, 0.999)[b % 3])[growth])
    own = np.zeros((n, H), np.int64)
    case.qrope[:] = 0
    rng = np.random.default_rng(seed)
    for s in range(len(case.ctx)):
        held, ctx = case.cu[s + 1] - case.cu[s], int(case.ctx[s])
        rows, _ = rows_of(case.pool, case.tables[s], case.page, width, ctx + held)
        start = int(rng.integers(0, ctx + 1))
        for i in range(held):
            turn = (start + apart * (i * H + np.arange(H))) % (ctx + 1)
            t = np.where(turn < ctx, turn, ctx + i)
            own[case.cu[s] + i] = t
            q = rows[t, :kvl]
            case.qabs[case.cu[s] + i] = f32_to_bf16_rne((q * (80 / (case.scale * (q ** 2).sum(1)))[:, None]).astype(np.float32))
    return own


def check_singled_out(case, own, got):
    """Against 64 bits, element by element: a result rounded to bf16 once, every weight to fp16 once (HALF of the magnitudes it is summed from, which are the result's own where
    one token has all the weight) and the smallest lost (FLOOR). A score is off by 72 2^-24 sqrt(sum (q k)^2) <= 1.5e-4 (that root is some 80 growth / sqrt(kvl), 14 to 20,
    or somewhat more), a difference of two by twice that: so much of the lesser tokens' weight may lie on the other row."""
    n, H, kvl = case.qabs.shape
    width = kvl + case.qrope.shape[2]
    alone = 0
    for s in range(len(case.ctx)):
        a, b = case.cu[s], case.cu[s + 1]
        if a == b:
            continue
        ctx = case.ctx[s]
        rows, there = rows_of(case.pool, case.tables[s], case.page, width, ctx + b - a)
        q = np.concatenate([bf16_to_f32(case.qabs[a:b]), bf16_to_f32(case.qrope[a:b])], 2).astype(np.float64)
        x = (q.reshape(-1, width) @ rows.T * case.scale).reshape(b - a, H, -1)
        for i in range(b - a):
            seen = there.copy()
            for j in range(b - a):
                seen[ctx + j] &= j <= i if case.masks is None else bool(case.masks[a + i][j >> 5] >> (j & 31) & 1)
            x[i][:, ~seen] = -np.inf
        w = np.exp(x - x.max(2, keepdims=True))
        w /= w.sum(2, keepdims=True)
        lesser = (1 - w.max(2))[..., None]
        alone += int((np.take_along_axis(w, own[a:b, :, None], 2) > 0.99).sum())
        w = w.reshape(-1, w.shape[2])
        want, mass = ((w @ v).reshape(b - a, H, kvl) for v in (rows[:, :kvl], np.abs(rows[:, :kvl])))
        most = np.abs(rows[:, :kvl]).max()
        far = 2.0 ** -8 * np.abs(want) + (1 + 2.0 ** -8) * (HALF * mass + FLOOR * most) + 3e-4 * 2 * np.minimum(lesser, 0.5) * most
        off = np.abs(bf16_to_f32(got[a:b]).astype(np.float64) - want)
        assert (off <= far).all(), (s, np.argwhere(~(off <= far).all(2))[:5], own[a:b][~(off <= far).all(2)][:5])
    assert alone > 0.9 * own[:case.cu[-1]].size


def emulated(case, kept, moved=None):
    """A case's results with the weights, exponential times scale under about the row's largest (the largest of a first tile may be any other token's), rounded
    by `kept` where they meet the values; moved(values) may change the value rows of a sequence. [n][H][kvl], bf16 as uint16."""
    n, H, kvl = case.qabs.shape
    width = kvl + case.qrope.shape[2]
    q = np.concatenate([bf16_to_f32(case.qabs), bf16_to_f32(case.qrope)], 2).astype(np.float64)
    out, rng = np.zeros((n, H, kvl)), np.random.default_rng(1)
    for s in range(len(case.ctx)):
        held, ctx = case.cu[s + 1] - case.cu[s], case.ctx[s]
        rows, there = rows_of(case.pool, case.tables[s], case.page, width, ctx + held)
        scales = np.array([case.pool[case.tables[s][t // case.page], case.page * width:].view(np.float32)[t % case.page] for t in range(ctx + held)], np.float64)
        codes = rows[:, :kvl] / np.where(there, scales, 1)[:, None]
        if moved:
            codes = moved(codes)
        for i in range(held):
            node, seen = case.cu[s] + i, there.copy()
            for j in range(held):
                seen[ctx + j] &= j <= i if case.masks is None else bool(case.masks[case.cu[s] + i][j >> 5] >> (j & 31) & 1)
            if not seen.any():
                continue
            x = q[node] @ rows[seen].T * case.scale
            e = np.exp(x - x.max(1, keepdims=True))
            w = e * scales[seen]
            top = w.max(1, keepdims=True) * np.exp2(rng.random((H, 1)))
            out[node] = np.asarray(kept(w / top), np.float64) * top @ codes[seen] / e.sum(1, keepdims=True)
    return f32_to_bf16_rne(out.astype(np.float32))
