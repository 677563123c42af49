"""Tokens drawn from logits (rivoli_sample_rows) against the definition in numpy: the same token and the same number of
kept ones, shares within their rounding."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import F32
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.sample_cases import as_bits, rows, sample_row

pytestmark = pytest.mark.gpu


def opt(a, kind):
    return None if a is None else dev(np.asarray(a, kind))


def sample(x, t, k, p, m, u, bf16, stride=None, probs=True, shift=0):
    n, vocab = x.shape
    stride = stride or vocab
    buf = np.full(n * stride + shift, 0x7FC0 if bf16 else 0, np.uint16 if bf16 else np.float32)
    for r in range(n):
        buf[shift + r * stride: shift + r * stride + vocab] = as_bits(x[r], bf16)
    buf = dev(buf)
    tokens, kept, logprobs, out = dzeros(4 * n, 0xEE), dzeros(4 * n, 0xEE), dzeros(4 * n, 0xEE), dzeros(4 * n * vocab, 0xEE) if probs else None
    work = dzeros(hip.sample_rows_workspace_bytes(n, vocab), 0xEE)
    hip.launch_sample_rows(buf.data_ptr() + shift * (2 if bf16 else 4), opt(t, np.float32), opt(k, np.int32), opt(p, np.float32), opt(m, np.float32),
                           dev(np.asarray(u, np.float32)), n, vocab, stride, bf16, tokens, kept, logprobs, out, vocab, work)
    return (back(tokens, np.int32), back(kept, np.int32), back(logprobs, np.float32).astype(np.float64),
            back(out, np.float32).reshape(n, vocab).astype(np.float64) if probs else None)


def check(got, x, t, k, p, m, u):
    n = len(x)
    f32 = lambda a, off: np.full(n, off, np.float32) if a is None else np.asarray(a, np.float32)  # noqa: E731
    t, p, m, u = f32(t, 1), f32(p, 1), f32(m, 0), f32(u, 0)
    tokens, kept, logprobs, probs = got
    for r in range(n):
        token, count, share = sample_row(x[r], t[r], 0 if k is None else k[r], float(p[r]), float(m[r]), float(u[r]))
        assert (tokens[r], kept[r]) == (token, count), r
        if token < 0:
            assert logprobs[r] == -np.inf
        else:
            # 2^-42 of the largest weight a token, half a step; a share of no more than 2^-149 is any or none
            want = np.log(share[token])
            assert abs(logprobs[r] - want) <= F32 * abs(want) + 2.0 ** -40 * len(x[r]) / (share.max() / share[token] or 1) + 1e-9, r
        if probs is not None:
            off = np.abs(probs[r] - share)
            assert (off <= (F32 + len(x[r]) * 2.0 ** -42) * share + 2.0 ** -149).all(), (r, off.max())
            assert ((probs[r] > 0) <= (share > 0)).all()


SIZES = [1, 2, 7, 1000, 8191, 8192, 8193, 32001]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("vocab", SIZES)
def test_sizes(vocab, bf16):
    rng = np.random.default_rng(vocab)
    n = 6
    x = rows(rng, "normal", n, vocab, bf16)
    t, k, p, m = [1, 0.7, 1.3, 1, 0.5, 0], [0, 40, 0, 3, 20, 9], [1, 1, 0.9, 0.7, 0.95, 0.5], [0, 0, 0, 0.02, 0.1, 0]
    u = rng.random(n).astype(np.float32)
    check(sample(x, t, k, p, m, u, bf16), x, t, k, p, m, u)


KINDS = ["model", "normal", "wide", "narrow", "equal", "steps", "masked", "odd"]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_filters_over_rows_of_all_kinds(kind, bf16):
    """Every filter alone and together; borders inside of bins of few tokens, of thousands, of nothing but equal ones, and far below the first."""
    vocab = 50001
    rng = np.random.default_rng(KINDS.index(kind))
    filters = [(0, 1.0, 0.0), (1, 1.0, 0.0), (50, 1.0, 0.0), (9000, 1.0, 0.0), (40000, 1.0, 0.0), (vocab, 1.0, 0.0), (0, 0.5, 0.0), (0, 0.95, 0.0),
               (0, 0.999999, 0.0), (0, 1e-6, 0.0), (0, 0.0, 0.0), (0, 1.0, 0.05), (0, 1.0, 1e-7), (0, 1.0, 2.0), (50, 0.9, 0.02), (30000, 0.97, 0.0),
               (300, 0.8, 0.3), (-3, 1.5, -1.0)]
    x = rows(rng, kind, len(filters), vocab, bf16)
    k, p, m = (list(v) for v in zip(*filters))
    for temperature in (1.0, 0.3):
        t, u = [temperature] * len(filters), rng.random(len(filters)).astype(np.float32)
        check(sample(x, t, k, p, m, u, bf16), x, t, k, p, m, u)


def test_temperatures_and_random_numbers_at_their_ends():
    rng = np.random.default_rng(5)
    t = [1e-30, 1e-3, 1e3, 1e38, np.inf, 0.0, -1.0, np.nan, 1e-40, 1.0, 1.0, 1.0, 1.0]
    n = len(t)
    u = [0.3, 0.6, 0.5, 0.5, 0.25, 0.5, 0.5, 0.5, 0.9, 0.0, 1 - 2.0 ** -24, 1.0, 0.0]
    x = rows(rng, "normal", n, 9001, False)
    for k, p, m in (([0] * n, [1.0] * n, [0.0] * n), ([100] * n, [0.9] * n, [0.01] * n), ([0] * n, [0.99] * n, [0.0] * n)):
        check(sample(x, t, k, p, m, u, False), x, t, k, p, m, u)


@pytest.mark.parametrize("bf16", [False, True])
def test_every_border_of_equal_weights(bf16):
    """Sums that are equal to a border: the token after it is drawn, and top-p's last token is the one that reaches it."""
    x = np.full((17, 16), 3.0, np.float32)
    u = np.arange(17) / 16
    got = sample(x, None, None, None, None, u, bf16)
    assert got[0].tolist() == list(range(16)) + [15] and (got[1] == 16).all()
    p = np.arange(17) / 16
    got = sample(x, None, None, p, None, np.full(17, 1 - 2.0 ** -24), bf16)
    assert got[1].tolist() == [1] + list(range(1, 17)) and got[0].tolist() == [0] + list(range(16))


def test_none_of_the_arrays_and_rows_that_start_anywhere():
    rng = np.random.default_rng(6)
    for bf16 in (False, True):
        for shift in (1, 3):
            x = rows(rng, "model", 3, 8195, bf16)
            u = rng.random(3).astype(np.float32)
            check(sample(x, None, None, None, None, u, bf16, stride=8201, shift=shift), x, None, None, None, None, u)
            check(sample(x, None, [5, 0, 70], [0.9] * 3, None, u, bf16, stride=8201, shift=shift, probs=False), x, None, [5, 0, 70], [0.9] * 3, None, u)


@pytest.mark.parametrize("kind", ["normal", "steps", "masked"])
def test_as_many_as_are_put_in_order_and_more(kind):
    """Numbers of tokens around those at which the rows' kernel goes another way, by k alone, with top-p and with min-p, and by min-p alone."""
    rng = np.random.default_rng(60 + len(kind))
    k = [127, 128, 129, 255, 256, 257, 300, 383, 447, 448, 449, 511, 512, 513, 640, 641]
    n = len(k)
    x, u = rows(rng, kind, n, 24001, False), rng.random(n).astype(np.float32)
    for t, p, m in ((0.25, 1.0, 0.0), (1.0, 0.97, 0.0), (1.0, 1.0, 0.01), (3.0, 0.9, 0.05)):
        check(sample(x, [t] * n, k, [p] * n, [m] * n, u, False), x, [t] * n, k, [p] * n, [m] * n, u)
    m = [float(f) for f in np.exp(-np.linspace(2, 9, n))]
    check(sample(x, None, None, None, m, u, False), x, None, None, None, m, u)


def test_what_lies_between_rows_of_shares_is_left_alone():
    rng = np.random.default_rng(61)
    n, vocab, apart = 4, 8197, 8200
    x, u = rows(rng, "model", n, vocab, False), dev(rng.random(n).astype(np.float32))
    k, p = dev(np.array([0, 20, 0, 1], np.int32)), dev(np.array([1, 1, 0.9, 1], np.float32))
    out, tokens = dzeros(4 * n * apart, 0xEE), dzeros(4 * n)
    hip.launch_sample_rows(dev(x), None, k, p, None, u, n, vocab, vocab, False, tokens, probs=out, probs_stride=apart,
                           workspace=dzeros(hip.sample_rows_workspace_bytes(n, vocab)))
    out = back(out, np.uint32).reshape(n, apart)
    assert (out[:, vocab:] == 0xEEEEEEEE).all()
    assert np.abs(out[:, :vocab].copy().view(np.float32).sum(1, dtype=np.float64) - 1).max() < 2.0 ** -20


def test_one_row_for_many_draws():
    """Stride 0: how often a token is drawn is its share, u going evenly through [0, 1)."""
    rng = np.random.default_rng(7)
    x = rows(rng, "model", 1, 32001, True)
    n = 512
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens = dzeros(4 * n)
    work = dzeros(hip.sample_rows_workspace_bytes(n, 32001))
    p = dev(np.full(n, 0.9, np.float32))
    hip.launch_sample_rows(dev(as_bits(x, True)), None, None, p, None, dev(u), n, 32001, 0, True, tokens, workspace=work)
    got = back(tokens, np.int32)
    share = sample_row(x[0], 1.0, 0, float(np.float32(0.9)), 0.0, 0.0)[2]
    assert (np.diff(got) >= 0).all()
    assert (np.abs(np.bincount(got, minlength=32001) - share * n) <= 1 + 1e-9).all()


@pytest.mark.parametrize("vocab,bf16,kind", [(131072, True, "model"), (131072, False, "normal"), (200003, False, "narrow"), (2 ** 21, True, "normal"),
                                             (2 ** 21, False, "equal")])
def test_large_rows(vocab, bf16, kind):
    n = 3 if vocab < 2 ** 20 else 2
    rng = np.random.default_rng(vocab)
    x = rows(rng, kind, n, vocab, bf16)
    u = rng.random(n).astype(np.float32)
    for k, p, m in (([0] * n, [1.0] * n, [0.0] * n), ([64] * n, [0.95] * n, [0.02] * n), ([0] * n, [0.9] * n, [0.0] * n)):
        check(sample(x, [0.9] * n, k, p, m, u, bf16), x, [0.9] * n, k, p, m, u)


def test_shares_are_what_verification_takes():
    """A chain of drafts drawn from the draft rows' own shares, judged against the target's: a draft row that is the target's is always accepted."""
    rng = np.random.default_rng(8)
    seqs, nodes, vocab = 4, 5, 32001
    n = seqs * nodes
    x = dev(rows(rng, "model", n, vocab, False))
    p, u = dev(np.full(n, 0.95, np.float32)), dev(rng.random(n).astype(np.float32))
    drawn, probs = dzeros(4 * n), dzeros(4 * n * vocab)
    work = dzeros(hip.sample_rows_workspace_bytes(n, vocab))
    hip.launch_sample_rows(x, None, None, p, None, u, n, vocab, vocab, False, drawn, probs=probs, probs_stride=vocab, workspace=work)
    drawn = back(drawn, np.int32).reshape(seqs, nodes)
    tokens = np.zeros((seqs, nodes), np.int32)
    tokens[:, 1:] = drawn[:, :-1]                    # node i is what was drawn after node i - 1
    parents = np.tile(np.arange(-1, nodes - 1, dtype=np.int32), (seqs, 1))
    path, n_path, following = dzeros(4 * n), dzeros(4 * seqs), dzeros(4 * seqs)
    room = dzeros(max(16, hip.draft_verify_workspace_bytes(seqs, nodes, vocab)))
    accept, last = dev(rng.random(n).astype(np.float32)), rng.random(seqs).astype(np.float32)
    hip.launch_draft_verify(probs, probs, dev(tokens), dev(parents), dev(np.arange(0, n + 1, nodes, dtype=np.int32)), accept, dev(last), seqs, n, nodes,
                            vocab, vocab, vocab, False, path, n_path, following, room)
    assert (back(n_path, np.int32) == nodes).all()
    share = back(probs, np.float32).reshape(seqs, nodes, vocab).astype(np.float64)
    for s in range(seqs):
        upto = np.cumsum(share[s, -1])
        assert back(following, np.int32)[s] == np.nonzero(upto > last[s] * upto[-1])[0][0]


def test_a_captured_draw_replays_and_two_streams_do_not_meet():
    torch = torch_cuda()
    rng = np.random.default_rng(9)
    n, vocab = 9, 32001
    x = [rows(rng, kind, n, vocab, True) for kind in ("model", "normal", "narrow", "equal")]
    t, k, p = [1.0] * 8 + [0.0], [0, 7, 100, 0, 20000, 0, 3, 0, 0], [0.9, 1, 0.95, 1, 0.9, 0.3, 0.99, 1, 1]
    u = rng.random(n).astype(np.float32)
    args = dev(np.asarray(t, np.float32)), dev(np.asarray(k, np.int32)), dev(np.asarray(p, np.float32)), None, dev(u)

    class Side:
        def __init__(self):
            self.x = dev(as_bits(x[0], True))
            self.tokens, self.kept, self.logprobs, self.probs = dzeros(4 * n), dzeros(4 * n), dzeros(4 * n), dzeros(4 * n * vocab)
            self.work = dzeros(hip.sample_rows_workspace_bytes(n, vocab))

        def go(self):
            hip.launch_sample_rows(self.x, *args, n, vocab, vocab, True, self.tokens, self.kept, self.logprobs, self.probs, vocab, self.work,
                                   torch.cuda.current_stream())

        def result(self):
            return (back(self.tokens, np.int32), back(self.kept, np.int32), back(self.logprobs, np.float32).astype(np.float64),
                    back(self.probs, np.float32).reshape(n, vocab).astype(np.float64))

    one, two = Side(), Side()
    one.go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.go()
    other = torch.cuda.Stream()
    for i in (1, 2, 3):
        one.x.copy_(dev(as_bits(x[i], True)))
        two.x.copy_(dev(as_bits(x[(i + 1) % 4], True)))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            two.go()
        torch.cuda.synchronize()
        check(one.result(), x[i], t, k, p, None, u)
        check(two.result(), x[(i + 1) % 4], t, k, p, None, u)
