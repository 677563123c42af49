"""Draws (rivoli_sample_rows) from rows whose largest logits lie past 2^25 temperatures, where neighbouring f32 numbers are two temperatures apart and more: by their distances, as
of any other row."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import F32
from tests.gpu_util import dev, dzeros, torch_cuda
from tests.sample_cases import as_bits
from tests.test_gpu_sample import sample

pytestmark = pytest.mark.gpu

FLT_MAX = np.finfo(np.float32).max
FILTERS = [(0, 1.0, 0.0), (1, 1.0, 0.0), (50, 1.0, 0.0), (5000, 1.0, 0.0), (2500, 0.9, 0.0), (20000, 0.97, 0.02), (0, 0.5, 0.0), (0, 0.95, 0.0), (0, 0.999999, 0.0),
           (0, 0.0, 0.0), (0, 1.0, 0.05), (0, 1.0, 1e-7), (300, 0.8, 0.3), (3, 1.0, 0.001)]


def drawn(x, t, k, p, m, u):
    """(token, kept, share of every token, logarithms of shares) of a row by the definition, whatever its logits' size."""
    t = float(np.float32(t))
    x = np.where(x > -2.0 ** 25 * t, np.minimum(x.astype(np.float64), float(FLT_MAX)), -np.inf)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    z = ((x - x[order[0]]) / t).astype(np.longdouble)
    w, n = np.exp(z[order]), len(order)
    if p <= 0:
        k = 1
    if k > 0:
        n = min(n, k)
    if 0 < p < 1:
        upto = np.cumsum(w[:n])
        n = int(np.sum(np.concatenate([[0], upto[:-1]]) < np.longdouble(p) * upto[-1]))
    if m > 0:
        n = max(1, int(np.sum(w[:n] >= np.longdouble(m))))
    weight = np.zeros(len(x), np.longdouble)
    weight[order[:n]] = w[:n]
    upto = np.cumsum(weight)
    return int(np.nonzero(upto > np.longdouble(u) * upto[-1])[0][0]), n, (weight / upto[-1]).astype(np.float64), (z - np.log(upto[-1])).astype(np.float64)


def check(got, x, t, k, p, m, u):
    tokens, kept, logprobs, probs = got
    f32 = lambda a: [float(np.float32(v)) for v in a]  # noqa: E731
    for r, (tr, kr, pr, mr, ur) in enumerate(zip(f32(t), k, f32(p), f32(m), f32(u))):
        token, count, share, logs = drawn(x[r], tr, kr, pr, mr, ur)
        assert (tokens[r], kept[r]) == (token, count), (r, kr, pr, mr)
        # a weight's 2^-29, and among whole numbers half of 2^-42 of the largest a token
        assert abs(logprobs[r] - logs[token]) <= F32 * abs(logs[token]) + 2.0 ** -29 + len(x[r]) * 2.0 ** -43 / (share[token] / share.max()), r
        off = np.abs(probs[r] - share)
        assert (off <= (F32 + len(x[r]) * 2.0 ** -42) * share + 2.0 ** -149).all() and ((probs[r] > 0) <= (share > 0)).all(), r


def far_rows(rng, n, vocab, t, kind, bf16):
    """Logits whose largest are some steps of f32 (bf16: all alike) below a number past 2^25 t, thousands of each, over others of any size."""
    top = np.float32(2.0 ** 25 * t * 1.6)
    step = np.spacing(top)
    assert step >= 2 * t
    x = (np.float64(top) - step * np.floor(rng.exponential(2 if kind == "few steps" else 6, (n, vocab)))).astype(np.float32)
    if kind == "some":
        x = np.where(rng.random((n, vocab)) < 0.002, x, (rng.normal(size=(n, vocab)) * 100 * t).astype(np.float32))
        x[:, vocab // 3] = top
    if kind == "masked":
        x = np.where(rng.random((n, vocab)) < 0.3, x, np.array([-np.inf, np.nan, -FLT_MAX], np.float32)[rng.integers(0, 3, (n, vocab))])
        x[:, vocab // 3] = top
    if bf16:
        x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)
    return x


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["few steps", "many steps", "some", "masked"])
@pytest.mark.parametrize("t", [2.0 ** -15, 1e-4, 1.0, 1.3, 1e20])
def test_rows_past_the_bins(t, kind, bf16):
    rng = np.random.default_rng(len(kind) + 100 + int(np.log2(t)))
    n, vocab = len(FILTERS), 20001
    x = far_rows(rng, n, vocab, t, kind, bf16)
    k, p, m = (list(v) for v in zip(*FILTERS))
    u = rng.random(n).astype(np.float32)
    check(sample(x, [t] * n, k, p, m, u, bf16), x, [t] * n, k, p, m, u)
    x[:, 7:9], x[:, 19000] = np.inf, np.inf              # infinite ones are the largest
    check(sample(x, [t] * n, k, p, m, u, bf16), x, [t] * n, k, p, m, u)


def test_such_rows_beside_others_from_a_graph():
    """Rows of either kind in one call, from a graph whose rows change their kinds; a large row."""
    torch = torch_cuda()
    rng = np.random.default_rng(4)
    n, vocab = 8, 70001
    t, k, p, m = [0.5] * n, [0, 50, 0, 0, 9000, 0, 20, 3000], [1, 1, 0.9, 1, 0.95, 0.5, 0.9, 1], [0, 0, 0, 0.02, 0, 0, 0.01, 0]
    u = rng.random(n).astype(np.float32)
    near, past = (rng.normal(size=(n, vocab)) * 2).astype(np.float32), far_rows(rng, n, vocab, 0.5, "many steps", False)
    args = [dev(np.asarray(a, kind)) for a, kind in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32), (u, np.float32))]
    xs, tokens, kept, logprobs, probs = dev(near), dzeros(4 * n), dzeros(4 * n), dzeros(4 * n), dzeros(4 * n * vocab)
    work = dzeros(hip.sample_rows_workspace_bytes(n, vocab), 0xEE)

    def go():
        hip.launch_sample_rows(xs, *args, n, vocab, vocab, False, tokens, kept, logprobs, probs, vocab, work, torch.cuda.current_stream())

    go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for which in (np.arange(n) % 2 == 0, np.arange(n) % 2 == 1, np.arange(n) < 0):
        x = np.where(which[:, None], past, near)
        xs.copy_(dev(as_bits(x, False)))
        graph.replay()
        torch.cuda.synchronize()
        got = (tokens.cpu().numpy().view(np.int32), kept.cpu().numpy().view(np.int32), logprobs.cpu().numpy().view(np.float32).astype(np.float64),
               probs.cpu().numpy().view(np.float32).reshape(n, vocab).astype(np.float64))
        check(got, x, t, k, p, m, u)
