"""Sampling from logits in plain numpy, in 64 bits and sums in 80, and rows for it."""
import numpy as np

from tests.util import bf16_to_f32, f32_to_bf16_rne

FLT_MAX = np.finfo(np.float32).max


def sample_row(x, t, k, p, m, u):
    """(token, kept, share of every token) of one row of f32 logits, by the definition."""
    t = np.float32(t)
    if t > 0 and t > 2.0 ** -16:
        most = min(float(t) * 2.0 ** 25, float(FLT_MAX))
        x = np.where(x > -most, np.minimum(x.astype(np.float64), most), -np.inf)
    else:
        t, x = np.float32(0), np.where(x > -2.0 ** 25, x.astype(np.float64), -np.inf)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    share = np.zeros(len(x))
    if not len(order):
        return -1, 0, share
    if not t > 0:
        share[order[0]] = 1.0
        return int(order[0]), 1, share
    w = np.exp((x[order] - x[order[0]]).astype(np.longdouble) / np.longdouble(min(float(t), float(FLT_MAX))))
    n = len(order)
    if p <= 0:
        k = 1
    if k > 0:
        n = min(n, int(k))
    if 0 < p < 1:
        upto = np.cumsum(w[:n])
        n = int(np.sum(np.concatenate([[0], upto[:-1]]) < np.longdouble(p) * upto[-1]))
    if m > 0:
        n = max(1, int(np.sum(w[:n] >= np.longdouble(m))))
    weight = np.zeros(len(x), np.longdouble)
    weight[order[:n]] = w[:n]
    upto = np.cumsum(weight)
    past = np.nonzero(upto > np.longdouble(u) * upto[-1])[0]
    token = past[0] if len(past) else np.nonzero(weight)[0][-1]
    return int(token), n, (weight / upto[-1]).astype(np.float64)


def rows(rng, kind, n, vocab, bf16):
    """Logits of a kind, as the f32 values that the call gets."""
    x = rng.normal(size=(n, vocab))
    if kind == "model":                # a broad body and a few dozen tokens above it
        x *= 2
        for r in x:
            at = rng.integers(0, vocab, 40)
            r[at] = np.abs(r[at]) + 4 + rng.exponential(3, 40)
    elif kind == "wide":
        x *= 6
    elif kind == "narrow":             # thousands of tokens are as likely as the first
        x *= 0.01
    elif kind == "equal":
        x[:] = 1.25
    elif kind == "steps":              # many equal ones
        x = np.round(x * 2) * 0.5
    elif kind == "masked":             # what a grammar leaves, the rest at -inf or at the type's lowest value
        keep = rng.random(x.shape) < 0.01
        keep[:, vocab // 2] = True
        x = np.where(keep, x * 3, np.where(np.arange(n)[:, None] % 2 == 0, -np.inf, -3.3895313892515355e38))
    elif kind == "odd":                # values that are none, and infinite ones
        x *= 2
        x[rng.random(x.shape) < 0.1] = np.nan
        x[rng.random(x.shape) < 0.1] = -np.inf
        x[0] = -np.inf
        if n > 1:
            x[1] = np.nan
        if n > 2:
            x[2, rng.integers(0, vocab, 3)] = np.inf
        if n > 3:
            x[3, :] = -0.0
            x[3, ::2] = 0.0
    else:
        assert kind == "normal", kind
        x *= 2.5
    x = x.astype(np.float32)
    if bf16:
        odd = ~np.isfinite(x)
        x = np.where(odd, x, bf16_to_f32(f32_to_bf16_rne(np.where(odd, 0, x))))
    return x


def as_bits(x, bf16):
    """The array that the call gets."""
    return (np.ascontiguousarray(x).view(np.uint32) >> 16).astype(np.uint16) if bf16 else np.ascontiguousarray(x)
