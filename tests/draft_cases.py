"""A step of drafted tokens in plain 64-bit numpy, and inputs for it: what the GPU tests of the rotation, the tree
attention, the verification and the commit compare with. Written from the definitions, loop by loop."""
import math

import numpy as np

from tests.util import bf16_to_f32, f32_to_bf16_rne

# what half a step is, relative to a value
BF16, F32 = 2.0 ** -8, 2.0 ** -24


# ---- trees -----------------------------------------------------------------------------------------------

def random_parents(rng, n, back=4):
    return np.array([-1] + [max(0, i - int(rng.integers(1, back + 1))) for i in range(1, n)][: max(n - 1, 0)], np.int32)[:n]


def ancestors(parents):
    """[n][n] bool: j is i or above it."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        if parents[i] >= 0:
            seen[i] = seen[parents[i]]
        seen[i, i] = True
    return seen


def pack_masks(seen, max_nodes):
    """[n][<= max_nodes] bool -> [n][ceil(max_nodes / 32)] u32."""
    out = np.zeros((seen.shape[0], (max_nodes + 31) // 32), np.uint32)
    for j in range(seen.shape[1]):
        out[:, j >> 5] |= seen[:, j].astype(np.uint32) << np.uint32(j & 31)
    return out


# ---- the paged cache -------------------------------------------------------------------------------------

_E4M3 = None


def e4m3_values():
    """The 256 codes' values in 64 bits."""
    global _E4M3
    if _E4M3 is None:
        c = np.arange(256)
        e, m = (c >> 3) & 15, c & 7
        v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
        v[(c & 0x7F) == 0x7F] = np.nan
        _E4M3 = np.where(c & 0x80, -v, v)
    return _E4M3


def random_pool(rng, n_pages, page, width, spread=0.3):
    """Pages as the append leaves them: codes with no NaN among them, positive scales."""
    codes = rng.integers(0, 127, (n_pages, page, width), dtype=np.uint8) | (rng.integers(0, 2, (n_pages, page, width), dtype=np.uint8) << 7)
    # values spread like a normal's, not like the codes: mostly in the upper binades
    codes = np.where((codes & 0x7F) < 64, codes + 48, codes).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] -= 1
    scales = (np.exp(rng.normal(0, spread, (n_pages, page))) / 300).astype(np.float32)
    pool = np.zeros((n_pages, page * (width + 4)), np.uint8)
    pool[:, : page * width] = codes.reshape(n_pages, -1)
    pool[:, page * width:] = scales.view(np.uint8).reshape(n_pages, -1)
    return pool


def rows_of(pool, table, page, width, n):
    """The first n rows of a sequence in 64 bits, and which of them are there."""
    out, there = np.zeros((n, width)), np.zeros(n, bool)
    for t in range(n):
        b = t // page
        if b >= len(table) or not 0 <= table[b] < len(pool):
            continue
        p, o = pool[table[b]], t % page
        scale = p[page * width + 4 * o: page * width + 4 * o + 4].view(np.float32)[0]
        if not scale > 0:
            continue
        out[t] = e4m3_values()[p[o * width:(o + 1) * width]] * np.float64(scale)
        there[t] = True
    return out, there


# ---- tree attention --------------------------------------------------------------------------------------

def tree_attention(qabs, qrope, pool, tables, ctx, cu, masks, page, scale):
    """(clat, lse, bound of clat, bound of lse) in 64 bits; masks: None or [n][words] u32. Rows of no sequence stay NaN. A masked
    token's row is never used.

    The bounds. A product of a bf16 and a code is exact in f32 (8 + 4 bits); a dot of `width` of them in f32, in any order, is off by at
    most width half steps of the sum of magnitudes, the two scalings by three more: d = (width + 3) 2^-24 max_t sum |q k| |scale|. A weight is then
    off by d relative, by 8 steps of its exponential and exponent's argument (|x| < 2^7 in powers of two: 2^-17 relative), and by half a step of 16 bits where
    it meets the values (2^-8, bf16's, is the most that is allowed; fp16's is 2^-11, or 2^-25 of the row's largest); sums of n weights by n half steps. Against mass = sum_t w_t |L_t|:
    |clat error| <= 2^-8 |clat| + (2^-8 + 2 (d + 2^-16 + n 2^-24)) mass;   |lse error| <= d + 2^-16 + n 2^-24 + 2^-22 |lse|."""
    n, H, kvl = qabs.shape
    width = kvl + qrope.shape[2]
    q = np.concatenate([bf16_to_f32(qabs), bf16_to_f32(qrope)], 2).astype(np.float64)
    out, lse = np.full((n, H, kvl), np.nan), np.full((n, H), np.nan)
    far, lse_far = np.zeros((n, H, kvl)), np.zeros((n, H))
    for s in range(len(ctx)):
        held = cu[s + 1] - cu[s]
        rows, there = rows_of(pool, tables[s], page, width, ctx[s] + held)
        for i in range(held):
            node = cu[s] + i
            seen = there.copy()
            for j in range(held):
                sees = j <= i if masks is None else bool(masks[node][j >> 5] >> (j & 31) & 1)
                seen[ctx[s] + j] &= sees
            at = np.flatnonzero(seen)
            if len(at) == 0:
                out[node], lse[node] = 0, -np.inf
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                x = q[node] @ rows[at].T * scale
                top = x.max(1, keepdims=True)
                e = np.exp(x - top)
                total = e.sum(1, keepdims=True)
                out[node] = e @ rows[at, :kvl] / total
                lse[node] = (top + np.log(total))[:, 0]
                d = (width + 3) * F32 * abs(scale) * (np.abs(q[node]) @ np.abs(rows[at]).T).max(1) + 2.0 ** -16 + len(at) * F32
                far[node] = BF16 * np.abs(out[node]) + (BF16 + 2 * d[:, None]) * (e @ np.abs(rows[at, :kvl]) / total)
                lse_far[node] = d + 2.0 ** -22 * np.abs(lse[node])
    return out, lse, far, lse_far


# ---- verification ----------------------------------------------------------------------------------------

def counted(row):
    """Probabilities as they count, in 64 bits."""
    x = np.asarray(row, np.float64)
    x = np.where(np.isnan(x) | (x < 0), 0.0, x)
    return np.minimum(x, np.float64(np.finfo(np.float32).max))


def verify(target, draft, tokens, parents, u, u_final):
    """One sequence: (path, next token); rows of target and draft by node."""
    n, vocab = len(tokens), target.shape[1]
    cur, path = 0, [0]
    w, c = counted(target[0]), 1.0
    for i in range(1, n):
        x = int(tokens[i])
        if not (0 <= parents[i] < i and 0 <= x < vocab) or parents[i] != cur:
            continue
        q = 1.0 if draft is None else counted(draft[cur])[x]
        if float(u[i]) * q * c < w[x]:
            cur = i
            path.append(i)
            w, c = counted(target[i]), 1.0
        elif draft is None:
            c, w = c - w[x], w.copy()
            w[x] = 0
        else:
            w = np.maximum(w - c * counted(draft[cur]), 0)
            c = w.sum()
    if not w.sum() > 0:
        w = counted(target[cur])
    if not w.sum() > 0:
        return path, -1
    upto = np.cumsum(w)
    past = np.flatnonzero(upto > float(u_final) * upto[-1])
    return path, int(past[0]) if len(past) else int(np.flatnonzero(w > 0)[-1])


# ---- rotation --------------------------------------------------------------------------------------------

def frequencies(rd, base, factor=1.0, orig=0, fast=32.0, slow=1.0):
    out = []
    for j in range(rd // 2):
        f = float(base) ** (-2 * j / rd)
        stretched = 1.0
        if orig:
            pair = [rd * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow)]
            low, high = max(math.floor(pair[0]), 0), max(min(math.ceil(pair[1]), rd - 1), 0)
            if high <= low:
                high = low + 0.001
            stretched = min(1.0, max(0.0, (j - low) / (high - low)))
        out.append(f / factor * stretched + f * (1 - stretched))
    return np.array(out)


def rope_table(first, n, rd, base, mscale=1.0, **scaling):
    """[n][rd / 2][2] in 64 bits."""
    angle = (first + np.arange(n, dtype=np.float64))[:, None] * frequencies(rd, base, **scaling)
    return np.stack([np.cos(angle), np.sin(angle)], -1) * mscale


def rotate(x, pairs, half):
    """x [tokens][heads][rd] by pairs [tokens][rd / 2][2]."""
    x, c, s = x.astype(np.float64), pairs[:, None, :, 0], pairs[:, None, :, 1]
    out, m = np.empty_like(x), x.shape[2] // 2
    a, b = (x[..., :m], x[..., m:]) if half else (x[..., ::2], x[..., 1::2])
    if half:
        out[..., :m], out[..., m:] = a * c - b * s, a * s + b * c
    else:
        out[..., ::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    return out


def bf16_rows(rng, shape, scale=1.0):
    return f32_to_bf16_rne((rng.standard_normal(shape) * scale).astype(np.float32))
