"""Norm and rotation of a token's rows in one pass (rivoli_norm_rope_rows, rivoli_kv_norm_append_paged) against the
formulas in 64 bits."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import BF16, F32, e4m3_values
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.util import bf16_to_f32, f32_to_bf16_rne

pytestmark = pytest.mark.gpu

EPS = float(np.float32(1e-6))
# A value's way in 32 bits, in half steps: a row's sum of up to 1 024 squares by 22 additions in turn and six more across lanes, half of which reaches
# the root, with the division and the root 16; the mean 28 of the mean size; the difference, two products and a sum 4; the turn 2.
SLACK = 56 * F32


def table_of(n, rd):
    at = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, rd, 2) / rd)
    return np.stack([np.cos(at), np.sin(at)], -1).astype(np.float32).reshape(n, rd)


def normed(x, weight, bias, table, positions, norm_n, rope_at, rd, center, half):
    """[tokens][heads][width] f32 -> the rows in 64 bits, and by how much 32 bits may be off them."""
    x = x.astype(np.float64)
    z = x[..., :norm_n]
    c = z.mean(-1, keepdims=True) if center else 0.0
    r = 1 / np.sqrt(((z - c) ** 2).mean(-1, keepdims=True) + EPS)
    w = np.broadcast_to(np.float64(1) if weight is None else weight.astype(np.float64), x.shape[1:2] + (norm_n,))
    b = np.broadcast_to(np.float64(0) if bias is None else bias.astype(np.float64), x.shape[1:2] + (norm_n,))
    y, far = x.copy(), np.abs(x) * 0
    y[..., :norm_n] = (z - c) * r * w + b
    far[..., :norm_n] = np.abs(z - c) * r * np.abs(w) + np.abs(b)
    if center:
        far[..., :norm_n] += np.abs(z).mean(-1, keepdims=True) * r * np.abs(w)
    if rd:
        far[..., rope_at:rope_at + rd] += np.abs(y[..., rope_at:rope_at + rd])
        turn = table[np.clip(positions, 0, len(table) - 1)].astype(np.float64).reshape(len(x), 1, rd // 2, 2)
        i, j = (np.arange(rd // 2), np.arange(rd // 2) + rd // 2) if half else (np.arange(0, rd, 2), np.arange(1, rd, 2))
        i, j, (c, s) = i + rope_at, j + rope_at, (turn[..., 0], turn[..., 1])
        y[..., i], y[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
        far[..., i], far[..., j] = far[..., i] * abs(c) + far[..., j] * abs(s), far[..., i] * abs(s) + far[..., j] * abs(c)
    return y, SLACK * far


def inputs(seed, tokens, heads, width, norm_n, rd, bf16, plain=False, per_head=False):
    rng = np.random.default_rng(seed)
    x = (rng.normal(size=(tokens, heads, width)) * np.exp(rng.normal(size=(tokens, heads, 1))) + 0.2).astype(np.float32)
    x = bf16_to_f32(f32_to_bf16_rne(x)) if bf16 else x
    shape = (heads, norm_n) if per_head else (norm_n,)
    weight, bias = (None, None) if plain else ((1 + 0.3 * rng.normal(size=shape)).astype(np.float32), (0.2 * rng.normal(size=shape)).astype(np.float32))
    return x, weight, bias, table_of(97, max(rd, 2)), rng.integers(0, 97, tokens).astype(np.int32)


def bits(x, bf16):
    return f32_to_bf16_rne(x) if bf16 else x


def opt(a):
    return None if a is None else dev(a)


def check(got, want, far, bf16):
    far = far + (BF16 if bf16 else F32) * (np.abs(want) + far)
    off = np.abs(got - want)
    assert (off <= far).all(), (np.argwhere(off > far)[:5], (off > far).sum(), (off / np.maximum(far, 1e-30)).max())


@pytest.mark.parametrize("x_bf16,out_bf16", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("tokens,heads,width,norm_n,rope_at,rd,center,half,kind", [
    (1, 1, 8, 8, 0, 8, False, False, "weights"),           # one piece
    (1, 16, 128, 128, 64, 64, False, False, "weights"),    # a token's heads
    (5, 7, 128, 128, 0, 64, True, True, "weights"),        # heads that are no multiple of what a thread has, a mean
    (33, 4, 192, 128, 128, 64, False, True, "per head"),   # the part that is turned is not normed; weights of each head
    (3, 3, 96, 96, 32, 32, False, False, "plain"),         # twelve pieces in sixteen lanes, no weights
    (9, 2, 576, 512, 512, 64, False, True, "weights"),     # more than 512 values: two steps
    (2, 5, 1024, 1024, 480, 64, True, True, "weights"),    # halves that meet across the steps
    (4, 3, 640, 640, 0, 640, False, True, "weights"),      # all of it turned
    (6, 6, 256, 200, 0, 0, True, False, "weights"),        # nothing turned
    (7, 3, 70, 70, 10, 30, False, True, "weights"),        # off the 16 bytes: by ones
    (7, 3, 71, 33, 31, 6, True, False, "per head"),
    (2, 2, 1023, 1023, 1, 1022, False, False, "plain"),
    (2, 2, 1, 1, 0, 0, False, False, "weights"),
])
def test_rows_against_the_formula(tokens, heads, width, norm_n, rope_at, rd, center, half, kind, x_bf16, out_bf16):
    x, weight, bias, table, positions = inputs(width + heads, tokens, heads, width, norm_n, rd, x_bf16, kind == "plain", kind == "per head")
    out = dzeros(tokens * heads * width * (2 if out_bf16 else 4), 0xEE)
    hip.launch_norm_rope_rows(dev(bits(x, x_bf16)), out, opt(weight), opt(bias), dev(table) if rd else None, dev(positions) if rd else None, None,
                              tokens, heads, width, norm_n, rope_at, rd, 97 if rd else 0, 0, heads * width, width, heads * width, width,
                              norm_n if kind == "per head" else 0, EPS, center, half, x_bf16, out_bf16)
    got = bf16_to_f32(back(out, np.uint16)) if out_bf16 else back(out, np.float32)
    want, far = normed(x, weight, bias, table, positions, norm_n, rope_at, rd, center, half)
    check(got.reshape(x.shape).astype(np.float64), want, far, out_bf16)


@pytest.mark.parametrize("width,bf16", [(128, True), (66, False)])
def test_strides_in_place_and_what_lies_between(width, bf16):
    """Heads of a wider row, turned where they are: what lies between and behind them stays."""
    tokens, heads, row, token = 11, 5, width + 8, 5 * (width + 8) + 24
    rng = np.random.default_rng(3)
    all_of = rng.normal(size=tokens * token).astype(np.float32)
    all_of = bf16_to_f32(f32_to_bf16_rne(all_of)) if bf16 else all_of
    at = np.arange(tokens)[:, None, None] * token + np.arange(heads)[:, None] * row + np.arange(width)
    _, weight, bias, table, positions = inputs(1, tokens, heads, width, width, 32, bf16)
    buf = dev(bits(all_of, bf16))
    hip.launch_norm_rope_rows(buf, buf, dev(weight), dev(bias), dev(table), dev(positions), None, tokens, heads, width, width, 16, 32, 97, 0,
                              token, row, token, row, 0, EPS, False, True, bf16, bf16)
    got = bf16_to_f32(back(buf, np.uint16)) if bf16 else back(buf, np.float32)
    want, far = normed(all_of[at], weight, bias, table, positions, width, 16, 32, False, True)
    check(got[at].astype(np.float64), want, far, bf16)
    rest = np.ones(len(all_of), bool)
    rest[at.reshape(-1)] = False
    assert (got[rest] == all_of[rest]).all()


@pytest.mark.parametrize("width", [128, 60])
def test_index_keys_by_slot(width):
    """f32 keys into the paged bf16 keys: padding, slots and positions out of range are left out, counted once, and nothing else changes."""
    tokens, slots_there = 41, 64
    x, weight, bias, table, positions = inputs(9, tokens, 1, width, width, 32, False)
    rng = np.random.default_rng(4)
    slots = rng.permutation(slots_there)[:tokens].astype(np.int32)
    slots[3], slots[8], slots[9], positions[5], positions[6], positions[3] = -1, slots_there, 2 ** 31 - 1, 97, -1, 97
    held = f32_to_bf16_rne(rng.normal(size=(slots_there, width)).astype(np.float32))
    kpool, bad = dev(held), dzeros(4)
    hip.launch_norm_rope_rows(dev(x), kpool, dev(weight), dev(bias), dev(table), dev(positions), dev(slots), tokens, 1, width, width, 0, 32, 97,
                              slots_there, width, width, width, width, 0, EPS, True, True, False, True, bad)
    assert back(bad, np.uint32)[0] == 4
    got = back(kpool, np.uint16).reshape(slots_there, width)
    want, far = normed(x, weight, bias, table, positions, width, 0, 32, True, True)
    live = (slots >= 0) & (slots < slots_there) & (positions >= 0) & (positions < 97)
    check(bf16_to_f32(got[slots[live]]).astype(np.float64), want[live, 0], far[live, 0], True)
    rest = np.setdiff1d(np.arange(slots_there), slots[live])
    assert (got[rest] == held[rest]).all()


def test_rows_of_zeros_infinities_and_nans_stay_with_themselves():
    x, weight, bias, table, positions = inputs(2, 6, 4, 128, 128, 64, False)
    x[1, 2], x[3, 1, 5], x[4, 0, 127] = 0.0, np.inf, np.nan
    for bf16 in (False, True):
        out = dzeros(x.size * 4)
        hip.launch_norm_rope_rows(dev(bits(x, False)), out, dev(weight), dev(bias), dev(table), dev(positions), None, 6, 4, 128, 128, 0, 64, 97, 0,
                                  512, 128, 512, 128, 0, EPS, False, bf16, False, False)
        got = back(out, np.float32).reshape(x.shape)
        clean = np.ones((6, 4), bool)
        clean[3, 1] = clean[4, 0] = False
        want, far = normed(np.where(clean[..., None], x, 1), weight, bias, table, positions, 128, 0, 64, False, bf16)
        check(got[clean].astype(np.float64), want[clean], far[clean], False)
        assert np.isnan(got[4, 0]).all() and np.isnan(got[3, 1]).any()


def nearest_codes(v):
    """The 8-bit codes nearest to a row's values under its scale, in 64 bits: the even one of two, below 2^-6 the larger."""
    top = np.abs(v).max()
    q = np.abs(v) * (448 / top) if top > 0 else np.abs(v)
    values = e4m3_values()[:127].astype(np.float64)
    middles = (values[1:] + values[:-1]) / 2
    low, high = np.searchsorted(middles, q), np.searchsorted(middles, q, side="right")  # (they differ at a middle alone)
    code = np.where((low % 2 == 0) & (q >= 2.0 ** -6), low, high)
    return np.where(np.signbit(v), code + 128, code).astype(np.uint8)


@pytest.mark.parametrize("tokens,half,bf16", [(6000, True, True), (6000, False, False), (2000, False, True), (1900, True, False)])
def test_codes_next_to_a_middle(tokens, half, bf16):
    """A few of a million quotients lie where sums in 32 bits decide: the codes are those of 64."""
    x, weight, _, table, positions = inputs(40 + tokens, tokens, 1, 576, 512, 64, bf16)
    x[5, 0, 512:576], x[6] = np.where(np.arange(64) % 2, 1.0, 1 + 2.0 ** -6), np.float32(2.0 ** 66) * (1 + np.arange(576) % 3)  # products that cancel; squares past 32 bits
    slots, n_pages = np.arange(tokens, dtype=np.int32), -(-tokens // 64)
    pool = dev(np.zeros((n_pages, 64 * 580), np.uint8))
    hip.launch_kv_norm_append_paged(dev(bits(x, bf16)), dev(slots), dev(weight), dev(table), dev(positions), pool, tokens, 576, 512, 64, 97, 64, n_pages, EPS,
                                    half, bf16, None)
    got = back(pool).reshape(n_pages, -1)[:, :64 * 576].reshape(-1, 576)[:tokens]
    want, _ = normed(x, weight, None, table, positions, 512, 512, 64, False, half)
    off = [t for t in range(tokens) if not (got[t] == nearest_codes(want[t, 0])).all()]
    assert off == []


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens,kvl,rope,page,half,weighted", [
    (1, 512, 64, 64, False, True), (32, 512, 64, 64, True, True), (777, 512, 64, 48, False, True), (5, 512, 64, 16, False, False),
    (9, 384, 64, 64, True, True), (9, 8, 8, 4, False, True), (6, 960, 64, 64, True, True), (6, 240, 272, 32, True, True),
])
def test_append_against_the_formula_and_the_rule(tokens, kvl, rope, page, half, weighted, bf16):
    """Scales to their rounding, codes the nearest of the quotients, as in 64 bits."""
    width, n_pages = kvl + rope, -(-tokens // page) + 2
    x, weight, _, table, positions = inputs(tokens, tokens, 1, width, kvl, rope, bf16)
    if tokens > 5:
        x[2], x[3, 0, :kvl] = 0.0, 0.0               # nothing in it; nothing to be normed
    weight = weight if weighted else None
    rng = np.random.default_rng(8)
    slots = rng.permutation(n_pages * page)[:tokens].astype(np.int32)
    bad_ones = tokens > 20
    if bad_ones:
        slots[4], slots[7], positions[9], slots[11], positions[11] = -1, n_pages * page, 97, -5, -1
    held = rng.integers(0, 256, (n_pages, page * (width + 4)), dtype=np.uint8)
    pool, bad = dev(held), dzeros(4)
    hip.launch_kv_norm_append_paged(dev(bits(x, bf16)), dev(slots), opt(weight), dev(table), dev(positions), pool, tokens, width, kvl, rope, 97,
                                    page, n_pages, EPS, half, bf16, bad)
    assert back(bad, np.uint32)[0] == (2 if bad_ones else 0)
    got = back(pool).reshape(n_pages, -1)
    want, _ = normed(x, weight, None, table, positions, kvl, kvl, rope, False, half)
    expect = held.copy()
    for t in range(tokens):
        if not (0 <= slots[t] < n_pages * page and 0 <= positions[t] < 97):
            continue
        pg, off = divmod(int(slots[t]), page)
        scale_at = slice(page * width + 4 * off, page * width + 4 * off + 4)
        scale = got[pg, scale_at].view(np.float32)[0]
        v = want[t, 0]
        top = np.abs(v).max() or 448.0
        assert abs(float(scale) * 448.0 - top) <= F32 * top * (1 + 2.0 ** -20)
        expect[pg, off * width:(off + 1) * width] = nearest_codes(v)
        expect[pg, scale_at] = np.float32(scale).reshape(1).view(np.uint8)
    assert (got == expect).all()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("half", [True, False])
def test_a_prompts_rows_are_those_of_its_parts(half, bf16):
    """Many tokens take another kernel: every token's row is the same to the bit, whatever the call it comes in."""
    tokens, page = 2500, 48
    x, weight, _, table, positions = inputs(11, tokens, 1, 576, 512, 64, bf16)
    x[7], x[8, 0, :512], x[9, 0, 100], x[10, 0, 540], x[11] = 0.0, 0.0, np.inf, np.nan, x[11] * 1e-30
    rng = np.random.default_rng(12)
    n_pages = -(-tokens // page) + 2
    slots = rng.permutation(n_pages * page)[:tokens].astype(np.int32)
    slots[4], slots[2100], positions[9], slots[2499], positions[2300] = -1, n_pages * page, 97, -5, -1
    held = rng.integers(0, 256, n_pages * page * 580, dtype=np.uint8)
    xs, w, tb = dev(bits(x, bf16)), dev(weight), dev(table)
    pos, at = dev(positions), dev(slots)
    size = 576 * (2 if bf16 else 4)

    def append(pool, bad, lo, hi, weight):
        hip.launch_kv_norm_append_paged(xs.data_ptr() + lo * size, at.data_ptr() + 4 * lo, weight, tb, pos.data_ptr() + 4 * lo, pool, hi - lo, 576, 512, 64,
                                        97, page, n_pages, EPS, half, bf16, bad)

    for weights in (w, None):
        whole, parts, bad, bad_parts = dev(held), dev(held), dzeros(4), dzeros(4)
        append(whole, bad, 0, tokens, weights)
        for lo, hi in ((0, 1), (1, 40), (40, 2048), (2048, tokens)):
            append(parts, bad_parts, lo, hi, weights)
        assert (back(whole) == back(parts)).all()
        assert back(bad, np.uint32)[0] == back(bad_parts, np.uint32)[0] == 3


def test_a_captured_step_replays():
    torch = torch_cuda()
    x, weight, _, table, positions = inputs(5, 32, 1, 576, 512, 64, True)
    xs, w, tb = dev(bits(x, True)), dev(weight), dev(table)
    pos, slots = dev(positions), dev(np.arange(32, dtype=np.int32))
    pool, out, again = dzeros(64 * 580), dzeros(32 * 576 * 2), dzeros(64 * 580)

    def step(pool):
        s = torch.cuda.current_stream()
        hip.launch_norm_rope_rows(xs, out, w, None, tb, pos, None, 32, 1, 576, 512, 512, 64, 97, 0, 576, 576, 576, 576, 0, EPS, False, False, True,
                                  True, None, s)
        hip.launch_kv_norm_append_paged(xs, slots, w, tb, pos, pool, 32, 576, 512, 64, 97, 64, 1, EPS, False, True, None, s)

    step(pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pool)
    for seed in (6, 7):
        x = inputs(seed, 32, 1, 576, 512, 64, True)[0]
        xs.copy_(dev(bits(x, True)))
        graph.replay()
        torch.cuda.synchronize()
        rows = out.clone()
        step(again)
        torch.cuda.synchronize()
        assert (rows == out).all() and (pool[:64 * 580] == again).all()
