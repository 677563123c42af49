"""Norm and rotation (rivoli_norm_rope_rows) of heads whose rows have 33 to 64 lanes in one step: 257 to 512 values, as wide as this cache's latent rows."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.gpu_util import back, dev, dzeros
from tests.test_gpu_norm_rope import EPS, bits, check, inputs, normed, opt
from tests.util import bf16_to_f32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x_bf16,out_bf16", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,width,norm_n,rope_at,rd,center,kind", [
    (1, 1, 264, 264, 200, 64, False, "weights"),         # one head of 33 lanes
    (7, 1, 512, 512, 448, 64, True, "weights"),          # one head of all lanes, its end turned
    (7, 2, 512, 512, 0, 512, False, "weights"),          # all of it turned
    (5, 7, 512, 448, 448, 64, False, "per head"),        # an odd number, the part that is turned not normed
    (9, 3, 320, 320, 128, 128, True, "per head"),        # in the middle
    (3, 5, 504, 496, 16, 480, True, "weights"),          # pairs far apart, a border within the row's last lanes
    (4, 4, 384, 256, 240, 64, False, "plain"),           # a turned part across the norm's border
    (3, 16, 512, 512, 64, 0, True, "weights"),           # nothing turned
])
def test_rows_of_many_lanes(tokens, heads, width, norm_n, rope_at, rd, center, kind, half, x_bf16, out_bf16):
    x, weight, bias, table, positions = inputs(width + heads, tokens, heads, width, norm_n, rd, x_bf16, kind == "plain", kind == "per head")
    size = 2 if out_bf16 else 4
    out = dzeros(tokens * heads * width * size + 512, 0xEE)
    hip.launch_norm_rope_rows(dev(bits(x, x_bf16)), out, opt(weight), opt(bias), dev(table) if rd else None, dev(positions) if rd else None, None,
                              tokens, heads, width, norm_n, rope_at, rd, 97 if rd else 0, 0, heads * width, width, heads * width, width,
                              norm_n if kind == "per head" else 0, EPS, center, half, x_bf16, out_bf16)
    assert (back(out)[-512:] == 0xEE).all()
    got = bf16_to_f32(back(out[:-512], np.uint16)) if out_bf16 else back(out[:-512], np.float32)
    want, far = normed(x, weight, bias, table, positions, norm_n, rope_at, rd, center, half)
    check(got.reshape(x.shape).astype(np.float64), want, far, out_bf16)


@pytest.mark.parametrize("bf16", [True, False])
def test_wide_heads_in_place_and_by_slot(bf16):
    tokens, heads, width = 6, 5, 512
    x, weight, bias, table, positions = inputs(21, tokens, heads, width, width, 64, bf16)
    want, far = normed(x, weight, bias, table, positions, width, 448, 64, False, True)
    buf = dev(bits(x, bf16))
    hip.launch_norm_rope_rows(buf, buf, dev(weight), dev(bias), dev(table), dev(positions), None, tokens, heads, width, width, 448, 64, 97, 0,
                              heads * width, width, heads * width, width, 0, EPS, False, True, bf16, bf16)
    got = bf16_to_f32(back(buf, np.uint16)) if bf16 else back(buf, np.float32)
    check(got.reshape(x.shape).astype(np.float64), want, far, bf16)
    slots, bad = np.array([9, -1, 0, 20, 4, 11], np.int32), dzeros(4)
    out = dzeros(12 * heads * width * 2, 0xEE)
    hip.launch_norm_rope_rows(dev(bits(x, bf16)), out, dev(weight), dev(bias), dev(table), dev(positions), dev(slots), tokens, heads, width, width, 448, 64, 97, 12,
                              heads * width, width, heads * width, width, 0, EPS, False, True, bf16, True, bad)
    assert back(bad, np.uint32)[0] == 1
    rows = back(out, np.uint16).reshape(12, heads, width)
    live = (slots >= 0) & (slots < 12)
    check(bf16_to_f32(rows[slots[live]]).astype(np.float64), want[live], far[live], True)
    assert (rows[np.setdiff1d(np.arange(12), slots[live])] == 0xEEEE).all()
