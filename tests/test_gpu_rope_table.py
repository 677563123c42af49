"""The rotation table (rivoli_rope_table) rounded once: every element within half a step of 32 bits of the definition in 64."""
import math

import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import F32, rope_table
from tests.gpu_util import back, dzeros

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,n,rd,base,mscale,scaling", [
    (0, 5000, 64, 1e4, 1.0, {}), (0, 163840, 64, 1e4, 1.25, dict(factor=16.0, orig=4096)), (7, 4099, 64, 1e4, 0.1 * math.log(40) + 1, dict(factor=40.0, orig=4096)),
    (1000000, 333, 128, 5e5, 0.7, dict(factor=8.0)), (0, 300, 1024, 1e4, -1 / 3, {}), (12345, 17, 2, 10.0, 1e-3, {}),
])
def test_a_table_is_rounded_once(first, n, rd, base, mscale, scaling):
    out = dzeros(n * rd * 4, 0xEE)
    names = dict(factor="factor", orig="orig_ctx", fast="beta_fast", slow="beta_slow")
    hip.launch_rope_table(out, first, n, rd, base, mscale=mscale, **{names[k]: v for k, v in scaling.items()})
    held = float(np.float32(mscale))                     # what the call's argument holds
    want = rope_table(first, n, rd, base, held, **scaling)
    # half a step, and an angle's 64 bits: a frequency to 4 half steps (2^-x x of an exponent's error is 0.53 at most), its turns to two, a position's
    # product to one, of up to first + n radians, the same again on this side; sixteen steps of turning of four half steps each
    far = F32 * np.abs(want) + (14 * (first + n) + 64) * 2.0 ** -53 * abs(held)
    off = np.abs(back(out, np.float32).reshape(n, rd // 2, 2).astype(np.float64) - want)
    assert (off <= far).all(), (np.argwhere(off > far)[:5], (off > far).sum(), (off / np.maximum(np.abs(want), 1e-30) / F32).max())
