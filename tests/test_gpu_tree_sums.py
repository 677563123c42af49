"""Tree attention's sums over as many tokens as a work item may have, where scales are so small that an exponential stands for more than its weight."""
import math

import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import e4m3_values
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.tree_precision import FLOOR, HALF
from tests.util import bf16_to_f32

pytestmark = pytest.mark.gpu


def test_a_sum_of_exponentials_stays_a_number():
    """2^25 tokens a work item, all of them one page's equal rows, under a softmax scale of nothing (which is held to 1e-20): a weight of 2^-96 at most."""
    torch = torch_cuda()
    seqs, H, page, ctx = 256, 64, 1 << 16, 1 << 25
    blocks = ctx // page + 1
    codes = np.random.default_rng(3).integers(0x30, 0x70, 576).astype(np.uint8)
    pool = torch.empty(page * 580, dtype=torch.uint8, device="cuda")
    pool[:page * 576] = dev(codes).repeat(page)
    pool[page * 576:] = torch.full((page,), 2.0 ** -30, device="cuda").view(torch.uint8)
    tables = torch.zeros(seqs * blocks, dtype=torch.int32, device="cuda")
    q = torch.zeros(seqs * H * 512, dtype=torch.bfloat16, device="cuda")
    floats = hip.mla_attend_tree_paged_scratch_floats(seqs, H, seqs, 1, ctx)
    out, lse, partial = dzeros(seqs * H * 1024, 0xEE), dzeros(seqs * H * 4, 0xEE), dzeros(max(floats, 4) * 4, 0xFF)
    hip.launch_mla_attend_tree_paged(q, q, pool, tables, dev(np.full(seqs, ctx, np.int32)), dev(np.arange(seqs + 1, dtype=np.int32)), None, seqs, H, seqs, 1, ctx, blocks,
                                     512, 64, page, 1, 0.0, out, lse, partial)
    got, want = bf16_to_f32(back(out, np.uint16)).reshape(-1, 512).astype(np.float64), e4m3_values()[codes[:512]] * 2.0 ** -30
    # one rounding of the weight, one of the result, an exponential's 2^-22; and the value sums: a matrix instruction adds sixteen tokens' products, of 15 bits each, to
    # f32, so that 2^21 additions are each off by half a step, 2^-24, of a sum that is no larger than the last: 2^-3 in all. (The weights' own sum, of powers of two, is exact.)
    assert (np.abs(got - want) <= (2.0 ** -8 + HALF + FLOOR + 2.0 ** -22 + 2.0 ** -3) * np.abs(want)).all(), (got[0][:4], want[:4])
    assert (np.abs(back(lse, np.float32) - math.log(ctx + 1)) <= 2.0 ** -20 * math.log(ctx + 1) + 90 * 2.0 ** -22).all(), back(lse, np.float32)[:4]
