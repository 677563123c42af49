"""What the attention for groups of sequences (rivoli_mla_attend_tree_shared_paged) writes: its rows, its scratch as the sizing function counts it, and nothing in front of
them or behind, whatever the lengths and borders on the device say."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.gpu_util import back, dev, dzeros
from tests.test_gpu_shared_attend import Shared, many
from tests.util import bf16_to_f32

pytestmark = pytest.mark.gpu

GUARD = 1 << 16                          # bytes in front of a buffer and behind it
FILL = 0xEE


class Guarded:
    def __init__(self, nbytes):
        self.nbytes, self.all = nbytes, dzeros(nbytes + 2 * GUARD, FILL)
        self.at = self.all.data_ptr() + GUARD

    def check(self):
        rest = back(self.all)
        assert (rest[:GUARD] == FILL).all() and (rest[GUARD + self.nbytes:] == FILL).all()
        return rest[GUARD:GUARD + self.nbytes]


def guarded(case):
    """The case's call on buffers with guards: rows, lse, the count."""
    case.buffers()
    floats = hip.mla_attend_tree_shared_paged_scratch_floats(*case.sizes())
    out, lse, partial, bad = (Guarded(n) for n in (case.n * case.H * case.kvl * 2, case.n * case.H * 4, floats * 4, 4))
    case.out, case.lse, case.partial, case.bad = out.at, lse.at, partial.at, bad.at
    bad.all[GUARD:GUARD + 4] = 0
    return out, lse, partial, bad


def after(case, out, lse, partial, bad):
    partial.check()
    return (out.check().view(np.uint16).reshape(case.n, case.H, case.kvl), lse.check().view(np.float32).reshape(case.n, case.H), int(bad.check().view(np.uint32)[0]))


def run(case):
    held = guarded(case)
    case.launch()
    return after(case, *held)


@pytest.mark.parametrize("cu,groups", [([0, 5, 0, 5], [0, 2, 3]), ([5, 0, 3, 5], [2, 0, 3]), ([-4, 9, 2, 5], [-1, 7, 3]), ([0, 2, 4, 5], [3, 2, 1]),
                                       ([0, 2, 4, 1000], [0, 3, 1000]), ([2 ** 31 - 1, -2 ** 31, 0, 5], [-2 ** 31, 2 ** 31 - 1, 0])])
def test_borders_that_are_none_reach_no_other_memory(cu, groups):
    case = Shared(14, [0, 2, 3], [128, 0], [300, 200, 150], [2, 2, 1], 16, masks="chain", behind=2)
    held = guarded(case)
    case.dev[5], case.dev[7] = dev(np.array(cu, np.int32)), dev(np.array(groups, np.int32))
    case.launch()
    after(case, *held)


def test_borders_that_are_none_in_a_call_that_shares():
    """The same of groups that are attended apart, and of more of them than lanes."""
    ctx, nodes = many(32, 1000)
    n = len(nodes)
    for n_groups, borders in ((1, [5, 1]), (1, [-3, 1000]), (3, [0, 40, -1, 32]), (70, list(range(70, -1, -1))), (70, [0, 32] * 35 + [9])):
        for sums in (np.arange(n + 1), np.arange(n, -1, -1), np.arange(n + 1) * 7 - 50, np.where(np.arange(n + 1) % 2, n, 0)):
            case = Shared(15, [0] * n_groups + [n], [1000] * n_groups, ctx, nodes, 8, masks="chain")
            held = guarded(case)
            case.dev[5], case.dev[7] = dev(sums.astype(np.int32)), dev(np.array(borders, np.int32))
            case.launch()
            after(case, *held)


@pytest.mark.parametrize("masks", ["chain", "tree"])
def test_scratch_is_what_the_sizing_function_says(masks):
    """Right calls between guards: small, a whole page of groups, more groups than lanes, a group that is attended apart."""
    ctx, nodes = many(40, 1024, nodes=lambda i: i % 3)
    for case in (Shared(70, [0, 1], [64], [64], [1], 1, masks=masks), Shared(71, [0, 2, 5], [64, 200], [70, 80, 200, 250, 333], [3, 1, 1, 4, 2], 33, masks=masks, behind=1),
                 Shared(72, [0, 40], [1024], ctx, nodes, 8, masks=masks), Shared(73, list(range(71)), [64] * 70, [64 + i for i in range(70)], [1] * 70, 4, masks=masks)):
        case.check(run(case))


def test_rows_beside_codes_that_are_no_number_are_numbers():
    case = Shared(52, [0, 2], [128], [260, 130], [2, 1], 16)
    for t, bad in ((0, 0.0), (63, np.nan), (64, -0.0), (127, -np.inf), (259, 0.0)):
        case.pool[case.tables[0][t // 64]][64 * 576:].view(np.float32)[t % 64] = bad
    case.pool[case.tables[0][1]][0:576:5] = 0x7F             # under a scale of none
    case.pool[case.tables[1][2]][2 * 576:3 * 576:5] = 0x7F   # the second's own row: its answer alone is none
    out, _ = case.check()
    x = bf16_to_f32(out)
    assert np.isfinite(x[:2]).all() and np.isnan(x[2]).any()
