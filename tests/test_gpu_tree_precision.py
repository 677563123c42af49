"""Tree attention (rivoli_mla_attend_tree_paged) held to the precision of its weights and to every value row being the right one
(tests/tree_precision.py has the bounds)."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.gpu_util import back, dev, dzeros
from tests.test_gpu_tree_attend import Case
from tests.tree_precision import SINK_PAGE, SINK_TOKENS, Sink, check_norm, check_singled_out, single_out
from tests.util import bf16_to_f32

pytestmark = pytest.mark.gpu


def as_long_work_items(qabs, qrope, pool, table, ctx, page, scale):
    """One node's 64 heads over a long prefix, 256 times over the same pages, so that all of it is one work item. [64][512], bf16 as uint16."""
    seqs = 256
    floats = hip.mla_attend_tree_paged_scratch_floats(seqs, 64, seqs, 1, ctx)
    out, partial = dzeros(seqs * 64 * 1024, 0xEE), dzeros(max(floats, 4) * 4, 0xFF)
    every = lambda x: dev(np.broadcast_to(x, (seqs,) + x.shape))
    hip.launch_mla_attend_tree_paged(every(qabs), every(qrope), dev(pool), every(table), dev(np.full(seqs, ctx, np.int32)),
                                     dev(np.arange(seqs + 1, dtype=np.int32)), None, seqs, 64, seqs, 1, ctx, len(table), 512, 64, page, len(pool), scale,
                                     out, None, partial)
    got = back(out, np.uint16).reshape(seqs, 64, 512)
    assert (got == got[0]).all()
    return got[0]


def test_a_dominant_first_token_over_a_long_flat_tail():
    sink = Sink()
    got = as_long_work_items(sink.qabs, sink.qrope, sink.pool, np.arange(sink.pages, dtype=np.int32), SINK_TOKENS, SINK_PAGE, sink.scale)
    sink.check(bf16_to_f32(got).astype(np.float64))


@pytest.mark.parametrize("growth", ["flat", "grow", "swing"])
@pytest.mark.parametrize("ctx", [4300, 40000])
def test_long_work_items_whose_references_move(ctx, growth):
    case = Case(ctx, [ctx], [1], 64, masks="chain")
    own = single_out(case, growth, apart=ctx // 64)
    got = as_long_work_items(case.qabs[0], case.qrope[0], case.pool, case.tables[0], ctx, 64, case.scale)
    check_singled_out(case, own, got[None])


@pytest.mark.parametrize("ctx,nodes,H,kw", [
    ([3000], [4], 16, {}), ([2000, 5, 900, 0, 1500], [8, 8, 3, 8, 0], 64, dict(masks="empty")), ([4000, 3990], [2, 3], 128, {}), ([130], [64], 8, {}),
    ([40, 10], [33, 65], 5, dict(masks="chain")), ([500, 0, 0, 1, 300], [0, 2, 0, 1, 7], 33, dict(masks="chain")), ([150, 0, 301, 64], [5, 9, 1, 12], 24, dict(page=48)),
    ([150, 0, 301, 64], [5, 9, 1, 12], 24, dict(page=60)), ([90, 0, 140], [4, 7, 0], 6, dict(kvl=256, rope=32)),
])
def test_results_are_as_far_off_as_their_own_rounding(ctx, nodes, H, kw):
    case = Case(len(ctx) * 13 + H, ctx, nodes, H, **kw)
    check_norm(case, case.run()[0])


@pytest.mark.parametrize("scale", [0.0, -0.07, 3.0])
def test_so_they_are_under_other_softmax_scales(scale):
    case = Case(60, [300, 70], [5, 3], 20)
    case.scale = scale
    check_norm(case, case.run()[0])


@pytest.mark.parametrize("growth", ["flat", "grow", "swing"])
@pytest.mark.parametrize("ctx,nodes,H,kw", [
    ([700], [6], 128, dict(masks="chain")), ([1000], [9], 120, dict(page=48)), ([2100], [17], 128, dict(masks="chain")), ([333, 0, 512, 65], [4, 2, 5, 1], 128, dict(page=60)),
    ([1500], [13], 128, dict(page=256, masks="chain")), ([400], [8], 64, dict(page=4)), ([300] * 40, [1] * 40, 320, dict(masks="chain")),
    ([200], [5], 50, dict(kvl=256, rope=32)),
])
def test_every_token_is_the_answer_of_some_row(ctx, nodes, H, kw, growth):
    """A value row that is missing, doubled or another token's shows, at the edges of runs, tiles, work items and pages too, whatever the scores do."""
    case = Case(len(ctx) * 17 + H, ctx, nodes, H, **kw)
    own = single_out(case, growth)
    check_singled_out(case, own, case.run()[0])
