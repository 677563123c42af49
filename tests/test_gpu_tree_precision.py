"""Tree attention (rivoli_mla_attend_tree_paged) held to the precision of its weights (tests/tree_precision.py has the bounds)."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.gpu_util import back, dev, dzeros
from tests.tree_precision import SINK_PAGE, SINK_TOKENS, Sink
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
