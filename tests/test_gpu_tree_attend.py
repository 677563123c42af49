"""Attention of drafted nodes over the paged cache (rivoli_mla_attend_tree_paged) against 64 bits."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import ancestors, bf16_rows, pack_masks, random_parents, random_pool, tree_attention
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.util import bf16_to_f32, shuffled_block_tables

pytestmark = pytest.mark.gpu


class Case:
    """A batch: ctx and nodes by sequence; masks "chain", "tree" or "empty" (trees, and some nodes that see nothing drafted)."""

    def __init__(self, seed, ctx, nodes, H, page=64, kvl=512, rope=64, masks="tree", behind=0, max_nodes=None, q_scale=2.0):
        rng = np.random.default_rng(seed)
        self.ctx, self.H, self.page, self.kvl, self.rope = np.array(ctx, np.int32), H, page, kvl, rope
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.n, self.max_nodes = int(self.cu[-1]) + behind, max_nodes or max(max(nodes), 1)
        blocks = max(1, max(-(-(c + m) // page) for c, m in zip(ctx, nodes)))
        self.n_pages = len(ctx) * blocks + 1
        self.tables = shuffled_block_tables(len(ctx), blocks, self.n_pages, seed)
        self.pool = random_pool(rng, self.n_pages, page, kvl + rope)
        self.qabs, self.qrope = bf16_rows(rng, (self.n, H, kvl), q_scale), bf16_rows(rng, (self.n, H, rope), q_scale)
        self.scale = float(np.float32(1 / np.sqrt(192)))
        self.masks = None
        if masks != "chain":
            seen = np.zeros((self.n, self.max_nodes), bool)
            for s, m in enumerate(nodes):
                seen[self.cu[s]:self.cu[s + 1], :m] = ancestors(random_parents(rng, m))
            if masks == "empty":
                seen[rng.random(self.n) < 0.4] = False
            self.masks = pack_masks(seen, self.max_nodes)

    def buffers(self):
        n_scratch = hip.mla_attend_tree_paged_scratch_floats(len(self.ctx), self.H, self.n, self.max_nodes, int(self.ctx.max()))
        self.out, self.lse, self.bad = dzeros(self.n * self.H * self.kvl * 2, 0xEE), dzeros(self.n * self.H * 4, 0xEE), dzeros(4)
        self.partial = dzeros(n_scratch * 4, 0xFF) if n_scratch else None      # what it holds is nobody's business: NaNs
        self.dev = [dev(x) for x in (self.qabs, self.qrope, self.pool, self.tables, self.ctx, self.cu)]
        self.dev.append(None if self.masks is None else dev(self.masks))

    def launch(self, stream=None, lse=True, max_ctx=None):
        hip.launch_mla_attend_tree_paged(*self.dev, len(self.ctx), self.H, self.n, self.max_nodes, int(self.ctx.max()) if max_ctx is None else max_ctx,
                                         self.tables.shape[1], self.kvl, self.rope, self.page, self.n_pages, self.scale, self.out,
                                         self.lse if lse else None, self.partial, self.bad, stream)

    def results(self):
        return (back(self.out, np.uint16).reshape(self.n, self.H, self.kvl), back(self.lse, np.float32).reshape(self.n, self.H),
                int(back(self.bad, np.uint32)[0]))

    def run(self, **kw):
        self.buffers()
        self.launch(**kw)
        return self.results()

    def check(self, got=None, bad=0):
        out, lse, counted = got or self.run()
        want, want_lse, far, lse_far = tree_attention(self.qabs, self.qrope, self.pool, self.tables, self.ctx, self.cu, self.masks, self.page, self.scale)
        live = self.cu[-1]
        x = bf16_to_f32(out[:live]).astype(np.float64)
        assert np.array_equal(np.isnan(x), np.isnan(want[:live]))
        ok = np.isnan(want[:live]) | (np.abs(x - want[:live]) <= far[:live])
        assert ok.all(), (np.argwhere(~ok)[:5], np.nanmax(np.abs(x - want[:live]) - far[:live]))
        empty = np.isneginf(want_lse[:live])
        assert np.array_equal(np.isneginf(lse[:live]), empty)
        with np.errstate(invalid="ignore"):
            ok = empty | np.isnan(want_lse[:live]) | (np.abs(lse[:live] - want_lse[:live]) <= lse_far[:live])
        assert ok.all(), (np.argwhere(~ok)[:5], lse[:live][~ok][:5], want_lse[:live][~ok][:5])
        assert (out[live:] == 0xEEEE).all() and (lse[live:].view(np.uint32) == 0xEEEEEEEE).all(), "rows of no sequence were written"
        assert counted == bad
        return out, lse


@pytest.mark.parametrize("ctx,nodes,H", [
    ([0], [1], 1), ([1], [1], 16), ([0], [5], 16), ([63], [1], 64), ([64], [1], 128), ([60], [9], 20), ([127, 0, 65, 200], [3, 4, 0, 2], 16),
    ([500, 0, 0, 1, 300], [0, 2, 0, 1, 7], 33), ([130], [64], 8), ([70], [100], 3), ([40, 10], [33, 65], 5), ([200], [7], 129),
])
@pytest.mark.parametrize("masks", ["chain", "tree", "empty"])
def test_small_batches(ctx, nodes, H, masks):
    Case(hash((len(ctx), H, len(masks))) % 1000, ctx, nodes, H, masks=masks).check()


@pytest.mark.parametrize("page", [4, 16, 48, 60, 128, 256])
def test_pages_of_any_size(page):
    Case(page, [150, 0, 301, 64], [5, 9, 1, 12], 24, page=page).check()


@pytest.mark.parametrize("ctx,nodes,H,masks", [
    ([3000], [4], 16, "tree"), ([2000, 5, 900, 0, 1500], [8, 8, 3, 8, 0], 64, "empty"), ([1100], [40], 64, "chain"), ([4000, 3990], [2, 3], 128, "tree"),
    ([700] * 9, [6, 0, 1, 6, 5, 4, 3, 2, 6], 40, "chain"), ([64] * 70, [1] * 70, 16, "chain"),
])
def test_long_and_many(ctx, nodes, H, masks):
    case = Case(len(ctx) * 31 + H, ctx, nodes, H, masks=masks)
    first = case.check()
    again = case.run()                                   # the same call: the same bits
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1].view(np.uint32), again[1].view(np.uint32))


@pytest.mark.parametrize("kvl,rope", [(128, 8), (256, 32), (384, 64), (512, 56)])
def test_other_widths(kvl, rope):
    Case(kvl + rope, [90, 0, 140], [4, 7, 0], 6, kvl=kvl, rope=rope).check()


def test_scores_far_apart_and_growing():
    """Rows whose scores grow along the sequence, by far more than a weight's range from its first tile to its last."""
    case = Case(5, [900], [6], 16)
    scales = case.pool[:, 64 * 576:].view(np.float32)
    for b, page in enumerate(case.tables[0]):
        scales[page] *= np.float32(1.0 + 3.0 * b)
    case.check()


def test_rows_behind_the_last_sequence_are_left_alone():
    Case(6, [100, 30], [3, 5], 16, behind=4).check()


def test_masked_garbage_reaches_nobody():
    """A branch of NaN codes and infinite or zero scales: its own nodes answer for it, the others do not."""
    for bad_scale in (None, np.inf, 0.0, np.nan):
        case = Case(7, [61], [8], 16, masks="tree")
        seen = np.eye(8, dtype=bool)
        seen[:, 0] = True
        seen[5, 3] = True                                # node 5 hangs on node 3
        case.masks = pack_masks(seen, 8)
        for j in (3, 6):
            t = 61 + j
            page = case.pool[case.tables[0][t // 64]]
            page[(t % 64) * 576:(t % 64) * 576 + 576:5] = 0x7F
            if bad_scale is not None:
                page[64 * 576:].view(np.float32)[t % 64] = bad_scale
        out, _ = case.check()
        clean = ~np.isnan(bf16_to_f32(out)).any((1, 2))
        assert clean[[0, 1, 2, 4, 7]].all()
        if bad_scale is None or bad_scale == np.inf:
            assert not clean[[3, 5, 6]].any()


def test_pages_outside_the_pool_are_left_out_and_counted():
    case = Case(8, [200, 100], [6, 3], 40)
    case.tables[0, 1], case.tables[1, 0] = case.n_pages, -1
    case.check(bad=64 + 64)
    chain = Case(9, [200], [6], 40, masks="chain")
    chain.tables[0, 3] = 2 ** 30
    chain.check(bad=200 + 6 - 192)


def test_lengths_are_held_to_what_the_call_says():
    """More cached rows than max_ctx, more nodes than max_nodes, a table too short: what is past counts as absent."""
    case = Case(10, [128, 40], [6, 6], 16, masks="chain", max_nodes=6)
    case.buffers()
    case.launch(max_ctx=100)
    got = case.results()
    case.ctx = np.minimum(case.ctx, 100).astype(np.int32)
    case.check(got)
    case = Case(11, [30], [9], 16, masks="chain", max_nodes=4)
    got = case.run()
    want = Case(11, [30], [9], 16, masks="chain")
    want.cu = np.array([0, 4], np.int32)
    want.check(got)


def test_without_lse():
    case = Case(12, [300], [5], 32)
    want = case.run()
    got = case.run(lse=False)
    assert np.array_equal(want[0], got[0]) and (got[1].view(np.uint32) == 0xEEEEEEEE).all()


def test_two_streams_at_once():
    torch = torch_cuda()
    cases = [Case(20 + i, [1500, 800], [5, 9], 32) for i in range(2)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for c in cases:
        c.buffers()
    torch.cuda.synchronize()
    for _ in range(5):
        for c, st in zip(cases, streams):
            c.launch(st)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        got = c.results()
        assert np.array_equal(got[0], w[0]) and np.array_equal(got[1], w[1])


def test_replayed_from_a_graph_with_lengths_that_change():
    torch = torch_cuda()
    case = Case(30, [2500, 40], [6, 6], 32)
    case.buffers()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        case.launch(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.launch(torch.cuda.current_stream())
    for ctx in ([2500, 40], [17, 2000], [0, 0], [2499, 1234]):
        case.ctx = np.array(ctx, np.int32)
        case.dev[4].copy_(dev(case.ctx))
        case.out.fill_(0xEE)
        case.lse.fill_(0xEE)
        graph.replay()
        torch.cuda.synchronize()
        case.check(case.results())


def test_pool_past_four_gigabytes():
    torch = torch_cuda()
    case = Case(40, [200], [5], 16)
    case.buffers()
    want = case.run()
    far = (1 << 32) // 37120 + 100                       # pages from here on start past 2^32
    big = torch.zeros((far + case.n_pages) * 37120, dtype=torch.uint8, device="cuda")
    big[far * 37120:].copy_(dev(case.pool))
    case.buffers()
    case.dev[2], case.dev[3], case.n_pages = big, dev((case.tables + far).astype(np.int32)), far + case.n_pages
    case.launch()
    got = case.results()
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("seqs,span,H", [(100, 900, 24), (150, 700, 40), (300, 640, 16)])
def test_more_sequences_than_lanes_cut_among_workgroups(seqs, span, H):
    """Ragged batches whose blocks of rows are cut: fewer blocks than workgroups and more, sequences without nodes or rows among them."""
    rng = np.random.default_rng(seqs)
    ctx = rng.integers(0, span, seqs) * (rng.random(seqs) < 0.8)
    nodes = rng.integers(0, 5, seqs)
    ctx[0], nodes[-1], nodes[0] = span, 4, 1
    case = Case(seqs, [int(x) for x in ctx], [int(x) for x in nodes], H, masks="tree" if seqs % 100 else "chain")
    assert hip.mla_attend_tree_paged_scratch_floats(seqs, H, case.n, case.max_nodes, span) > 0
    case.check()


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.07, 3.0])
def test_softmax_scales(scale):
    """Nothing, less than nothing and a lot: even weights, the smallest score first, one row's."""
    case = Case(50, [300, 70], [5, 3], 20)
    case.scale = scale
    case.check()


def test_scores_that_go_up_and_down():
    """Rows' scales that swing by 2^12 from page to page, larger ones later: references are replaced again and again, in some rows only."""
    case = Case(51, [1500, 640], [6, 2], 24, q_scale=1.0)
    scales = case.pool[:, 64 * 576:].view(np.float32)
    for s in range(2):
        for b, page in enumerate(case.tables[s]):
            scales[page] *= np.float32((1.0 if b % 3 else 2.0 ** -12) * (1.0 + b))
    case.qabs[::2] ^= 0x8000                             # every other node's scores have the other sign
    case.check()


def test_cached_rows_without_a_scale_are_left_out():
    case = Case(52, [260], [4], 16)
    for t, bad in ((0, 0.0), (1, -1.0), (63, np.nan), (64, -0.0), (130, -np.inf), (259, 0.0), (261, 0.0)):
        case.pool[case.tables[0][t // 64]][64 * 576:].view(np.float32)[t % 64] = bad
    case.check()


@pytest.mark.parametrize("masks", ["chain", "tree"])
def test_many_nodes(masks):
    """A prompt's worth of nodes behind a prefix that ends inside a page: many words of masks, many blocks of rows."""
    Case(53, [70, 0, 9], [700, 1, 333], 2, masks=masks).check()


def test_a_batch_of_nothing_but_prefixes_and_of_single_tokens():
    case = Case(54, [5000, 0, 1], [0, 0, 1], 16)         # one node in all
    case.check()
    Case(55, [0] * 200, [1] * 200, 128, masks="chain").check()


@pytest.mark.parametrize("ctx,nodes,H", [([700, 300], [6, 3], 16), ([2500], [2], 8)])
def test_scales_of_very_different_rows(ctx, nodes, H):
    """Rows whose scales lie up to 2^16 apart: weights carry them."""
    case = Case(56 + H, ctx, nodes, H)
    rng = np.random.default_rng(9)
    scales = case.pool[:, 64 * 576:].view(np.float32)
    scales *= np.exp2(rng.uniform(-16, 0, scales.shape)).astype(np.float32)
    case.check()
