"""Attention for groups of sequences whose first pages are the same (rivoli_mla_attend_tree_shared_paged) against 64 bits,
and against the call that knows nothing of groups."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.gpu_util import back, dev, torch_cuda
from tests.test_gpu_tree_attend import Case

pytestmark = pytest.mark.gpu


class Shared(Case):
    """A batch of groups (cu_groups) with prefix lengths; members' tables name their group's first pages."""

    def __init__(self, seed, groups, prefixes, ctx, nodes, H, **kw):
        super().__init__(seed, ctx, nodes, H, **kw)
        self.groups, self.prefixes = np.array(groups, np.int32), np.array(prefixes, np.int32)
        for lo, hi, p in zip(groups, groups[1:], prefixes):
            if lo < hi:
                self.tables[lo:hi, :p // self.page] = self.tables[lo, :p // self.page]

    def sizes(self):
        return len(self.ctx), len(self.prefixes), self.H, self.n, self.max_nodes, int(self.prefixes.max()), int(self.ctx.max())

    def buffers(self):
        super().buffers()
        floats = hip.mla_attend_tree_shared_paged_scratch_floats(*self.sizes())
        torch = torch_cuda()
        self.partial = torch.full((floats * 4,), 0xFF, dtype=torch.uint8, device="cuda") if floats else None
        self.dev += [dev(self.groups), dev(self.prefixes)]

    def launch(self, stream=None, lse=True, max_ctx=None):
        n_seqs, n_groups, H, n, max_nodes, max_prefix, longest = self.sizes()
        hip.launch_mla_attend_tree_shared_paged(*self.dev, n_seqs, n_groups, H, n, max_nodes, max_prefix, longest if max_ctx is None else max_ctx,
                                                self.tables.shape[1], self.kvl, self.rope, self.page, self.n_pages, self.scale, self.out,
                                                self.lse if lse else None, self.partial, self.bad, stream)


@pytest.mark.parametrize("groups,prefixes,ctx,nodes,H", [
    ([0, 2], [64], [64, 64], [1, 1], 1),                                     # nothing but the prefix and the node itself
    ([0, 4], [128], [130, 200, 128, 191], [1, 1, 1, 1], 16),
    ([0, 3], [300], [300, 301, 400], [1, 2, 5], 20),                         # a prefix that ends inside a page
    ([0, 2, 5], [64, 200], [70, 80, 200, 250, 333], [3, 1, 1, 4, 2], 33),
    ([1, 3], [128], [500, 140, 150, 10], [1, 1, 2, 1], 16),                  # sequences in front of the groups and behind them
    ([0, 4], [256], [256, 100, 300, 0], [1, 1, 1, 1], 16),                   # some that end within the prefix
    ([0, 3], [128], [130, 140, 150], [1, 0, 2], 16),                         # one without nodes
    ([0, 1, 2], [128, 64], [150, 100], [2, 1], 40),                          # groups of one
    ([0, 0, 2, 2], [64, 64, 0], [100, 70], [1, 1], 64),                      # empty ones, one that shares nothing
    ([0, 3], [63], [100, 70, 63], [1, 1, 1], 128),                           # less than a page
    ([0, 40], [192], [192 + 3 * i for i in range(40)], [1 + i % 3 for i in range(40)], 8),
])
@pytest.mark.parametrize("masks", ["chain", "tree", "empty"])
def test_small_groups(groups, prefixes, ctx, nodes, H, masks):
    Shared(len(ctx) * 7 + H, groups, prefixes, ctx, nodes, H, masks=masks).check()


@pytest.mark.parametrize("page", [4, 16, 48, 60, 128, 256])
def test_pages_of_any_size(page):
    Shared(page, [0, 3, 5], [301, 150], [310, 301, 400, 150, 170], [2, 3, 1, 5, 1], 24, page=page).check()


@pytest.mark.parametrize("groups,prefixes,ctx,nodes,H,masks", [
    ([0, 6], [3000], [3000, 3100, 3050, 3001, 3000, 3500], [1] * 6, 16, "chain"),
    ([0, 3, 9], [2000, 1000], [2000, 2500, 2001] + [1000 + 90 * i for i in range(6)], [4, 1, 2, 1, 8, 3, 0, 1, 2], 20, "tree"),
    ([0, 64], [700], [700 + 5 * i for i in range(64)], [1] * 64, 16, "chain"),
    ([0, 2], [4000], [4000, 4100], [3, 2], 128, "empty"),
])
def test_long_and_many(groups, prefixes, ctx, nodes, H, masks):
    case = Shared(len(ctx) * 31 + H, groups, prefixes, ctx, nodes, H, masks=masks)
    first = case.check()
    again = case.run()                                   # the same call: the same bits
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1].view(np.uint32), again[1].view(np.uint32))


@pytest.mark.parametrize("n_groups", [40, 70, 130])
def test_more_groups_than_lanes(n_groups):
    rng = np.random.default_rng(n_groups)
    sizes = rng.integers(0, 4, n_groups)
    sizes[0] = 3
    groups = np.concatenate([[0], np.cumsum(sizes)])
    prefixes = rng.integers(0, 400, n_groups)
    of = np.repeat(np.arange(n_groups), sizes)
    ctx = prefixes[of] + rng.integers(0, 200, len(of))
    Shared(n_groups, [int(x) for x in groups], [int(x) for x in prefixes], [int(x) for x in ctx], [1 + int(x) for x in rng.integers(0, 2, len(of))], 16,
           masks="chain").check()


def many(n, prefix, step=3, at=0, nodes=lambda i: 1):
    """A group large enough for its pages to be attended apart from its sequences' own: (cached rows, nodes) of each."""
    return [prefix + at + step * i for i in range(n)], [nodes(i) for i in range(n)]


@pytest.mark.parametrize("masks", ["chain", "tree", "empty"])
def test_groups_that_pay(masks):
    """Rows of many sequences in shared blocks: some that end within the prefix, begin, or have no nodes; one beside a small group; sequences of no group."""
    ctx, nodes = many(32, 1000)
    Shared(60, [0, 32], [1000], ctx, nodes, 8, masks=masks).check()
    ctx, nodes = many(40, 1024, nodes=lambda i: i % 3)
    ctx[5], ctx[6], ctx[7], nodes[5] = 1023, 100, 0, 2
    more, more_nodes = many(30, 900, at=10, nodes=lambda i: 1 + i % 2)
    Shared(61, [2, 42, 44, 74], [1024, 64, 900], [300, 7] + ctx + [100, 70] + more + [500], [1, 3] + nodes + [1, 1] + more_nodes + [2], 8, masks=masks).check()


@pytest.mark.parametrize("page", [4, 16, 48, 60, 128, 256])
def test_groups_that_pay_in_pages_of_any_size(page):
    ctx, nodes = many(32, 1290, nodes=lambda i: 1 + i % 2)
    Shared(page + 1, [0, 32], [1290], ctx, nodes, 8, page=page).check()


def test_groups_that_pay_among_more_than_lanes():
    rng = np.random.default_rng(62)
    sizes = rng.integers(0, 3, 90)
    sizes[3], sizes[80] = 32, 40
    prefixes = rng.integers(0, 200, 90)
    prefixes[3], prefixes[80] = 1000, 900
    of = np.repeat(np.arange(90), sizes)
    ctx = prefixes[of] + rng.integers(0, 100, len(of))
    Shared(62, [int(x) for x in np.concatenate([[0], np.cumsum(sizes)])], [int(x) for x in prefixes], [int(x) for x in ctx], [1] * len(of), 8, masks="chain").check()


def test_groups_that_pay_whatever_their_scores():
    ctx, nodes = many(32, 1000)
    case = Shared(63, [0, 32], [1000], ctx, nodes, 8, q_scale=1.0)
    scales = case.pool[:, 64 * 576:].view(np.float32)
    for page in range(case.n_pages):
        scales[page] *= np.float32((1.0 if page % 3 else 2.0 ** -12) * (1.0 + page % 7))
    case.qabs[::2] ^= 0x8000
    case.check()
    for scale in (0.0, -0.07, 3.0):
        case = Shared(64, [0, 32], [1000], ctx, nodes, 8)
        case.scale = scale
        case.check()


def test_groups_that_pay_with_rows_that_are_not_there():
    """A shared page outside of the pool is counted once for the group, codes that are no number and scales that are none reach nobody."""
    ctx, nodes = many(32, 1024)
    case = Shared(65, [0, 32], [1024], ctx, nodes, 8)
    case.tables[:, 3] = case.n_pages
    case.tables[2, 16] = -1                              # the rest of the third's rows, 6 and its node
    case.check(bad=64 + 7)
    case = Shared(66, [0, 32], [1024], ctx, nodes, 8)
    for t, bad in ((0, 0.0), (63, np.nan), (64, -0.0), (127, -np.inf)):
        case.pool[case.tables[0][t // 64]][64 * 576:].view(np.float32)[t % 64] = bad
    case.pool[case.tables[0][1]][0:576:5] = 0x7F         # under a scale of none
    case.pool[case.tables[3][16]][1 * 576:2 * 576:5] = 0x7F  # a row of the fourth's own: its answer alone is none
    out, _ = case.check()


def test_groups_that_pay_with_places_that_are_empty():
    """Sequences that are not there (no rows, no nodes, tables of nothing) or are not as far yet, in front of the group's others and among them; a group of such alone."""
    ctx, nodes = many(40, 1024)
    for empty in (0, 1, 7, 39):
        ctx[empty] = nodes[empty] = 0
    ctx[2] = 1023
    case = Shared(80, [0, 40, 42], [1024, 1024], ctx + [0, 1000], nodes + [0, 1], 16)
    for empty in (0, 1, 7, 39, 40):
        case.tables[empty] = -1
    case.tables[2, :3] = case.tables[2, 3:6]             # its own pages in another order
    case.check(bad=0)
    ctx, nodes = many(40, 1024)
    case = Shared(81, [0, 40], [1024], [1000] * 40, nodes, 16)  # as far as nobody is
    case.check(bad=0)


def test_groups_that_pay_from_a_graph_beside_another_stream():
    torch = torch_cuda()
    ctx, nodes = many(32, 1024)
    one, two = (Shared(67 + i, [0, 32, 32], [1024, 0], ctx, nodes, 16, masks="chain") for i in range(2))
    for c in (one, two):
        c.buffers()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        one.launch(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.launch(torch.cuda.current_stream())
    for lens, groups, prefixes in ((ctx, [0, 32, 32], [1024, 0]), ([c + 5 for c in ctx], [0, 16, 32], [1024, 1000]), ([1024] * 31 + [3], [1, 31, 32], [1000, 64])):
        lens = [min(x, max(ctx)) for x in lens]
        for c in (one, two):
            c.ctx, c.groups, c.prefixes = (np.array(x, np.int32) for x in (lens, groups, prefixes))
            for at, x in ((4, c.ctx), (7, c.groups), (8, c.prefixes)):
                c.dev[at].copy_(dev(x))
            c.out.fill_(0xEE)
            c.lse.fill_(0xEE)
        torch.cuda.synchronize()
        graph.replay()
        two.launch(side)
        torch.cuda.synchronize()
        one.check(one.results())
        two.check(two.results())


def test_other_widths_go_sequence_by_sequence():
    Shared(3, [0, 2], [64], [90, 140], [4, 2], 6, kvl=256, rope=32).check()


def test_rows_behind_the_last_sequence_are_left_alone():
    Shared(6, [0, 2], [64], [100, 70], [3, 5], 16, behind=4).check()


def test_scores_that_go_up_and_down():
    """Scales that swing by 2^12 from page to page: references that differ between a group's records and the sequences' own."""
    case = Shared(51, [0, 3], [640], [700, 1200, 650], [2, 1, 1], 24, q_scale=1.0)
    scales = case.pool[:, 64 * 576:].view(np.float32)
    for page in range(case.n_pages):
        scales[page] *= np.float32((1.0 if page % 3 else 2.0 ** -12) * (1.0 + page % 7))
    case.qabs[::2] ^= 0x8000
    case.check()


@pytest.mark.parametrize("scale", [0.0, -0.07, 3.0])
def test_softmax_scales(scale):
    case = Shared(50, [0, 2], [256], [300, 256], [1, 3], 20)
    case.scale = scale
    case.check()


def test_pages_outside_the_pool_are_left_out_and_counted():
    """A small group's rows are attended sequence by sequence, and so counted."""
    case = Shared(8, [0, 3], [192], [200, 250, 300], [1, 1, 1], 40)
    case.tables[:, 1] = case.n_pages
    case.tables[2, 4] = -1
    case.check(bad=3 * 64 + 45)


def test_rows_without_a_scale_and_codes_that_are_no_number():
    case = Shared(52, [0, 2], [128], [260, 130], [2, 1], 16)
    for t, bad in ((0, 0.0), (63, np.nan), (64, -0.0), (127, -np.inf), (259, 0.0)):
        case.pool[case.tables[0][t // 64]][64 * 576:].view(np.float32)[t % 64] = bad
    case.pool[case.tables[1][2]][2 * 576:3 * 576:5] = 0x7F   # the second's own row: its answer alone is none
    out, _ = case.check()
    assert not np.isnan(out[:2].astype(np.uint32).astype(np.float64)).any()


def test_against_the_call_without_groups():
    """Sums in another order, the same sums: as far from each other as two roundings to bf16 and of the weights."""
    case = Shared(13, [0, 5, 8], [1280, 640], [1300, 1400, 1281, 2000, 1350, 700, 640, 900], [1, 2, 1, 1, 3, 1, 1, 2], 16)
    shared = case.run()
    plain = Case.__new__(Case)
    plain.__dict__.update(case.__dict__)
    Case.buffers(plain)
    Case.launch(plain)
    want = plain.results()
    from tests.util import bf16_to_f32
    x, y = bf16_to_f32(shared[0]).astype(np.float64), bf16_to_f32(want[0]).astype(np.float64)
    assert np.linalg.norm(x - y) <= 2 * 2.0 ** -8 * np.linalg.norm(y)
    assert np.abs(shared[1] - want[1]).max() <= 2.0 ** -14 * np.abs(want[1]).max()


def test_two_streams_at_once():
    torch = torch_cuda()
    cases = [Shared(20 + i, [0, 2, 4], [1024, 640], [1500, 1100, 800, 640], [1, 2, 1, 1], 32) for i in range(2)]
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


def test_replayed_from_a_graph_with_lengths_and_groups_that_change():
    torch = torch_cuda()
    case = Shared(30, [0, 3, 4], [2048, 64], [2500, 2100, 2048, 100], [1, 1, 1, 1], 32, masks="chain")
    case.buffers()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        case.launch(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.launch(torch.cuda.current_stream())
    for ctx, groups, prefixes in (([2500, 2100, 2048, 100], [0, 3, 4], [2048, 64]), ([2048, 2300, 2400, 2499], [0, 2, 3], [2048, 1000]),
                                  ([17, 2000, 2048, 0], [0, 3, 3], [640, 0]), ([0, 0, 0, 0], [0, 4, 4], [0, 0])):
        case.ctx, case.groups, case.prefixes = (np.array(x, np.int32) for x in (ctx, groups, prefixes))
        for at, x in ((4, case.ctx), (7, case.groups), (8, case.prefixes)):
            case.dev[at].copy_(dev(x))
        case.out.fill_(0xEE)
        case.lse.fill_(0xEE)
        graph.replay()
        torch.cuda.synchronize()
        case.check(case.results())


def test_borders_that_are_no_prefix_sums_end():
    """Whatever they say, the call ends and writes no row that there is not (its numbers are nobody's business)."""
    for cu, groups in (([0, 5, 0, 5], [0, 2, 3]), ([5, 0, 3, 5], [2, 0, 3]), ([-4, 9, 2, 5], [-1, 7, 3]), ([0, 2, 4, 5], [3, 2, 1])):
        case = Shared(14, [0, 2, 3], [128, 0], [300, 200, 150], [2, 2, 1], 16, masks="chain", behind=2)
        case.buffers()
        case.dev[5], case.dev[7] = dev(np.array(cu, np.int32)), dev(np.array(groups, np.int32))
        case.launch()
        assert back(case.out, np.uint16).reshape(case.n, -1).shape[0] == 7
