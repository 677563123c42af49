"""Which drafts stand (rivoli_draft_verify) against the definition in 64 bits: whole numbers, equal or not."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import random_parents, verify
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.util import bf16_to_f32, f32_to_bf16_rne

pytestmark = pytest.mark.gpu


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


class Case:
    def __init__(self, seed, nodes, vocab, draft, chain=False, bf16=False, pad=0, near=0.8, peaked=1.5):
        rng = np.random.default_rng(seed)
        self.nodes, self.vocab, self.bf16 = list(nodes), vocab, bf16
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.n, self.max_nodes, self.stride = int(self.cu[-1]), max(max(nodes), 1), vocab + pad
        self.parents = np.concatenate([np.arange(-1, m - 1, dtype=np.int32) if chain else random_parents(rng, m) for m in nodes] + [np.zeros(0, np.int32)])
        logits = rng.normal(0, peaked, (max(self.n, 1), self.stride))
        self.target, self.draft = softmax(logits), softmax(logits + rng.normal(0, near, logits.shape)) if draft else None
        self.tokens = np.zeros(max(self.n, 1), np.int32)
        for s, m in enumerate(nodes):
            for i in range(1, m):
                row = self.cu[s] + self.parents[self.cu[s] + i]
                p = (self.draft if draft else self.target)[row, :vocab].astype(np.float64)
                self.tokens[self.cu[s] + i] = rng.choice(vocab, p=p / p.sum())
        self.u, self.u_final = rng.random(max(self.n, 1)).astype(np.float32), rng.random(len(nodes)).astype(np.float32)

    def rows(self, x):
        if x is None:
            return None
        if not self.bf16:
            return x
        with np.errstate(invalid="ignore"):
            return f32_to_bf16_rne(x)

    def buffers(self):
        b = len(self.nodes)
        self.out = [dzeros(b * self.max_nodes * 4, 0xEE), dzeros(b * 4, 0xEE), dzeros(b * 4, 0xEE)]
        bytes_ = hip.draft_verify_workspace_bytes(b, self.max_nodes, self.vocab)
        self.work, self.bad = dzeros(bytes_, 0xFF) if bytes_ else None, dzeros(4)
        t, d = self.rows(self.target), self.rows(self.draft)
        self.dev = [dev(t), None if d is None else dev(d)] + [dev(x) for x in (self.tokens, self.parents if self.n else self.tokens, self.cu, self.u, self.u_final)]

    def launch(self, stream=None):
        hip.launch_draft_verify(*self.dev, len(self.nodes), max(self.n, 1), self.max_nodes, self.vocab, self.stride, self.stride, self.bf16, *self.out,
                                self.work, self.bad, stream)

    def results(self):
        return (back(self.out[0], np.int32).reshape(-1, self.max_nodes), back(self.out[1], np.int32), back(self.out[2], np.int32), int(back(self.bad, np.uint32)[0]))

    def check(self, got=None, bad=0):
        if got is None:
            self.buffers()
            self.launch()
            got = self.results()
        path, n_path, token, counted = got
        t, d = self.rows(self.target), self.rows(self.draft)
        if self.bf16:
            t, d = bf16_to_f32(t), None if d is None else bf16_to_f32(d)
        for s, m in enumerate(self.nodes):
            a, b = self.cu[s], self.cu[s + 1]
            if m == 0:
                want, want_token = [], -1
            else:
                want, want_token = verify(t[a:b, :self.vocab], None if d is None else d[a:b, :self.vocab], self.tokens[a:b], self.parents[a:b],
                                          self.u[a:b], self.u_final[s])
            assert n_path[s] == len(want) and list(path[s]) == want + [-1] * (self.max_nodes - len(want)), (s, path[s], want)
            assert token[s] == want_token, (s, token[s], want_token)
        assert counted == bad
        return path, n_path, token


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab,nodes,chain", [
    (1, [3, 1], False), (2, [5] * 40, False), (7, [8] * 60, False), (64, [16] * 50, True), (511, [9] * 30, False), (513, [4, 0, 1, 7, 12, 3], False),
    (5000, [6] * 20, False), (50021, [5, 3], False), (8192, [40], False), (300, [130, 70, 1], False),
])
@pytest.mark.parametrize("bf16", [False, True])
def test_trees_and_chains(draft, vocab, nodes, chain, bf16):
    Case(vocab + len(nodes), nodes, vocab, draft, chain, bf16, pad=vocab % 3).check()


def test_many_siblings_are_judged_against_residuals():
    """All of a root's children are drawn from one row that differs much from the target's: several rejections in a row."""
    for seed in range(6):
        case = Case(seed, [12] * 20, 97, True, near=3.0)
        case.parents = np.concatenate([[-1] + [0] * 11] * 20).astype(np.int32)
        for s in range(20):
            a = case.cu[s]
            p = case.draft[a, :97].astype(np.float64)
            case.tokens[a:a + 12] = np.random.default_rng(seed * 50 + s).choice(97, 12, p=p / p.sum())
        case.u[:] = np.sqrt(case.u)
        _, n_path, _ = case.check()
        assert (n_path == 1).any() and (n_path == 2).any()


def test_edges_of_the_random_numbers():
    below_one = np.float32(1 - 2.0 ** -24)
    for draft in (False, True):
        for u, u_final in ((0.0, 0.0), (below_one, below_one), (0.0, below_one), (below_one, 0.0)):
            case = Case(3, [6] * 10, 777, draft)
            case.u[:], case.u_final[:] = u, u_final
            case.check()


def test_the_same_token_twice_and_zero_probabilities():
    for draft in (False, True):
        case = Case(4, [7] * 8, 33, draft)
        case.parents = np.concatenate([[-1, 0, 0, 0, 1, 1, 2]] * 8).astype(np.int32)
        case.tokens = np.concatenate([[0, 5, 5, 6, 5, 5, 6]] * 8).astype(np.int32)
        case.target[:, 6] = 0
        if draft:
            case.draft[::2, 5] = 0
        case.check()


def test_nothing_left_of_a_residual():
    """A draft row at least the target's everywhere leaves nothing: the node's own row answers; a row of nothing answers -1."""
    case = Case(5, [3] * 6, 40, True)
    case.draft[:] = np.maximum(case.draft, case.target)
    case.tokens[:] = 7
    case.u[:] = np.float32(1 - 2.0 ** -24)
    case.draft[:, 7] = 2 * case.target[:, 7]
    case.check()
    case.target[:] = 0
    _, _, token = case.check()
    assert (token == -1).all()


def test_what_is_no_probability_counts_as_nothing():
    for draft in (False, True):
        case = Case(6, [6] * 12, 100, draft)
        rng = np.random.default_rng(1)
        for rows in (case.target, case.draft):
            if rows is not None:
                rows[rng.random(rows.shape) < 0.1] = np.nan
                rows[rng.random(rows.shape) < 0.1] = -0.5
        case.check()


def test_nodes_out_of_range_are_nobodys_children():
    case = Case(7, [6, 6, 6], 50, False)
    case.parents[2], case.parents[8], case.parents[13] = 5, -1, 13
    case.tokens[4], case.tokens[9] = 50, -1
    case.check(bad=5)


def test_emitted_tokens_are_distributed_as_the_target():
    """The first token a step emits, over 60 000 steps of three siblings each: five standard deviations of a count."""
    torch_cuda()
    rng = np.random.default_rng(8)
    b, vocab = 60000, 6
    p, q = softmax(rng.normal(0, 1, vocab)), softmax(rng.normal(0, 1, vocab))
    for draft in (False, True):
        case = Case(9, [1], vocab, draft)
        case.nodes, case.n, case.max_nodes = [4] * b, 4 * b, 4
        case.cu = np.arange(0, 4 * b + 1, 4, dtype=np.int32)
        case.parents = np.tile(np.array([-1, 0, 0, 0], np.int32), b)
        case.target = np.tile(p, (4 * b, 1)).astype(np.float32)
        case.draft = np.tile(q, (4 * b, 1)).astype(np.float32) if draft else None
        case.tokens = rng.choice(vocab, 4 * b, p=(q / q.sum(dtype=np.float64)).astype(np.float64) / (q / q.sum(dtype=np.float64)).sum()).astype(np.int32)
        case.u, case.u_final = rng.random(4 * b).astype(np.float32), rng.random(b).astype(np.float32)
        case.buffers()
        case.launch()
        path, n_path, token, _ = case.results()
        first = np.where(n_path > 1, case.tokens[np.arange(b) * 4 + np.maximum(path[:, 1], 0)], token)
        counts = np.bincount(first, minlength=vocab)
        assert (np.abs(counts - b * p) <= 5 * np.sqrt(b * p * (1 - p))).all(), (counts / b, p)


def test_replayed_from_a_graph_and_on_two_streams():
    torch = torch_cuda()
    cases = [Case(50 + i, [8] * 5, 20000, i == 0) for i in range(2)]
    for c in cases:
        c.buffers()
        c.launch()
    torch.cuda.synchronize()
    want = [c.results() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for c, st in zip(cases, streams):
            c.launch(st)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert all(np.array_equal(x, y) for x, y in zip(c.results(), w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cases[0].launch(torch.cuda.current_stream())
    rng = np.random.default_rng(2)
    for _ in range(3):
        cases[0].u[:], cases[0].u_final[:] = rng.random(cases[0].n), rng.random(5)
        cases[0].dev[5].copy_(dev(cases[0].u))
        cases[0].dev[6].copy_(dev(cases[0].u_final))
        graph.replay()
        torch.cuda.synchronize()
        cases[0].check(cases[0].results())


WIDE = 98304 + 1029  # rows that many workgroups share in a call of few sequences; the last block is a part of one


def test_wide_rows_take_a_workspace_in_calls_of_few_sequences():
    assert hip.draft_verify_workspace_bytes(5, 5, WIDE) > 0 and hip.draft_verify_workspace_bytes(64, 3, 49152) > 0


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_wide_rows(draft, bf16):
    Case(60, [3, 0, 4, 1, 2], WIDE, draft, bf16=bf16, pad=1, peaked=3.0).check()


def test_rows_shared_by_workgroups_that_walk_for_themselves():
    """Picked drafts: bad nodes counted once, sequences without nodes, a last workgroup with less than a block a wave."""
    case = Case(68, [7, 0, 5, 9, 1], 49152 + 5 * 1024 + 3, False, bf16=True, pad=2)
    case.parents[3], case.tokens[15] = 6, -1
    case.check(bad=2)


@pytest.mark.parametrize("draft", [False, True])
def test_wide_rows_of_siblings(draft):
    case = Case(61, [6] * 4, WIDE, draft, near=3.0)
    case.parents = np.concatenate([[-1] + [0] * 5] * 4).astype(np.int32)
    case.u[:] = np.float32(1 - 2.0 ** -24)
    _, n_path, _ = case.check()
    assert (n_path == 1).any()


def test_wide_rows_with_nothing_left():
    case = Case(62, [2] * 3, WIDE, True)
    case.draft[:] = np.maximum(case.draft, case.target)
    case.tokens[:] = 7
    case.u[:] = np.float32(1 - 2.0 ** -24)
    case.draft[:, 7] = 2 * case.target[:, 7]
    case.check()
    case.target[-2:] = 0
    _, _, token = case.check()
    assert (token >= 0).tolist() == [True, True, False]


def test_wide_rows_replayed_from_a_graph_and_on_two_streams():
    torch = torch_cuda()
    cases = [Case(63 + i, [3] * 3, WIDE, i == 0) for i in range(2)]
    for c in cases:
        c.buffers()
        c.launch()
    torch.cuda.synchronize()
    want = [c.results() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for c, st in zip(cases, streams):
            c.launch(st)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert all(np.array_equal(x, y) for x, y in zip(c.results()[:3], w[:3]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cases[0].launch(torch.cuda.current_stream())
    rng = np.random.default_rng(3)
    for _ in range(3):
        cases[0].u[:], cases[0].u_final[:] = rng.random(cases[0].n), rng.random(3)
        cases[0].dev[5].copy_(dev(cases[0].u))
        cases[0].dev[6].copy_(dev(cases[0].u_final))
        graph.replay()
        torch.cuda.synchronize()
        cases[0].check(cases[0].results())


@pytest.mark.parametrize("bf16", [False, True])
def test_infinities_and_signalling_nans(bf16):
    """Infinity counts as the largest number of 32 bits, every NaN as nothing, also where conversions would quieten it."""
    case = Case(65, [2] * 8, 500, False, bf16=bf16)
    rows = case.rows(case.target)
    rng = np.random.default_rng(4)
    odd = rng.random(rows.shape) < 0.2
    bits = rows.view(np.uint32) if not bf16 else rows
    bits[odd] = rng.choice([0x7F81, 0x7FFF, 0xFF81, 0xFFC0, 0x7F80, 0xFF80, 0x8000], int(odd.sum())).astype(bits.dtype) << (0 if bf16 else 16)
    case.rows = lambda x: rows if x is not None else None
    case.check()


@pytest.mark.parametrize("draft", [False, True])
def test_the_most_nodes(draft):
    """1024 nodes, the root's children all but one of them and all rejected: as many rejections as there can be."""
    case = Case(66, [1024, 5], 300, draft)
    case.parents[:1024] = [-1] + [0] * 1023
    case.u[:1024] = np.float32(1 - 2.0 ** -24)
    if not draft:                                        # the likeliest token is nobody's
        case.tokens[:1024] = np.where(case.tokens[:1024] == case.target[0, :300].argmax(), 0, case.tokens[:1024])
    _, n_path, _ = case.check()
    assert draft or n_path[0] == 1


@pytest.mark.parametrize("bf16", [False, True])
def test_the_longest_rows(bf16):
    Case(67, [2], 2 ** 21, False, bf16=bf16, peaked=2.0).check()
