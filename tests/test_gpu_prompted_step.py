"""Decode steps of a batch that continues one prompt, as an engine strings the calls together: queries, index keys and latent rows normed,
rotated and cached, attention over the shared and the sequences' own pages, tokens drawn; eager and from a graph whose steps feed each other."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import e4m3_values, tree_attention
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.sample_cases import sample_row
from tests.test_gpu_norm_rope import EPS, normed, table_of
from tests.util import bf16_to_f32, f32_to_bf16_rne

pytestmark = pytest.mark.gpu

B, H, V, PT, PROMPT, STEPS, HD = 32, 8, 4001, 64, 1003, 5, 128
BLOCKS, SHARED = (PROMPT + STEPS + PT - 1) // PT, PROMPT // PT
N_PAGES = SHARED + B * (BLOCKS - SHARED)


class Engine:
    """What it owns for its life, and a step's buffers."""

    def __init__(self, seed):
        torch = self.torch = torch_cuda()
        rng = np.random.default_rng(seed)
        order = rng.permutation(N_PAGES).astype(np.int32)
        self.tables = np.concatenate([np.tile(order[:SHARED], (B, 1)), order[SHARED:].reshape(B, -1)], 1).astype(np.int32)
        self.weight, self.q_weight = (1 + 0.2 * rng.normal(size=512)).astype(np.float32), (1 + 0.2 * rng.normal(size=64)).astype(np.float32)
        self.k_weight, self.k_bias = (1 + 0.2 * rng.normal(size=HD)).astype(np.float32), (0.1 * rng.normal(size=HD)).astype(np.float32)
        self.table = table_of(2048, 64)
        # what a token makes of itself: latent row, queries, index key, the logits but for what attention adds to them
        self.latent = f32_to_bf16_rne(rng.normal(size=(V, 576)).astype(np.float32))
        self.q_abs, self.q_rope = rng.normal(size=(V, H, 512)).astype(np.float32), rng.normal(size=(V, H, 64)).astype(np.float32)
        self.key = rng.normal(size=(V, HD)).astype(np.float32)
        self.bias = (3 * rng.normal(size=(V, V))).astype(np.float32)
        put = lambda x, kind: torch.from_numpy(np.ascontiguousarray(x)).cuda().view(kind)  # noqa: E731
        self.d = dict(latent=put(self.latent.view(np.int16), torch.bfloat16), q_abs=put(self.q_abs, torch.float32), q_rope=put(self.q_rope, torch.float32),
                      key=put(self.key, torch.float32), bias=put(self.bias, torch.float32), weight=dev(self.weight), q_weight=dev(self.q_weight),
                      k_weight=dev(self.k_weight), k_bias=dev(self.k_bias), table=dev(self.table), tables=dev(self.tables),
                      cu=dev(np.arange(B + 1, dtype=np.int32)), groups=dev(np.array([0, B], np.int32)), prefixes=dev(np.array([PROMPT], np.int32)),
                      t=dev(np.where(np.arange(B) % 7 == 3, 0, 0.8).astype(np.float32)), k=dev((np.arange(B) % 5 * 20).astype(np.int32)),
                      p=dev(np.where(np.arange(B) % 3 == 0, 1, 0.9).astype(np.float32)), m=dev(np.where(np.arange(B) % 4 == 1, 0.05, 0).astype(np.float32)))
        self.pool, self.kpool = dzeros(N_PAGES * PT * 580, 0x30), dzeros(N_PAGES * PT * HD * 2)
        # a prompt's rows, by the same calls, through the first sequence's table (the last page of its own: each sequence's copy)
        prompt = rng.integers(0, V, PROMPT)
        for s in range(B):
            some = np.arange(PROMPT) if s == 0 else np.arange(SHARED * PT, PROMPT)
            self.rows(torch.from_numpy(prompt[some]).cuda(), some, self.tables[s, some // PT] * PT + some % PT)
        self.token = torch.from_numpy(rng.integers(0, V, B).astype(np.int32)).cuda()
        self.position = torch.full((B,), PROMPT, dtype=torch.int32, device="cuda")
        self.u = dev(np.zeros(B, np.float32)).view(torch.float32)
        self.qa, self.qr = (torch.empty(B, H, w, dtype=torch.bfloat16, device="cuda") for w in (512, 64))
        self.out, self.lse = torch.empty(B, H, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(B, H, device="cuda")
        self.partial = torch.empty(hip.mla_attend_tree_shared_paged_scratch_floats(B, 1, H, B, 1, PROMPT, PROMPT + STEPS), device="cuda")
        self.work = dzeros(hip.sample_rows_workspace_bytes(B, V))
        self.logits, self.probs = (torch.empty(B, V, device="cuda") for _ in range(2))
        self.next, self.kept = (torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(2))
        self.pages = torch.from_numpy(self.tables).cuda()

    def rows(self, tokens, positions, slots, stream=None):
        """Latent rows and index keys of tokens into their pages."""
        d, n = self.d, len(tokens)
        positions, slots = (x if hasattr(x, "data_ptr") else dev(np.asarray(x, np.int32)) for x in (positions, slots))
        latent, key = d["latent"][tokens.long()], d["key"][tokens.long()]
        hip.launch_kv_norm_append_paged(latent, slots, d["weight"], d["table"], positions, self.pool, n, 576, 512, 64, 2048, PT, N_PAGES, EPS, False, True,
                                        None, stream)
        hip.launch_norm_rope_rows(key, self.kpool, d["k_weight"], d["k_bias"], d["table"], positions, slots, n, 1, HD, HD, 0, 64, 2048, N_PAGES * PT, HD, HD,
                                  HD, HD, 0, EPS, True, True, False, True, None, stream)
        self.held = (latent, key)

    def step(self):
        torch, d = self.torch, self.d
        stream = torch.cuda.current_stream()
        at = self.position.long()
        slots = (self.pages.gather(1, (at // PT)[:, None])[:, 0] * PT + (at % PT).int()).int()
        self.rows(self.token, self.position, slots, stream)
        q_abs, q_rope = d["q_abs"][self.token.long()], d["q_rope"][self.token.long()]
        hip.launch_norm_rope_rows(q_abs, self.qa, None, None, None, None, None, B, H, 512, 512, 0, 0, 0, 0, H * 512, 512, H * 512, 512, 0, EPS, False, False,
                                  False, True, None, stream)
        hip.launch_norm_rope_rows(q_rope, self.qr, d["q_weight"], None, d["table"], self.position, None, B, H, 64, 64, 0, 64, 2048, 0, H * 64, 64, H * 64, 64, 0,
                                  EPS, False, False, False, True, None, stream)
        hip.launch_mla_attend_tree_shared_paged(self.qa, self.qr, self.pool, d["tables"], self.position, d["cu"], None, d["groups"], d["prefixes"], B, 1, H, B, 1,
                                                PROMPT, PROMPT + STEPS, BLOCKS, 512, 64, PT, N_PAGES, 576 ** -0.5, self.out, self.lse, self.partial, None, stream)
        torch.add(d["bias"][self.token.long()], self.out.reshape(B, -1)[:, :V].float(), alpha=4.0, out=self.logits)
        hip.launch_sample_rows(self.logits, d["t"], d["k"], d["p"], d["m"], self.u, B, V, V, False, self.next, self.kept, None, self.probs, V, self.work, stream)
        self.token.copy_(self.next)
        self.position += 1


def check(e, token, position, u):
    """A step's results against the definitions, each from what the call before it left."""
    # the cached rows: what they stand for, within a code's half step of what the formula says
    want, _ = normed(bf16_to_f32(e.latent[token])[:, None], e.weight, None, e.table, np.full(B, position, np.int32), 512, 512, 64, False, False)
    pool = back(e.pool).reshape(N_PAGES, -1)
    for s in range(B):
        page, off = pool[e.tables[s, position // PT]], position % PT
        scale = page[PT * 576 + 4 * off:PT * 576 + 4 * off + 4].view(np.float32)[0]
        q = want[s, 0] / scale
        assert (np.abs(e4m3_values()[page[off * 576:(off + 1) * 576]] - q) <= 2.0 ** -4 * np.maximum(np.abs(q), 2.0 ** -6) * (1 + 2.0 ** -12)).all()
    key, far = normed(e.key[token][:, None], e.k_weight, e.k_bias, e.table, np.full(B, position, np.int32), HD, 0, 64, True, True)
    kpool = bf16_to_f32(back(e.kpool, np.uint16)).reshape(-1, HD)
    at = e.tables[:, position // PT] * PT + position % PT
    assert (np.abs(kpool[at] - key[:, 0]) <= 2.0 ** -8 * np.abs(key[:, 0]) + 2 * far[:, 0]).all()
    # attention
    bits = lambda t: back(t.view(e.torch.int16), np.uint16)  # noqa: E731
    qa, qr = bits(e.qa).reshape(B, H, 512), bits(e.qr).reshape(B, H, 64)
    scale = float(np.float32(576 ** -0.5))
    out, lse, far, lse_far = tree_attention(qa, qr, pool, e.tables, np.full(B, position), np.arange(B + 1), None, PT, scale)
    got = bf16_to_f32(bits(e.out)).reshape(B, H, 512)
    assert (np.abs(got - out) <= far).all() and (np.abs(back(e.lse, np.float32).reshape(B, H) - lse) <= lse_far).all()
    # the draw
    logits, drawn, kept = back(e.logits, np.float32).reshape(B, V), back(e.next, np.int32), back(e.kept, np.int32)
    t, k, p, m = (back(e.d[n], kind) for n, kind in (("t", np.float32), ("k", np.int32), ("p", np.float32), ("m", np.float32)))
    probs = back(e.probs, np.float32).reshape(B, V)
    for s in range(B):
        token, count, share = sample_row(logits[s], t[s], k[s], float(p[s]), float(m[s]), float(u[s]))
        assert (drawn[s], kept[s]) == (token, count)
        assert np.abs(probs[s] - share).max() <= 2.0 ** -23


def test_steps_of_a_batch_behind_one_prompt():
    rng = np.random.default_rng(1)
    draws = rng.random((STEPS, B)).astype(np.float32)
    eager = Engine(5)
    tokens = []
    for i in range(STEPS):
        token = back(eager.token, np.int32).copy()
        eager.u.copy_(dev(draws[i]).view(eager.torch.float32))
        eager.step()
        eager.torch.cuda.synchronize()
        check(eager, token, PROMPT + i, draws[i])
        tokens.append(back(eager.next, np.int32).copy())
    assert len(np.unique(tokens[-1])) > B // 2           # one prompt, many answers
    # the same from a graph of one step: same tokens, same cache
    torch = torch_cuda()
    replayed = Engine(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    token, position, pool, kpool = replayed.token.clone(), replayed.position.clone(), replayed.pool.clone(), replayed.kpool.clone()
    with torch.cuda.stream(side):
        replayed.step()
    torch.cuda.synchronize()
    for to, was in ((replayed.token, token), (replayed.position, position), (replayed.pool, pool), (replayed.kpool, kpool)):
        to.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed.step()
    for i in range(STEPS):
        replayed.u.copy_(dev(draws[i]).view(torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(back(replayed.next, np.int32), tokens[i]), i
    assert (back(replayed.pool) == back(eager.pool)).all() and (back(replayed.kpool) == back(eager.kpool)).all()
