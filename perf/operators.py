"""A step of drafted tokens over the paged latent cache, operator by operator, as cases that can be timed and compared.

A program that decodes several drafted tokens a step rotates their queries and keys to their
positions (`rope`), appends their rows, attends from every node of the drafted tree over the cached
prefix and the node's own ancestors (`tree`), decides against the target's probabilities which
drafts stand (`verify`) and moves the rows of those that do to where the next step expects them
(`commit`). `listed()` names the cases that are quoted; `draw()` makes more of the same ranges.

With `own` the framework's launchers run, without it the same operators in elementary torch
operations. What a serving program owns for the life of a layer (pools, block tables, trees, rotation
tables) is made by `prepare`; scratch and output buffers are made on a state's first pass.
"""
import math
import random

import torch

own = False

KVL, ROPE = 512, 64
W = KVL + ROPE                       # a cached row: 512 latent and 64 roped codes, then one f32 scale
LAYERS = 48                          # of the benchmark's decode configuration
YARN = dict(factor=16.0, orig=4096, fast=32.0, slow=1.0)


def listed():
    return [
        # one user, a chain of three drafts behind the last token, a short context: latency is all there is
        dict(name="tree_b1_chain4_ctx200", op="tree", seqs=1, nodes=4, heads=16, ctx=200, page=64, chain=True, ragged=False),
        # a ragged batch of odd sizes, pages that end inside a tile, some sequences without a prefix or without a node
        dict(name="tree_b13_ragged_odd", op="tree", seqs=13, nodes=9, heads=20, ctx=5003, page=48, chain=False, ragged=True),
        # the benchmark's full decode batch, a small tree a sequence
        dict(name="tree_b32_nodes8_32k", op="tree", seqs=32, nodes=8, heads=64, ctx=32768, page=64, chain=False, ragged=False),
        # one long conversation and a wide tree, all heads of a large layer
        dict(name="tree_b1_nodes64_128k", op="tree", seqs=1, nodes=64, heads=128, ctx=131072, page=64, chain=False, ragged=False),
        # one user's chain, drafted with probabilities
        dict(name="verify_b1_chain4", op="verify", seqs=1, nodes=4, vocab=32001, draft=True, chain=True, bf16=False),
        # a decode batch of trees whose drafts were picked, not drawn: the target's probabilities alone, as bf16
        dict(name="verify_b32_tree16", op="verify", seqs=32, nodes=16, vocab=131072, draft=False, chain=False, bf16=True),
        # a large batch of drawn trees with both distributions in f32: siblings are judged against residuals
        dict(name="verify_b256_tree8", op="verify", seqs=256, nodes=8, vocab=131072, draft=True, chain=False, bf16=False),
        # the kept rows of one sequence in one layer
        dict(name="commit_b1_one_layer", op="commit", seqs=1, nodes=8, kept=4, layers=1, ctx=1000, page=64),
        # a batch's kept rows in every layer at once
        dict(name="commit_b64_48_layers", op="commit", seqs=64, nodes=16, kept=6, layers=LAYERS, ctx=700, page=64),
        # the roped part of a drafted step's query heads, adjacent pairs
        dict(name="rope_32x8_interleaved", op="rope", tokens=256, heads=64, rd=64, head_row=64, half=False, bf16=True, positions=131072),
        # a prompt's heads of 192 values whose last 64 are rotated, halves paired
        dict(name="rope_8192_half", op="rope", tokens=8192, heads=128, rd=64, head_row=192, half=True, bf16=True, positions=163840),
        # the rotation table of a long context, stretched by parts
        dict(name="rope_table_160k", op="rope_table", positions=163840, rd=64, base=10000.0, scaling="parts"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm (odd ones as likely as even)."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "verify", "verify", "commit", "rope", "rope_table"])
    if op == "tree":
        heads = rng.choice([8, 16, 20, 32, 64, 128])
        nodes = _log(rng, 1, 64)
        seqs = _log(rng, 1, 48)
        # no more scores than the largest listed case has, and a quarter of its rows times batch
        top = min(131072, (1 << 29) // (seqs * nodes * heads))
        return dict(op=op, seqs=seqs, nodes=nodes, heads=heads, ctx=_log(rng, 1, max(2, top)), page=rng.choice([16, 48, 64, 64, 128]),
                    chain=rng.random() < 0.3, ragged=rng.random() < 0.5)
    if op == "verify":
        return dict(op=op, seqs=_log(rng, 1, 128), nodes=_log(rng, 1, 16), vocab=_log(rng, 1000, 131072), draft=rng.random() < 0.5,
                    chain=rng.random() < 0.4, bf16=rng.random() < 0.4)
    if op == "commit":
        nodes = _log(rng, 1, 32)
        return dict(op=op, seqs=_log(rng, 1, 64), nodes=nodes, kept=rng.randint(1, nodes), layers=_log(rng, 1, LAYERS), ctx=_log(rng, 1, 700),
                    page=rng.choice([16, 48, 64]))
    if op == "rope":
        rd = rng.choice([32, 64, 64, 128])
        return dict(op=op, tokens=_log(rng, 1, 8192), heads=_log(rng, 1, 64), rd=rd, head_row=rd + rng.choice([0, 64, 128]), half=rng.random() < 0.5,
                    bf16=rng.random() < 0.7, positions=_log(rng, 2048, 163840))
    return dict(op=op, positions=_log(rng, 1024, 163840), rd=rng.choice([32, 64, 128]), base=rng.choice([10000.0, 500000.0]),
                scaling=rng.choice(["none", "linear", "parts"]))


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """Cached rows and drafted nodes of every sequence: the case's own, whatever the seed."""
    seqs, nodes, ctx = case["seqs"], case["nodes"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * seqs, [nodes] * seqs
    rng = random.Random(seqs * 1000003 + nodes * 1009 + ctx)
    lens, held = [rng.randint(0, ctx) for _ in range(seqs)], [rng.randint(0, nodes) for _ in range(seqs)]
    lens[0], held[0] = ctx, nodes                    # the longest there is
    if seqs > 2:
        lens[1], held[1] = 0, nodes                  # nothing cached yet
        held[2] = 0                                  # a sequence that drafts nothing
    return lens, held


def _ints(g, lo, hi, shape):
    """Whole numbers lo..hi, both ends included."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _parents(g, seqs, nodes, chain):
    """[seqs][nodes] parents, the root's -1: a chain, or trees whose nodes hang on any of the four nodes before them."""
    at = torch.arange(nodes, device="cuda", dtype=torch.int32).expand(seqs, nodes)
    back = torch.ones_like(at) if chain else _ints(g, 1, 4, (seqs, nodes))
    return torch.where(at == 0, -1, (at - back).clamp(min=0)).to(torch.int32).contiguous()


def _ancestors(parents):
    """[seqs][nodes][nodes] bool: j is i or above it."""
    seqs, nodes = parents.shape
    seen = torch.zeros(seqs, nodes, nodes, dtype=torch.bool, device="cuda")
    for i in range(nodes):  # a node sees itself and what its parent sees
        if i:
            seen[:, i] = seen[torch.arange(seqs, device="cuda"), parents[:, i].long()]
        seen[:, i, i] = True
    return seen


def _pack(seen):
    """[rows][nodes] bool -> [rows][ceil(nodes / 32)] int32 words, bit j & 31 of word j >> 5 first."""
    rows, nodes = seen.shape
    words = -(-nodes // 32)
    bits = torch.zeros(rows, words * 32, dtype=torch.int64, device="cuda")
    bits[:, :nodes] = seen
    word = (bits.reshape(rows, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).contiguous()


def _tables(g, seqs, blocks):
    """Every sequence's pages, shuffled over one pool."""
    return torch.randperm(seqs * blocks, generator=g, device="cuda").to(torch.int32).reshape(seqs, blocks).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op == "tree":
        seqs, nodes, heads, page = case["seqs"], case["nodes"], case["heads"], case["page"]
        blocks = -(-(case["ctx"] + nodes) // page)
        n_pages = seqs * blocks
        s["table"] = _tables(g, seqs, blocks)
        lens, held = _lengths(case)
        s["ctx_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        n = s["n"] = sum(held)
        held = torch.tensor(held, device="cuda")
        s["cu"] = torch.cat([held.new_zeros(1), held.cumsum(0)]).to(torch.int32)
        if case["chain"]:
            s["masks"] = None
        else:
            seen = _ancestors(_parents(g, seqs, nodes, False))
            if case["ragged"] and seqs > 2:
                seen[1, 0] = False                   # with no prefix either: a node that attends nothing
            live = torch.arange(nodes, device="cuda")[None] < held[:, None]
            s["masks"] = _pack(seen[live])
        s["qabs"] = (torch.randn(n, heads, KVL, generator=g, device="cuda") * 2).to(torch.bfloat16)
        s["qrope"] = (torch.randn(n, heads, ROPE, generator=g, device="cuda") * 2).to(torch.bfloat16)
        s["pool"] = torch.empty(n_pages, page * (W + 4), dtype=torch.uint8, device="cuda")
        for at in range(0, n_pages, 1024):           # rows as the append leaves them: largest code 448 under one scale
            some = min(1024, n_pages - at)
            x = torch.randn(some, page, W, generator=g, device="cuda")
            x *= torch.exp(0.3 * torch.randn(some, page, 1, generator=g, device="cuda"))
            scale = x.abs().amax(-1, keepdim=True) / 448
            s["pool"][at:at + some, :page * W] = (x / scale).to(torch.float8_e4m3fn).view(torch.uint8).reshape(some, -1)
            s["pool"][at:at + some, page * W:] = scale.reshape(some, page).contiguous().view(torch.uint8)
        s["scale"], s["blocks"], s["n_pages"] = 1 / math.sqrt(192), blocks, n_pages
    elif op == "verify":
        seqs, nodes, vocab = case["seqs"], case["nodes"], case["vocab"]
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        s["parents"] = _parents(g, seqs, nodes, case["chain"])
        n = seqs * nodes
        target = torch.empty(n, vocab, dtype=kind, device="cuda")
        draft = torch.empty(n, vocab, dtype=kind, device="cuda") if case["draft"] else None
        tokens = torch.empty(n, dtype=torch.int32, device="cuda")
        for at in range(0, n, nodes * 16):           # peaked rows, and a draft model that nearly agrees
            end = min(n, at + nodes * 16)
            logits = 2.5 * torch.randn(end - at, vocab, generator=g, device="cuda")
            target[at:end] = torch.softmax(logits, -1).to(kind)
            logits += 0.6 * torch.randn(end - at, vocab, generator=g, device="cuda")
            if draft is not None:
                draft[at:end] = torch.softmax(logits, -1).to(kind)
            up = (torch.arange(at, end, device="cuda") // nodes) * nodes + s["parents"].reshape(-1)[at:end].clamp(min=0) - at
            if draft is not None:                    # each drawn from its parent's draft row
                drawn = torch.multinomial(draft[at:end].float(), nodes, replacement=True, generator=g)
                tokens[at:end] = drawn[up, torch.arange(at, end, device="cuda") % nodes].to(torch.int32)
            else:                                    # each among the likeliest after its parent
                best = torch.topk(logits, nodes, dim=-1).indices
                tokens[at:end] = best[up, torch.arange(at, end, device="cuda") % nodes].to(torch.int32)
        s["target"], s["draft"], s["tokens"] = target, draft, tokens
        s["cu"] = torch.arange(0, n + 1, nodes, dtype=torch.int32, device="cuda")
        s["u"] = torch.rand(n, generator=g, device="cuda")
        s["u_final"] = torch.rand(seqs, generator=g, device="cuda")
        s["n"] = n
    elif op == "commit":
        seqs, nodes, page, layers = case["seqs"], case["nodes"], case["page"], case["layers"]
        blocks = -(-(case["ctx"] + nodes) // page)
        s["table"] = _tables(g, seqs, blocks)
        s["ctx_lens"] = _ints(g, 0, case["ctx"], (seqs,))
        s["pool"] = torch.randint(0, 256, (layers, seqs * blocks, page * (W + 4)), generator=g, device="cuda", dtype=torch.uint8)
        order = torch.rand(seqs, nodes, generator=g, device="cuda")
        order[:, 0] = -1                             # the root is always kept
        kept = order.argsort(-1)[:, :case["kept"]].sort(-1).values.to(torch.int32)
        s["path"] = torch.full((seqs, nodes), -1, dtype=torch.int32, device="cuda")
        s["path"][:, :case["kept"]] = kept
        s["n_path"] = torch.full((seqs,), case["kept"], dtype=torch.int32, device="cuda")
        s["blocks"], s["n_pages"] = blocks, seqs * blocks
    elif op == "rope":
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        s["x"] = torch.randn(case["tokens"], case["heads"], case["head_row"], generator=g, device="cuda").to(kind)
        s["positions"] = _ints(g, 0, case["positions"] - 1, (case["tokens"],))
        at = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None]
        angle = at * 10000.0 ** (-torch.arange(0, case["rd"], 2, device="cuda", dtype=torch.float64) / case["rd"])
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().reshape(case["positions"], case["rd"]).contiguous()
    else:
        s["first"] = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
    return s


# ---- the plain forms ------------------------------------------------------------------------------------


def _plain_tree(s):
    seqs, nodes, heads, page = s["seqs"], s["nodes"], s["heads"], s["page"]
    ctx, cu = s["ctx_lens"].long(), s["cu"].long()
    span = s["blocks"] * page
    pages = s["pool"][s["table"].reshape(-1).long()]
    codes = pages[:, :page * W].contiguous().view(torch.float8_e4m3fn).float().reshape(seqs, span, W)
    scale = pages[:, page * W:].contiguous().view(torch.float32).reshape(seqs, span, 1)
    rows = codes * scale
    # every sequence's nodes in a rectangle, absent ones as zeros
    at = cu[:-1, None] + torch.arange(nodes, device="cuda")
    live = at < cu[1:, None]
    q = torch.cat([s["qabs"], s["qrope"]], -1).float()
    if s["n"] == 0:
        q = torch.zeros(1, heads, W, device="cuda")
    q = torch.where(live[..., None, None], q[torch.where(live, at, 0)], 0)
    x = torch.matmul(q.reshape(seqs, nodes * heads, W), rows.transpose(1, 2).contiguous()) * s["scale"]
    t = torch.arange(span, device="cuda")
    j = t[None] - ctx[:, None]                       # which node a cached position is, past the prefix
    if s["masks"] is None:
        seen = j[:, None] <= torch.arange(nodes, device="cuda")[None, :, None]
    else:
        words = s["masks"].long()[torch.where(live, at, 0)]
        word = words.gather(2, (j.clamp(0, nodes - 1) >> 5)[:, None].expand(-1, nodes, -1))
        seen = (((word >> (j.clamp(0, nodes - 1) & 31)[:, None]) & 1) == 1) & (j < nodes)[:, None]
    seen = torch.where((j < 0)[:, None], True, seen) & (j[:, None] < (cu[1:] - cu[:-1])[:, None, None])
    x = x.reshape(seqs, nodes, heads, span).masked_fill(~seen[:, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top.isinf(), 0, top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.reshape(seqs, nodes * heads, span), rows[..., :KVL]).reshape(seqs, nodes, heads, KVL)
    out = torch.where(total > 0, out / total, 0)
    lse = (top + total.log())[..., 0]
    return out[live].to(torch.bfloat16), lse[live]


def _weights(rows):
    """Probabilities as they count: in 64 bits, what is no number or negative as zero."""
    return rows.double().nan_to_num(nan=0.0).clamp(min=0)


def _plain_verify(s):
    seqs, nodes, vocab = s["seqs"], s["nodes"], s["vocab"]
    b = torch.arange(seqs, device="cuda")
    tokens, parents = s["tokens"].reshape(seqs, nodes).long(), s["parents"].long()
    u = s["u"].reshape(seqs, nodes).double()
    target = s["target"].reshape(seqs, nodes, vocab)
    draft = None if s["draft"] is None else s["draft"].reshape(seqs, nodes, vocab)
    cur = torch.zeros(seqs, dtype=torch.long, device="cuda")
    w = _weights(target[:, 0])
    c = torch.ones(seqs, dtype=torch.float64, device="cuda")
    path = torch.full((seqs, nodes), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    count = torch.ones(seqs, dtype=torch.long, device="cuda")
    for i in range(1, nodes):  # children come after their parent, so one walk in index order is the walk of the tree
        child = parents[:, i] == cur
        x = tokens[:, i]
        wx = w[b, x]
        if draft is None:
            ok = u[:, i] * c < wx
            left = w.clone()
            left[b, x] = 0
            c_left = c - wx
        else:
            q = _weights(draft[b, cur])
            ok = u[:, i] * q[b, x] * c < wx
            left = (w - c[:, None] * q).clamp(min=0)
            c_left = left.sum(-1)
        ok, lost = child & ok, child & ~ok
        path[b, torch.where(ok, count, 0)] = torch.where(ok, i, 0).to(torch.int32)
        count += ok
        cur = torch.where(ok, i, cur)
        w = torch.where(ok[:, None], _weights(target[:, i]), torch.where(lost[:, None], left, w))
        c = torch.where(ok, 1.0, torch.where(lost, c_left, c))
    w = torch.where((w.sum(-1) > 0)[:, None], w, _weights(target[b, cur]))
    upto = w.cumsum(-1)
    past = upto > (s["u_final"].double() * upto[:, -1])[:, None]
    token = past.to(torch.uint8).argmax(-1)          # the first past the drawn share
    return path, count.to(torch.int32), token.to(torch.int32)


def _plain_commit(s):
    nodes, page = s["nodes"], s["page"]
    pool = s["pool"]
    codes = pool[..., :page * W].unflatten(-1, (page, W))
    scales = pool[..., page * W:].unflatten(-1, (page, 4))
    k = torch.arange(nodes, device="cuda")
    live = k < s["n_path"][:, None]
    to = s["ctx_lens"].long()[:, None] + k
    at = s["ctx_lens"].long()[:, None] + torch.where(live, s["path"].long(), k)
    src, dst = s["table"].long().gather(1, at // page), s["table"].long().gather(1, to // page)
    rows, row_scales = codes[:, src, at % page], scales[:, src, at % page]
    # a row past the kept ones goes where it is, from what was read before anything moved: those go first
    codes[:, dst[live], (to % page)[live]] = rows[:, live]
    scales[:, dst[live], (to % page)[live]] = row_scales[:, live]
    return pool, s["ctx_lens"] + s["n_path"]


def _plain_rope(s):
    rd, half = s["rd"], s["half"]
    x = s["x"][..., s["head_row"] - rd:].float()
    pair = s["table"][s["positions"].long()].reshape(-1, 1, rd // 2, 2)
    c, n = pair[..., 0], pair[..., 1]
    a, b = (x[..., :rd // 2], x[..., rd // 2:]) if half else (x[..., ::2], x[..., 1::2])
    u, v = a * c - b * n, a * n + b * c
    out = torch.cat([u, v], -1) if half else torch.stack([u, v], -1).flatten(-2)
    return out.to(s["x"].dtype)


def _frequencies(rd, base, scaling):
    """[rd / 2] angles of one position, in 64 bits."""
    j = torch.arange(rd // 2, device="cuda", dtype=torch.float64)
    f = base ** (-2 * j / rd)
    if scaling == "none":
        return f
    if scaling == "linear":
        return f / YARN["factor"]
    # by parts: pairs that turn often within the original context keep their frequency, those that turn less
    # than once are stretched, a ramp between
    def where(turns):
        return rd * math.log(YARN["orig"] / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(where(YARN["fast"])), 0), min(math.ceil(where(YARN["slow"])), rd - 1)
    ramp = ((j - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / YARN["factor"] * ramp + f * (1 - ramp)


def _plain_table(s):
    at = torch.arange(s["first"], s["first"] + s["positions"], device="cuda", dtype=torch.float64)[:, None]
    angle = at * _frequencies(s["rd"], s["base"], s["scaling"])
    return (torch.stack([angle.cos(), angle.sin()], -1) * _mscale(s["scaling"])).float().reshape(s["positions"], s["rd"])


def _mscale(scaling):
    """What the rotated values are stretched by with the context: a number that f32 holds."""
    return 1.25 if scaling == "parts" else 1.0


# ---- the framework's calls ------------------------------------------------------------------------------


def _own_tree(s, hip):
    seqs, nodes, heads, ctx = s["seqs"], s["nodes"], s["heads"], s["ctx"]
    if "out" not in s:
        s["out"] = torch.empty(s["n"], heads, KVL, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.empty(s["n"], heads, dtype=torch.float32, device="cuda")
        floats = hip.mla_attend_tree_paged_scratch_floats(seqs, heads, s["n"], nodes, ctx)
        s["partial"] = torch.empty(max(floats, 4), dtype=torch.float32, device="cuda")
    if s["n"]:
        hip.launch_mla_attend_tree_paged(s["qabs"], s["qrope"], s["pool"], s["table"], s["ctx_lens"], s["cu"], s["masks"], seqs, heads,
                                         s["n"], nodes, ctx, s["blocks"], KVL, ROPE, s["page"], s["n_pages"], s["scale"], s["out"],
                                         s["lse"], s["partial"], None, torch.cuda.current_stream())
    return s["out"], s["lse"]


def _own_verify(s, hip):
    seqs, nodes, vocab = s["seqs"], s["nodes"], s["vocab"]
    if "path" not in s:
        s["path"] = torch.empty(seqs, nodes, dtype=torch.int32, device="cuda")
        s["n_path"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
        s["next"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
        s["work"] = torch.empty(max(hip.draft_verify_workspace_bytes(seqs, nodes, vocab), 16), dtype=torch.uint8, device="cuda")
    hip.launch_draft_verify(s["target"], s["draft"], s["tokens"], s["parents"], s["cu"], s["u"], s["u_final"], seqs, s["n"], nodes, vocab,
                            vocab, vocab, s["bf16"], s["path"], s["n_path"], s["next"], s["work"], None, torch.cuda.current_stream())
    return s["path"], s["n_path"], s["next"]


def _own_commit(s, hip):
    if "lens" not in s:
        s["lens"] = torch.empty_like(s["ctx_lens"])
    hip.launch_kv_commit_paged(s["pool"], s["table"], s["ctx_lens"], s["path"], s["n_path"], s["seqs"], s["nodes"], s["blocks"], W, s["page"],
                               s["n_pages"], s["layers"], s["pool"].stride(0), s["lens"], None, torch.cuda.current_stream())
    return s["pool"], s["lens"]


def _own_rope(s, hip):
    tokens, heads, rd, row = s["tokens"], s["heads"], s["rd"], s["head_row"]
    if "out" not in s:
        s["out"] = torch.empty(tokens, heads, rd, dtype=s["x"].dtype, device="cuda")
    hip.launch_rope_rows(s["x"][..., row - rd:], s["out"], s["table"], s["positions"], tokens, heads, rd, s["table"].shape[0],
                         heads * row, row, heads * rd, rd, s["half"], s["bf16"], None, torch.cuda.current_stream())
    return s["out"]


def _own_table(s, hip):
    if "out" not in s:
        s["out"] = torch.empty(s["positions"], s["rd"], device="cuda")
    factor = 1.0 if s["scaling"] == "none" else YARN["factor"]
    orig = YARN["orig"] if s["scaling"] == "parts" else 0
    hip.launch_rope_table(s["out"], s["first"], s["positions"], s["rd"], s["base"], factor, orig, YARN["fast"], YARN["slow"], _mscale(s["scaling"]),
                          torch.cuda.current_stream())
    return s["out"]


def run(state):
    op = state["op"]
    if own:
        from rivoli_amd import hip

        return dict(tree=_own_tree, verify=_own_verify, commit=_own_commit, rope=_own_rope, rope_table=_own_table)[op](state, hip)
    return dict(tree=_plain_tree, verify=_plain_verify, commit=_plain_commit, rope=_plain_rope, rope_table=_plain_table)[op](state)


def work(case):
    op = case["op"]
    if op == "tree":
        lens, held = _lengths(case)
        rows = sum(held) * case["heads"]
        tokens = sum(n + h for n, h in zip(lens, held) if h)
        products = sum(h * case["heads"] * (n + h) for n, h in zip(lens, held))
        return {"bytes": tokens * (W + 4) + rows * (2 * W + 2 * KVL + 4), "flops": 2.0 * products * (W + KVL)}
    if op == "verify":
        size = (2 if case["bf16"] else 4) * (2 if case["draft"] else 1)
        return {"bytes": case["seqs"] * (case["vocab"] * size + case["nodes"] * 16 + 8), "flops": 4.0 * case["seqs"] * case["vocab"]}
    if op == "commit":
        return {"bytes": 2.0 * case["seqs"] * max(case["kept"] - 1, 1) * case["layers"] * (W + 4) + 12 * case["seqs"], "flops": 0}
    if op == "rope":
        size = 2 if case["bf16"] else 4
        return {"bytes": case["tokens"] * case["rd"] * (2.0 * case["heads"] * size + 4), "flops": 3.0 * case["tokens"] * case["heads"] * case["rd"]}
    return {"bytes": 4.0 * case["positions"] * case["rd"], "flops": 0}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------


def exact(case, seed):
    op = case["op"]
    if op in ("verify", "commit"):
        return None                                  # whole numbers and moved bytes
    s = prepare(case, seed)
    if op == "rope":
        angle_c, angle_s = s["table"].double()[s["positions"].long()].reshape(case["tokens"], case["rd"] // 2, 2).unbind(-1)
        z = s["x"][:, :, case["head_row"] - case["rd"]:].double()
        out = torch.empty_like(z)
        for j in range(case["rd"] // 2):
            a, b = (j, j + case["rd"] // 2) if case["half"] else (2 * j, 2 * j + 1)
            out[:, :, a] = z[:, :, a] * angle_c[:, None, j] - z[:, :, b] * angle_s[:, None, j]
            out[:, :, b] = z[:, :, b] * angle_c[:, None, j] + z[:, :, a] * angle_s[:, None, j]
        return out
    if op == "rope_table":
        out = torch.empty(case["positions"], case["rd"], dtype=torch.float64, device="cuda")
        at = torch.arange(case["positions"], device="cuda", dtype=torch.float64) + s["first"]
        rd, base = case["rd"], case["base"]
        for j in range(rd // 2):
            f = math.exp(-2 * j / rd * math.log(base))
            stretched = 0.0 if case["scaling"] == "none" else 1.0
            if case["scaling"] == "parts":           # the pair whose wave fits `turns` times into the original context
                edge = [rd / 2 * math.log(YARN["orig"] / 2 / math.pi / turns) / math.log(base) for turns in (YARN["fast"], YARN["slow"])]
                first, last = max(0, math.floor(edge[0])), min(rd - 1, math.ceil(edge[1]))
                stretched = min(1.0, max(0.0, (j - first) / (last - first if last != first else 0.001)))
            f *= 1 - stretched + stretched / YARN["factor"]
            out[:, 2 * j], out[:, 2 * j + 1] = torch.cos(at * f) * _mscale(case["scaling"]), torch.sin(at * f) * _mscale(case["scaling"])
        return out
    page, heads = case["page"], case["heads"]
    out = torch.empty(s["n"], heads, KVL, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["n"], heads, dtype=torch.float64, device="cuda")
    cu, ctx = s["cu"].tolist(), s["ctx_lens"].tolist()
    for b in range(case["seqs"]):
        held = cu[b + 1] - cu[b]
        if not held:
            continue
        length = ctx[b] + held
        pages = s["pool"][s["table"][b].long()]
        value = pages[:, :page * W].contiguous().view(torch.float8_e4m3fn).double().reshape(-1, W)[:length]
        value = value * pages[:, page * W:].contiguous().view(torch.float32).double().reshape(-1, 1)[:length]
        step = max(1, (1 << 28) // (heads * length))
        for i in range(cu[b], cu[b + 1], step):
            end = min(i + step, cu[b + 1])
            q = torch.cat([s["qabs"][i:end], s["qrope"][i:end]], 2).double().reshape(-1, W)
            score = ((q @ value.T) * s["scale"]).reshape(end - i, heads, length)
            for n in range(i, end):
                if s["masks"] is None:
                    score[n - i, :, ctx[b] + n - cu[b] + 1:] = -math.inf
                else:
                    words = s["masks"][n].tolist()
                    hidden = [ctx[b] + j for j in range(held) if not words[j // 32] >> (j % 32) & 1]
                    score[n - i][:, hidden] = -math.inf
            lse[i:end] = torch.logsumexp(score, -1)
            weight = torch.exp(score - lse[i:end, :, None].nan_to_num(neginf=0.0))
            out[i:end] = (weight.reshape(-1, length) @ value[:, :KVL]).reshape(end - i, heads, KVL)
    return out, lse
