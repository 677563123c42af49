"""A decode step of a batch that continues shared prompts, operator by operator, as cases that can be timed and compared.

Around the cached attention a serving program norms a token's queries and keys and rotates them
to its position (`heads`; `keys` where they go to the paged index keys), does the same to its latent row and
quantizes it into the pages (`append`), attends over pages of which the first are the same for a whole group of
sequences (`shared`), and turns the logits into tokens (`sample`). `listed()` names the cases that are quoted;
`draw()` makes more of the same ranges.

With `own` the framework's launchers run, without it the same operators in elementary torch
operations. What a serving program owns for the life of a layer (pools, block tables, weights, rotation
tables) is made by `prepare`; scratch and output buffers are made on a state's first pass.
"""
import math
import random

import torch

own = False

KVL, ROPE = 512, 64
W = KVL + ROPE                       # a cached row: 512 latent and 64 roped codes, then one f32 scale
EPS = 1e-6


def listed():
    return [
        # one token's query heads: latency is all there is
        dict(name="heads_b1", op="heads", tokens=1, heads=16, width=128, norm=128, rope_at=64, rd=64, half=False, center=False, bf16=True),
        # a prompt's query heads, normed as a whole, the last half of them rotated
        dict(name="heads_8192_bf16", op="heads", tokens=8192, heads=64, width=128, norm=128, rope_at=64, rd=64, half=True, center=False, bf16=True),
        # a long prompt's index keys: mean and bias too, f32 from the projection, their first values rotated, into the paged bf16 keys
        dict(name="keys_8192", op="keys", tokens=8192, width=128, norm=128, rope_at=0, rd=64, half=True, center=True, bf16=False, page=64),
        # a decode step's latent rows in one layer
        dict(name="append_b32", op="append", tokens=32, page=64, half=False, bf16=True),
        # a prompt's
        dict(name="append_8192", op="append", tokens=8192, page=64, half=False, bf16=True),
        # four answers to one short prompt
        dict(name="shared_b4_h16_500", op="shared", seqs=4, groups=1, nodes=1, heads=16, prefix=448, rest=60, page=64, ragged=False),
        # three groups of unlike sizes and sequences of none, drafted chains of up to three, pages that end inside a tile
        dict(name="shared_b37_odd", op="shared", seqs=37, groups=3, nodes=3, heads=20, prefix=5003, rest=701, page=48, ragged=True),
        # a batch behind one long prompt, the heads of one part of eight of a layer
        dict(name="shared_b64_h16_32k", op="shared", seqs=64, groups=1, nodes=1, heads=16, prefix=32768, rest=1024, page=64, ragged=True),
        # the largest: a big batch, four long documents asked about
        dict(name="shared_b128_h32_64k", op="shared", seqs=128, groups=4, nodes=1, heads=32, prefix=65536, rest=1024, page=64, ragged=True),
        # one user's token
        dict(name="sample_b1_32k", op="sample", rows=1, vocab=32001, kinds="p", bf16=False, probs=False),
        # a decode batch, every filter set, logits as the projection leaves them
        dict(name="sample_b64_128k", op="sample", rows=64, vocab=131072, kinds="kpm", bf16=True, probs=False),
        # a large batch that asks for unlike things, some for no filter, and for the distributions that a draft is verified against
        dict(name="sample_b256_128k_probs", op="sample", rows=256, vocab=131072, kinds="mixed", bf16=False, probs=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm (odd ones as likely as even)."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["heads", "keys", "append", "shared", "shared", "shared", "sample", "sample", "sample"])
    if op in ("heads", "keys"):
        rd = rng.choice([32, 64, 64])
        width = rd * rng.choice([1, 2, 2, 3, 4])
        case = dict(op=op, tokens=_log(rng, 1, 8192), width=width, norm=rng.choice([width, width, max(32, width - rd)]),
                    rope_at=rng.choice([0, width - rd]), rd=rd, half=rng.random() < 0.5, center=rng.random() < 0.4, bf16=rng.random() < 0.6)
        return dict(case, heads=_log(rng, 1, 64)) if op == "heads" else dict(case, page=rng.choice([16, 48, 64]))
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 8192), page=rng.choice([16, 48, 64, 64]), half=rng.random() < 0.5, bf16=rng.random() < 0.7)
    if op == "shared":
        heads = rng.choice([8, 16, 16, 20, 32, 64, 128])
        nodes = rng.choice([1, 1, 1, 2, 3, 5])
        seqs = _log(rng, 2, 128)
        # no more scores than the largest listed case has
        top = min(65536, (1 << 28) // (seqs * nodes * heads))
        return dict(op=op, seqs=seqs, groups=_log(rng, 1, min(8, max(1, seqs // 2))), nodes=nodes, heads=heads, prefix=_log(rng, 16, max(32, top)),
                    rest=_log(rng, 1, 1024), page=rng.choice([16, 48, 64, 64, 128]), ragged=rng.random() < 0.6)
    return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 131072), kinds=rng.choice(["none", "k", "p", "m", "kp", "kpm", "mixed"]),
                bf16=rng.random() < 0.5, probs=rng.random() < 0.3)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """The case's own, whatever the seed: borders of the groups, their prefixes, cached rows and nodes of every sequence."""
    seqs, groups, nodes, prefix, rest = case["seqs"], case["groups"], case["nodes"], case["prefix"], case["rest"]
    if not case["ragged"]:
        cu = [seqs * i // groups for i in range(groups + 1)]
        return cu, [prefix] * groups, [prefix + rest] * seqs, [nodes] * seqs
    rng = random.Random(seqs * 1000003 + prefix * 1009 + rest)
    grouped = seqs - (seqs // 8 if groups > 1 else 0)                # the last ones share nothing
    inner = sorted(rng.sample(range(1, grouped), groups - 1)) if groups > 1 else []
    cu = [0] + inner + [grouped]
    prefixes = [prefix] + [rng.randint(prefix // 2, prefix) for _ in range(groups - 1)]
    lens, held = [], []
    for s in range(seqs):
        of = [p for p, lo, hi in zip(prefixes, cu, cu[1:]) if lo <= s < hi]
        lens.append(sum(of) + rng.randint(0, rest))
        held.append(rng.randint(1, nodes))
    if grouped < seqs:
        lens[-1] = 0                                                 # one that begins
    return cu, prefixes, lens, held


def _shared_pages(case):
    """Whole pages of every sequence that its group shares."""
    cu, prefixes, lens, held = _lengths(case)
    first = [0] * case["seqs"]
    for g, p in enumerate(prefixes):
        for s in range(cu[g], cu[g + 1]):
            first[s] = p // case["page"]
    return cu, prefixes, lens, held, first


def _angles(positions, rd):
    at = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None]
    angle = at * 10000.0 ** (-torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)
    return torch.stack([angle.cos(), angle.sin()], -1).float().reshape(positions, rd).contiguous()


def _slots(g, tokens, page, n_pages):
    """Where a prompt's tokens go: its pages lie anywhere in the pool, its rows in order in them."""
    pages = torch.randperm(n_pages, generator=g, device="cuda")
    at = torch.arange(tokens, device="cuda")
    return (pages[at // page] * page + at % page).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op in ("heads", "keys", "append"):
        tokens = case["tokens"]
        heads = case.get("heads", 1)
        width, norm, rd = (W, KVL, ROPE) if op == "append" else (case["width"], case["norm"], case["rd"])
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        x = torch.randn(tokens, heads, width, generator=g, device="cuda")
        x *= torch.exp(torch.randn(tokens, heads, 1, generator=g, device="cuda"))         # tokens are of unlike size
        s["x"] = (x + 0.1).to(kind)
        s["weight"] = 1 + 0.2 * torch.randn(norm, generator=g, device="cuda")
        s["bias"] = 0.1 * torch.randn(norm, generator=g, device="cuda") if case.get("center") else None
        s["table"] = _angles(16384, rd)
        s["positions"] = (torch.randint(0, 16384 - tokens, (1,), generator=g, device="cuda") + torch.arange(tokens, device="cuda")).to(torch.int32)
        if op != "heads":
            s["n_pages"] = -(-tokens // case["page"]) + 3
            s["slots"] = _slots(g, tokens, case["page"], s["n_pages"])
        if op == "keys":
            s["kpool"] = torch.randn(s["n_pages"] * case["page"], width, generator=g, device="cuda").to(torch.bfloat16)
        if op == "append":
            s["pool"] = torch.randint(0, 120, (s["n_pages"], case["page"] * (W + 4)), generator=g, device="cuda", dtype=torch.uint8)
            s["pool"][:, case["page"] * W:].view(torch.float32).fill_(0.01)
    elif op == "shared":
        seqs, heads, page = case["seqs"], case["heads"], case["page"]
        cu, prefixes, lens, held, first = _shared_pages(case)
        blocks = -(-max(n + h for n, h in zip(lens, held)) // page)
        n_pages = sum(p // page for p in prefixes) + sum(-(-(n + h) // page) - f for n, h, f in zip(lens, held, first))
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        table, at = [], 0
        for s_ in range(seqs):
            if s_ in cu[:-1]:                                        # a group's first sequence brings its pages
                common = order[at:at + first[s_]]
                at += first[s_]
            more = -(-(lens[s_] + held[s_]) // page) - first[s_]
            pages = (common if first[s_] else []) + order[at:at + more]
            at += more
            table.append(pages + [0] * (blocks - len(pages)))
        s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
        s["ctx_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["cu"] = torch.tensor([sum(held[:i]) for i in range(seqs + 1)], dtype=torch.int32, device="cuda")
        s["cu_groups"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        s["prefix_lens"] = torch.tensor(prefixes, dtype=torch.int32, device="cuda")
        n = s["n"] = sum(held)
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
        s["scale"], s["blocks"], s["n_pages"], s["max_ctx"] = 1 / math.sqrt(192), blocks, n_pages, max(lens)
    else:
        rows, vocab, kinds = case["rows"], case["vocab"], case["kinds"]
        kind = torch.bfloat16 if case["bf16"] else torch.float32
        # a model's logits: a broad body, and a few dozen tokens far above it, fewer the higher
        logits = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
        likely = torch.randint(0, vocab, (rows, 64), generator=g, device="cuda")
        lift = 4 + 3 * torch.empty(rows, 64, device="cuda").exponential_(generator=g).clamp(max=6)
        s["logits"] = logits.scatter(1, likely, logits.gather(1, likely).abs() + lift).to(kind)

        def some(which, values, off):
            """A filter's values of the rows: of all of them, of every other pair in a batch that asks for unlike things, or off."""
            on = torch.full((rows,), which in kinds, device="cuda")
            if kinds == "mixed":
                on = (torch.arange(rows, device="cuda") >> "kpm".index(which)) % 2 == 1
            return torch.where(on, values, torch.full_like(values, off))

        def between(lo, hi):
            return lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")

        s["t"] = between(0.6, 1.2)
        if rows > 4:
            s["t"][::9] = 0.0                                        # the likeliest token
        s["k"] = some("k", torch.randint(1, 201, (rows,), generator=g, device="cuda"), 0).to(torch.int32)
        s["p"] = some("p", between(0.8, 0.99), 1.0)
        s["m"] = some("m", between(0.01, 0.1), 0.0)
        s["u"] = torch.rand(rows, generator=g, device="cuda")
    return s


# ---- the plain forms ------------------------------------------------------------------------------------


def _normed(s, norm, rope_at, rd):
    """Rows normed over their first `norm` values and rotated, in 32 bits."""
    x = s["x"].float()
    y = x[..., :norm]
    if s["bias"] is not None:
        y = y - y.mean(-1, keepdim=True)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["weight"]
    if s["bias"] is not None:
        y = y + s["bias"]
    y = torch.cat([y, x[..., norm:]], -1)
    pair = s["table"][s["positions"].long()].reshape(-1, 1, rd // 2, 2)
    c, n = pair[..., 0], pair[..., 1]
    z = y[..., rope_at:rope_at + rd]
    a, b = (z[..., :rd // 2], z[..., rd // 2:]) if s["half"] else (z[..., ::2], z[..., 1::2])
    u, v = a * c - b * n, a * n + b * c
    z = torch.cat([u, v], -1) if s["half"] else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([y[..., :rope_at], z, y[..., rope_at + rd:]], -1)


def _plain_heads(s):
    return _normed(s, s["norm"], s["rope_at"], s["rd"]).to(s["x"].dtype)


def _plain_keys(s):
    s["kpool"][s["slots"].long()] = _normed(s, s["norm"], s["rope_at"], s["rd"])[:, 0].to(torch.bfloat16)
    return s["kpool"]


def _pool_values(pool, page):
    """What pages hold: the codes' values, and the scales."""
    return pool[:, :page * W].view(torch.float8_e4m3fn), pool[:, page * W:].view(torch.float32)


def _plain_append(s):
    page = s["page"]
    rows = _normed(s, KVL, KVL, ROPE)[:, 0]
    top = rows.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / 448, 1.0)
    slots = s["slots"].long()
    s["pool"][:, :page * W].unflatten(1, (page, W))[slots // page, slots % page] = (rows / scale).to(torch.float8_e4m3fn).view(torch.uint8)
    s["pool"][:, page * W:].unflatten(1, (page, 4))[slots // page, slots % page] = scale.view(torch.uint8)
    return _pool_values(s["pool"], page)


def _plain_shared(s):
    seqs, nodes, heads, page = s["seqs"], s["nodes"], s["heads"], s["page"]
    ctx, cu = s["ctx_lens"].long(), s["cu"].long()
    span = s["blocks"] * page
    pages = s["pool"][s["table"].reshape(-1).long()]
    rows = pages[:, :page * W].contiguous().view(torch.float8_e4m3fn).float().reshape(seqs, span, W)
    rows *= pages[:, page * W:].contiguous().view(torch.float32).reshape(seqs, span, 1)
    # every sequence's nodes in a rectangle, absent ones as zeros
    at = cu[:-1, None] + torch.arange(nodes, device="cuda")
    live = at < cu[1:, None]
    q = torch.cat([s["qabs"], s["qrope"]], -1).float()
    q = torch.where(live[..., None, None], q[torch.where(live, at, 0)], 0)
    x = torch.matmul(q.reshape(seqs, nodes * heads, W), rows.transpose(1, 2).contiguous()) * s["scale"]
    # a node sees the cached rows and its sequence's nodes up to itself
    seen = torch.arange(span, device="cuda") <= (ctx[:, None] + torch.arange(nodes, device="cuda"))[..., None]
    x = x.reshape(seqs, nodes, heads, span).masked_fill(~seen[:, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.reshape(seqs, nodes * heads, span), rows[..., :KVL]).reshape(seqs, nodes, heads, KVL) / total
    lse = (top + total.log())[..., 0]
    return out[live].to(torch.bfloat16), lse[live]


def _plain_sample(s):
    # in 64 bits: which tokens stay and which is drawn are decided by sums next to a border
    x = s["logits"].double()
    t = s["t"].double()[:, None]
    greedy = t <= 0
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    z = order.values - order.values[:, :1]
    rank = torch.arange(s["vocab"], device="cuda")
    w = torch.where(greedy, (rank == 0).double(), torch.exp(z / torch.where(greedy, 1.0, t)))
    k = s["k"][:, None].long()
    kept = (rank < k) | (k <= 0)
    w_k = torch.where(kept, w, 0)
    before = w_k.cumsum(-1) - w_k
    p = s["p"].double()[:, None]
    kept &= (before < p * w_k.sum(-1, keepdim=True)) | (p >= 1)
    kept &= w >= s["m"].double()[:, None]
    kept &= ~greedy | (rank == 0)
    w = torch.where(kept, w, 0)
    by_token = torch.zeros_like(w).scatter_(1, order.indices, w)
    upto = by_token.cumsum(-1)
    past = upto > s["u"].double()[:, None] * upto[:, -1:]
    token = past.to(torch.uint8).argmax(-1)
    p_token = by_token.gather(1, token[:, None])[:, 0] / upto[:, -1]
    out = [token.to(torch.int32), kept.sum(-1).to(torch.int32), p_token.log().float()]
    if s["probs"]:
        out.append((by_token / upto[:, -1:]).float())
    return tuple(out)


# ---- the framework's calls ------------------------------------------------------------------------------


def _own_heads(s, hip):
    tokens, heads, width = s["tokens"], s["heads"], s["width"]
    if "out" not in s:
        s["out"] = torch.empty_like(s["x"])
    hip.launch_norm_rope_rows(s["x"], s["out"], s["weight"], s["bias"], s["table"], s["positions"], None, tokens, heads, width, s["norm"],
                              s["rope_at"], s["rd"], s["table"].shape[0], 0, heads * width, width, heads * width, width, 0, EPS, s["center"],
                              s["half"], s["bf16"], s["bf16"], None, torch.cuda.current_stream())
    return s["out"]


def _own_keys(s, hip):
    width = s["width"]
    hip.launch_norm_rope_rows(s["x"], s["kpool"], s["weight"], s["bias"], s["table"], s["positions"], s["slots"], s["tokens"], 1, width,
                              s["norm"], s["rope_at"], s["rd"], s["table"].shape[0], s["kpool"].shape[0], width, width, width, width, 0, EPS,
                              s["center"], s["half"], s["bf16"], True, None, torch.cuda.current_stream())
    return s["kpool"]


def _own_append(s, hip):
    hip.launch_kv_norm_append_paged(s["x"], s["slots"], s["weight"], s["table"], s["positions"], s["pool"], s["tokens"], W, KVL, ROPE,
                                    s["table"].shape[0], s["page"], s["n_pages"], EPS, s["half"], s["bf16"], None, torch.cuda.current_stream())
    return _pool_values(s["pool"], s["page"])


def _own_shared(s, hip):
    seqs, groups, nodes, heads, prefix, ctx = s["seqs"], s["groups"], s["nodes"], s["heads"], s["prefix"], s["max_ctx"]
    if "out" not in s:
        s["out"] = torch.empty(s["n"], heads, KVL, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.empty(s["n"], heads, dtype=torch.float32, device="cuda")
        floats = hip.mla_attend_tree_shared_paged_scratch_floats(seqs, groups, heads, s["n"], nodes, prefix, ctx)
        s["partial"] = torch.empty(max(floats, 4), dtype=torch.float32, device="cuda")
    hip.launch_mla_attend_tree_shared_paged(s["qabs"], s["qrope"], s["pool"], s["table"], s["ctx_lens"], s["cu"], None, s["cu_groups"],
                                            s["prefix_lens"], seqs, groups, heads, s["n"], nodes, prefix, ctx, s["blocks"], KVL, ROPE,
                                            s["page"], s["n_pages"], s["scale"], s["out"], s["lse"], s["partial"], None,
                                            torch.cuda.current_stream())
    return s["out"], s["lse"]


def _own_sample(s, hip):
    rows, vocab = s["rows"], s["vocab"]
    if "tokens" not in s:
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["kept"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(rows, dtype=torch.float32, device="cuda")
        s["out"] = torch.empty(rows, vocab, dtype=torch.float32, device="cuda") if s["probs"] else None
        s["work"] = torch.empty(max(hip.sample_rows_workspace_bytes(rows, vocab), 16), dtype=torch.uint8, device="cuda")
    hip.launch_sample_rows(s["logits"], s["t"], s["k"], s["p"], s["m"], s["u"], rows, vocab, vocab, s["bf16"], s["tokens"], s["kept"],
                           s["logprobs"], s["out"], vocab, s["work"], torch.cuda.current_stream())
    return (s["tokens"], s["kept"], s["logprobs"]) + ((s["out"],) if s["probs"] else ())


def run(state):
    op = state["op"]
    if own:
        from rivoli_amd import hip

        return dict(heads=_own_heads, keys=_own_keys, append=_own_append, shared=_own_shared, sample=_own_sample)[op](state, hip)
    return dict(heads=_plain_heads, keys=_plain_keys, append=_plain_append, shared=_plain_shared, sample=_plain_sample)[op](state)


def work(case):
    op = case["op"]
    size = 2 if case.get("bf16") else 4
    if op in ("heads", "keys"):
        values = case["tokens"] * case.get("heads", 1) * case["width"]
        return {"bytes": values * (size + (2 if op == "keys" else size)) + case["tokens"] * 4.0 * case["rd"], "flops": 8.0 * values}
    if op == "append":
        return {"bytes": case["tokens"] * (W * size + W + 4 + 4.0 * ROPE + 8), "flops": 12.0 * case["tokens"] * W}
    if op == "shared":
        cu, prefixes, lens, held, first = _shared_pages(case)
        rows = sum(held) * case["heads"]
        tokens = sum(p // case["page"] * case["page"] for p in prefixes) + sum(n + h - f * case["page"] for n, h, f in zip(lens, held, first))
        scores = case["heads"] * sum(h * n + h * (h + 1) // 2 for n, h in zip(lens, held))
        return {"bytes": tokens * (W + 4) + rows * (2 * W + 2 * KVL + 4), "flops": 2.0 * scores * (W + KVL)}
    values = case["rows"] * case["vocab"]
    return {"bytes": values * (size + (4.0 if case["probs"] else 0)) + 32 * case["rows"], "flops": 8.0 * values}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------


def _exact_rows(s, norm, rope_at, rd):
    x = s["x"].double().clone()
    y = x[:, :, :norm]
    off = y.mean(2, keepdim=True) if s["bias"] is not None else 0.0
    size = torch.sqrt(((y - off) ** 2).sum(2, keepdim=True) / norm + EPS)
    x[:, :, :norm] = (y - off) / size * s["weight"].double() + (0.0 if s["bias"] is None else s["bias"].double())
    angle_c, angle_s = s["table"].double()[s["positions"].long()].reshape(-1, rd // 2, 2).unbind(-1)
    z = x[:, :, rope_at:rope_at + rd].clone()
    for j in range(rd // 2):
        a, b = (j, j + rd // 2) if s["half"] else (2 * j, 2 * j + 1)
        x[:, :, rope_at + a] = z[:, :, a] * angle_c[:, None, j] - z[:, :, b] * angle_s[:, None, j]
        x[:, :, rope_at + b] = z[:, :, b] * angle_c[:, None, j] + z[:, :, a] * angle_s[:, None, j]
    return x


def _exact_codes(x):
    """The nearest values of the 8-bit codes, to the even one of two."""
    code = torch.arange(127, device="cuda", dtype=torch.float64)
    value = torch.where(code < 8, code / 512, (8 + code % 8) * 2.0 ** ((code / 8).floor() - 10))
    mid = (value[1:] + value[:-1]) / 2
    low, high = torch.searchsorted(mid, x.abs().contiguous()), torch.searchsorted(mid, x.abs().contiguous(), right=True)
    at = torch.where(low % 2 == 0, low, high)                        # (they differ where x is a middle)
    return torch.copysign(value[at.clamp(max=126)], x)


def _exact_sample(s):
    logprob, probs = [], []
    for r in range(s["rows"]):
        x = s["logits"][r].double()
        t, k, p, m = (float(s[n][r]) for n in "tkpm")
        if t <= 0:
            keep = torch.zeros_like(x, dtype=torch.bool)
            keep[int((x == x.max()).nonzero()[0])] = True
            w = keep.double()
        else:
            w = torch.exp((x - x.max()) / t)
            # by value, from the largest down: the last value that is kept, and how many of those that have it
            value, count = torch.unique(x, return_counts=True)
            value, count = value.flip(0), count.flip(0)
            each = torch.exp((value - value[0]) / t)
            if k > 0:
                left = (k - (count.cumsum(0) - count)).clamp(min=0)
                count = torch.minimum(count, left.long())
            mass = each * count
            if p < 1:
                left = ((p * mass.sum() - (mass.cumsum(0) - mass)) / each).ceil().clamp(min=0)
                count = torch.minimum(count.double(), left).long()
            count = torch.where(each >= m, count, 0)
            last = int(count.nonzero()[-1])
            keep = x > value[last]
            keep[(x == value[last]).nonzero()[:int(count[last]), 0]] = True
        w = torch.where(keep, w, 0) / w[keep].sum()
        at = w.cumsum(0) > float(s["u"][r])
        at = int(at.nonzero()[0]) if bool(at.any()) else int(keep.nonzero()[-1])
        logprob.append(torch.log(w[at]))
        probs.append(w)
    return (None, None, torch.stack(logprob)) + ((torch.stack(probs),) if s["probs"] else ())


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "heads":
        return _exact_rows(s, case["norm"], case["rope_at"], case["rd"])
    if op == "keys":
        out = s["kpool"].double()
        out[s["slots"].long()] = _exact_rows(s, case["norm"], case["rope_at"], case["rd"])[:, 0]
        return out
    if op == "append":
        page = case["page"]
        rows = _exact_rows(s, KVL, KVL, ROPE)[:, 0]
        scale = rows.abs().amax(1) / 448
        codes, scales = (v.double() for v in _pool_values(s["pool"], page))
        slots = s["slots"].long()
        codes.unflatten(1, (page, W))[slots // page, slots % page] = _exact_codes(rows / scale[:, None])
        scales[slots // page, slots % page] = scale
        return codes, scales
    if op == "sample":
        return _exact_sample(s)
    page, heads = case["page"], case["heads"]
    out = torch.empty(s["n"], heads, KVL, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["n"], heads, dtype=torch.float64, device="cuda")
    cu, ctx = s["cu"].tolist(), s["ctx_lens"].tolist()
    for b in range(case["seqs"]):
        length = ctx[b] + cu[b + 1] - cu[b]
        pages = s["pool"][s["table"][b, :-(-length // page)].long()]
        value = pages[:, :page * W].contiguous().view(torch.float8_e4m3fn).double().reshape(-1, W)[:length]
        value = value * pages[:, page * W:].contiguous().view(torch.float32).double().reshape(-1, 1)[:length]
        for n in range(cu[b], cu[b + 1]):
            some = value[:ctx[b] + n - cu[b] + 1]
            score = (torch.cat([s["qabs"][n], s["qrope"][n]], 1).double() @ some.T) * s["scale"]
            lse[n] = torch.logsumexp(score, 1)
            out[n] = torch.exp(score - lse[n][:, None]) @ some[:, :KVL]
    return out, lse
