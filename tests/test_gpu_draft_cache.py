"""Rotation (rivoli_rope_table, rivoli_rope_rows) against 64 bits, the commit of kept rows against a loop, and a whole
step of drafted tokens against the same tokens decoded one after the other."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import BF16, F32, ancestors, bf16_rows, pack_masks, random_pool, rope_table, rotate
from tests.gpu_util import back, dev, dzeros, torch_cuda
from tests.util import bf16_to_f32, f32_to_bf16_rne, shuffled_block_tables, slots_for

pytestmark = pytest.mark.gpu


# ---- rotation --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("first,n,rd,base,mscale,scaling", [
    (0, 1, 2, 1e4, 1.0, {}), (0, 1000, 64, 1e4, 1.0, {}), (5, 33, 64, 5e5, 1.0, dict(factor=8.0)), (1000000, 77, 128, 8e6, 1.0, {}),
    (2 ** 31 - 101, 100, 64, 1e4, 1.0, {}), (0, 5000, 64, 1e4, 1.25, dict(factor=40.0, orig=4096)), (160000, 17, 32, 1e4, 0.5, dict(factor=16.0, orig=4096, fast=16.0, slow=2.0)),
    (3, 50, 64, 1e4, 1.0, dict(factor=4.0, orig=2 ** 30)), (3, 50, 16, 1e4, 1.0, dict(factor=4.0, orig=1)), (0, 300, 1024, 1e4, 1.0, {}),
])
def test_table(first, n, rd, base, mscale, scaling):
    out = dzeros((n + 1) * rd * 4, 0xEE)
    names = dict(factor="factor", orig="orig_ctx", fast="beta_fast", slow="beta_slow")
    hip.launch_rope_table(out, first, n, rd, base, mscale=mscale, **{names[k]: v for k, v in scaling.items()})
    got = back(out, np.float32)
    assert (got[n * rd:].view(np.uint32) == 0xEEEEEEEE).all()
    want = rope_table(first, n, rd, base, mscale, **scaling)
    # the angle: a frequency and a product of 53 bits each, some ten half steps of up to 2^31 radians; a fraction of a turn in f32, 2 pi
    # half steps of it at most; sine and cosine of two steps each (the library's bound for them is below that), one product
    far = (10 * 2.0 ** -53 * (first + n) + (np.pi + 4 + 2) * 2 * F32) * abs(mscale)
    assert np.abs(got[:n * rd].reshape(n, rd // 2, 2) - want).max() <= far


def check_rope(tokens, heads, rd, half, bf16, x_strides, out_strides, off=0, out_off=0, in_place=False, seed=0, n_positions=500):
    rng = np.random.default_rng(seed)
    size, kind = (2, np.uint16) if bf16 else (4, np.float32)
    room = off + (tokens - 1) * x_strides[0] + (heads - 1) * x_strides[1] + rd
    values = rng.standard_normal(room).astype(np.float32)
    x = f32_to_bf16_rne(values) if bf16 else values
    pairs = rope_table(0, n_positions, rd, 1e4)
    table = pairs.astype(np.float32).reshape(n_positions, rd)
    positions = rng.integers(0, n_positions, tokens).astype(np.int32)
    bad = dzeros(4)
    if tokens > 3:
        positions[1], positions[3] = -1, n_positions
    x_d = dev(x)
    out_room = out_off + (tokens - 1) * out_strides[0] + (heads - 1) * out_strides[1] + rd
    out_d = x_d if in_place else dzeros(out_room * size, 0xEE)
    before = back(out_d, kind).copy()
    hip.launch_rope_rows(x_d.data_ptr() + off * size, out_d.data_ptr() + out_off * size, dev(table), dev(positions), tokens, heads, rd, n_positions,
                         *x_strides, *out_strides, half, bf16, bad)
    got = back(out_d, kind)
    expect = before.copy()
    v = bf16_to_f32(x) if bf16 else x
    rows = np.stack([[v[off + t * x_strides[0] + h * x_strides[1]:][:rd] for h in range(heads)] for t in range(tokens)])
    want = rotate(rows, table[np.clip(positions, 0, n_positions - 1)].reshape(tokens, rd // 2, 2).astype(np.float64), half)
    live = (positions >= 0) & (positions < n_positions)
    reach = np.abs(rows).max()                            # |x c| + |y s| <= 2 reach: two products and a sum of f32
    for t in range(tokens):
        for h in range(heads):
            at = out_off + t * out_strides[0] + h * out_strides[1]
            if not live[t]:
                continue
            y = got[at:at + rd]
            y = bf16_to_f32(y) if bf16 else y
            assert (np.abs(y - want[t, h]) <= 6 * F32 * reach + (BF16 if bf16 else F32) * np.abs(want[t, h])).all(), (t, h)
            expect[at:at + rd] = got[at:at + rd]
    assert np.array_equal(expect.view(np.uint8), got.view(np.uint8)), "something else was written"
    assert int(back(bad, np.uint32)[0]) == int((~live).sum())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("tokens,heads,rd", [(1, 1, 2), (1, 1, 64), (5, 3, 64), (7, 4, 32), (3, 9, 128), (4, 17, 6), (300, 1, 64), (2, 128, 64), (5, 5, 62)])
def test_rows(tokens, heads, rd, half, bf16):
    check_rope(tokens, heads, rd, half, bf16, (heads * rd, rd), (heads * rd, rd), seed=heads)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_parts_of_heads_strides_and_places(half, bf16):
    check_rope(6, 5, 64, half, bf16, (5 * 192, 192), (5 * 64, 64), off=128)            # the last 64 of 192, packed
    check_rope(6, 5, 64, half, bf16, (5 * 192, 192), (5 * 192, 192), off=128, out_off=128, in_place=True)
    check_rope(6, 5, 64, half, bf16, (5 * 71 + 3, 71), (5 * 67 + 1, 67), off=1, out_off=3)  # off any boundary
    check_rope(6, 5, 64, half, bf16, (64, 6 * 64), (5 * 64, 64))                       # heads outermost
    check_rope(6, 5, 64, half, bf16, (5 * 65, 65), (5 * 65, 65), in_place=True)
    check_rope(6, 2, 64, half, bf16, (0, 64), (128, 64))                               # one row for every token


# ---- the commit ------------------------------------------------------------------------------------------

def commit_by_hand(pool, tables, ctx, path, n_path, page, row_bytes, scaled):
    """pool [n_pages][bytes], moved as if at once; how many entries are bad."""
    out, bad = pool.copy(), 0
    for s in range(len(ctx)):
        for k in range(min(max(n_path[s], 0), path.shape[1])):
            if path[s, k] == k:
                continue
            at, to = ctx[s] + path[s, k], ctx[s] + k
            ok = path[s, k] > k and at // page < tables.shape[1]
            ok = ok and 0 <= tables[s, at // page] < len(pool) and 0 <= tables[s, to // page] < len(pool)
            if not ok:
                bad += 1
                continue
            a, b = pool[tables[s, at // page]], out[tables[s, to // page]]
            i, j = at % page, to % page
            b[j * row_bytes:(j + 1) * row_bytes] = a[i * row_bytes:(i + 1) * row_bytes]
            if scaled:
                b[page * row_bytes + 4 * j:][:4] = a[page * row_bytes + 4 * i:][:4]
    return out, bad


@pytest.mark.parametrize("keys", [False, True])
@pytest.mark.parametrize("seqs,nodes,page,layers,width", [(1, 1, 64, 1, 576), (3, 8, 64, 2, 576), (5, 40, 16, 3, 576), (4, 70, 48, 1, 1024), (2, 33, 4, 2, 16), (70, 5, 64, 1, 576)])
def test_commit(seqs, nodes, page, layers, width, keys):
    rng = np.random.default_rng(seqs * 7 + nodes)
    if keys:
        width //= 2                                        # values of two bytes
    row_bytes = 2 * width if keys else width
    ctx = rng.integers(0, 150, seqs).astype(np.int32)
    ctx[0] = 0
    blocks = -(-(150 + nodes) // page)
    n_pages = seqs * blocks + 2
    tables = shuffled_block_tables(seqs, blocks, n_pages, 3)
    bytes_ = page * (row_bytes + (0 if keys else 4))
    gap = 48                                               # between two layers' pools
    pool = rng.integers(0, 256, (layers, n_pages * bytes_ + (gap if not keys else 2 * width * 3)), dtype=np.uint8)
    path = np.full((seqs, nodes), -1, np.int32)
    n_path = rng.integers(1, nodes + 1, seqs).astype(np.int32)
    for s in range(seqs):
        path[s, 1:n_path[s]] = np.sort(rng.permutation(np.arange(1, nodes))[:n_path[s] - 1])
        path[s, 0] = 0
    if seqs > 2:
        n_path[1], n_path[2] = 0, nodes + 9                # nothing kept; more than the table of paths has
        path[2] = np.arange(nodes)
        path[2, nodes // 2] = nodes - 1                    # the same row twice
        if nodes > 4:
            path[2, 3], path[2, 4] = 1, 10 ** 8            # from before its place, and past the table
    want, bad = pool.copy(), 0
    for l in range(layers):
        moved, bad = commit_by_hand(pool[l, :n_pages * bytes_].reshape(n_pages, bytes_), tables, ctx, path, n_path, page, row_bytes, not keys)
        want[l, :n_pages * bytes_] = moved.reshape(-1)
    pool_d, lens, counted = dev(pool), dzeros(seqs * 4, 0xEE), dzeros(4)
    launch = hip.launch_index_commit_paged if keys else hip.launch_kv_commit_paged
    launch(pool_d, dev(tables), dev(ctx), dev(path), dev(n_path), seqs, nodes, blocks, width, page, n_pages, layers,
           pool.shape[1] // row_bytes if keys else pool.shape[1], lens, counted)
    assert np.array_equal(back(pool_d), want.reshape(-1))
    assert np.array_equal(back(lens, np.int32), ctx + np.clip(n_path, 0, nodes))
    assert int(back(counted, np.uint32)[0]) == bad


def test_commit_leaves_out_rows_without_a_page():
    rng = np.random.default_rng(4)
    pool = random_pool(rng, 4, 64, 576)
    tables = np.array([[1, -1], [2, 3]], np.int32)
    ctx, n_path = np.array([60, 62], np.int32), np.array([3, 3], np.int32)
    path = np.array([[0, 2, 5], [0, 3, 4]], np.int32)
    want, bad = commit_by_hand(pool, tables, ctx, path, n_path, 64, 576, True)
    pool_d, counted = dev(pool), dzeros(4)
    hip.launch_kv_commit_paged(pool_d, dev(tables), dev(ctx), dev(path), dev(n_path), 2, 3, 2, 576, 64, 4, bad_rows=counted)
    assert np.array_equal(back(pool_d), want.reshape(-1)) and int(back(counted, np.uint32)[0]) == bad == 1


# ---- all of a step ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("graph", [False, True])
def test_a_step_of_drafts_leaves_what_decoding_one_by_one_leaves(graph):
    """Two steps of trees: rotate, append, attend, verify, commit. The cache is then byte for byte the one that the emitted tokens
    alone would have made, and the last root's attention bit for bit that of decoding it as a chain of one."""
    torch = torch_cuda()
    rng = np.random.default_rng(11)
    B, T, H, PT, W, V, HD = 3, 7, 16, 64, 576, 50, 128
    ctx0 = np.array([0, 61, 190], np.int32)
    blocks, n_pages = 5, 20
    tables = shuffled_block_tables(B, blocks, n_pages, 5)
    tables_d = dev(tables)
    table = dzeros(400 * 64 * 4)
    hip.launch_rope_table(table, 0, 400, 64, 1e4)
    # a token's key is its embedding, rotated to its position; a fixed target and draft row for every token
    embed = bf16_rows(rng, (V, W))
    embed_keys = rng.standard_normal((V, HD), dtype=np.float32)
    target = np.exp(rng.normal(0, 1.5, (V, V)))
    target = (target / target.sum(1, keepdims=True)).astype(np.float32)
    draft = np.exp(np.log(target) + rng.normal(0, 0.7, (V, V)))
    draft = (draft / draft.sum(1, keepdims=True)).astype(np.float32)
    queries = bf16_rows(rng, (V, H, W))
    # the prompt
    pool, kpool = dev(random_pool(rng, n_pages, PT, W)), dev(rng.integers(0, 60000, (n_pages * PT, HD)).astype(np.uint16))
    plain_pool, plain_kpool = pool.clone(), kpool.clone()
    history = [[] for _ in range(B)]                       # emitted tokens with their rows in the cache
    ctx, root = ctx0.copy(), rng.integers(0, V, B)
    n = B * T
    cu = np.arange(0, n + 1, T, dtype=np.int32)
    floats = hip.mla_attend_tree_paged_scratch_floats(B, H, n, T, 300)
    ws = hip.draft_verify_workspace_bytes(B, T, V)
    d = {k: dzeros(s) for k, s in dict(rows=n * W * 2, qa=n * H * 512 * 2, qr=n * H * 64 * 2, positions=n * 4, slots=n * 4, keys=n * HD * 4, masks=n * 4,
                                       tokens=n * 4, parents=n * 4, u=n * 4, uf=B * 4, target=n * V * 4, draft=n * V * 4, ctx=B * 4, out=n * H * 512 * 2,
                                       lse=n * H * 4, path=n * 4, n_path=B * 4, next=B * 4, lens=B * 4, partial=max(floats, 4) * 4, ws=max(ws, 16)).items()}
    cu_d = dev(cu)

    def step(stream):
        rope_at = d["rows"].data_ptr() + 512 * 2
        hip.launch_rope_rows(rope_at, rope_at, table, d["positions"], n, 1, 64, 400, W, W, W, W, False, True, None, stream)
        hip.launch_rope_rows(d["qr"], d["qr"], table, d["positions"], n, H, 64, 400, H * 64, 64, H * 64, 64, False, True, None, stream)
        hip.launch_kv_append_paged(d["rows"], d["slots"], pool, n, W, PT, n_pages, None, stream)
        hip.launch_index_append_paged(d["keys"], d["slots"], kpool, n, HD, PT, n_pages, None, stream)
        hip.launch_mla_attend_tree_paged(d["qa"], d["qr"], pool, tables_d, d["ctx"], cu_d, d["masks"], B, H, n, T, 300, blocks, 512, 64, PT, n_pages,
                                         192 ** -0.5, d["out"], d["lse"], d["partial"], None, stream)
        hip.launch_draft_verify(d["target"], d["draft"], d["tokens"], d["parents"], cu_d, d["u"], d["uf"], B, n, T, V, V, V, False, d["path"], d["n_path"],
                                d["next"], d["ws"], None, stream)
        hip.launch_kv_commit_paged(pool, tables_d, d["ctx"], d["path"], d["n_path"], B, T, blocks, W, PT, n_pages, 1, 0, d["lens"], None, stream)
        hip.launch_index_commit_paged(kpool, tables_d, d["ctx"], d["path"], d["n_path"], B, T, blocks, HD, PT, n_pages, 1, 0, None, None, stream)

    captured = None
    moved = 0
    for turn in range(3):
        parents = np.array([-1, 0, 0, 1, 1, 2, 3], np.int32)
        depth = np.array([0, 1, 1, 2, 2, 2, 3])
        tokens = np.zeros((B, T), np.int32)
        for s in range(B):
            tokens[s, 0] = root[s]
            for i in range(1, T):
                p = draft[tokens[s, parents[i]]].astype(np.float64)
                tokens[s, i] = rng.choice(V, p=p / p.sum())
        flat = tokens.reshape(-1)
        put = dict(rows=embed[flat], qa=queries[flat][:, :, :512], qr=queries[flat][:, :, 512:], keys=embed_keys[flat], tokens=flat,
                   positions=(ctx[:, None] + depth).astype(np.int32), slots=np.stack([slots_for(tables[s], ctx[s] + np.arange(T)) for s in range(B)]),
                   masks=np.tile(pack_masks(ancestors(parents), T), (B, 1)), parents=np.tile(parents, B), u=rng.random(n, dtype=np.float32),
                   uf=rng.random(B, dtype=np.float32), target=target[flat], draft=draft[flat], ctx=ctx)
        for k, v in put.items():
            d[k].copy_(dev(v))
        if graph and turn == 1:                             # (the first step warmed every kernel up)
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                step(torch.cuda.current_stream())
        if captured:
            captured.replay()
        else:
            step(None)
        torch.cuda.synchronize()
        path, n_path, after = back(d["path"], np.int32).reshape(B, T), back(d["n_path"], np.int32), back(d["next"], np.int32)
        out = back(d["out"], np.uint16).reshape(B, T, H, 512)
        # the same tokens one by one
        for s in range(B):
            for k in range(n_path[s]):
                node, pos = path[s, k], int(ctx[s]) + k
                moved += node != k
                row, qr = dev(embed[tokens[s, node]]), dev(queries[tokens[s, node]][:, 512:])
                at, slot = dev(np.array([pos], np.int32)), dev(slots_for(tables[s], [pos]))
                hip.launch_rope_rows(row.data_ptr() + 1024, row.data_ptr() + 1024, table, at, 1, 1, 64, 400, W, W, W, W, False, True)
                hip.launch_rope_rows(qr, qr, table, at, 1, H, 64, 400, H * 64, 64, H * 64, 64, False, True)
                hip.launch_kv_append_paged(row, slot, plain_pool, 1, W, PT, n_pages)
                hip.launch_index_append_paged(dev(embed_keys[tokens[s, node]]), slot, plain_kpool, 1, HD, PT, n_pages)
                one = dzeros(H * 512 * 2)
                hip.launch_mla_attend_tree_paged(dev(queries[tokens[s, node]][:, :512]), qr, plain_pool, dev(tables[s]), at, dev(np.array([0, 1], np.int32)), None,
                                                 1, H, 1, 1, 300, blocks, 512, 64, PT, n_pages, 192 ** -0.5, one, None,
                                                 dzeros(max(hip.mla_attend_tree_paged_scratch_floats(1, H, 1, 1, 300), 4) * 4))
                a, b = bf16_to_f32(out[s, node]).astype(np.float64), bf16_to_f32(back(one, np.uint16).reshape(H, 512)).astype(np.float64)
                # the same rows in another order and under other maxima: two bf16 roundings of a result and of its weights
                assert np.linalg.norm(a - b) <= 4 * BF16 * np.linalg.norm(b), (turn, s, k)
                history[s].append(tokens[s, node])
        assert np.array_equal(back(d["lens"], np.int32), ctx + n_path)
        ctx, root = ctx + n_path, after
        got, want = back(pool).reshape(n_pages, -1), back(plain_pool).reshape(n_pages, -1)
        got_k, want_k = back(kpool, np.uint16).reshape(n_pages * PT, HD), back(plain_kpool, np.uint16).reshape(n_pages * PT, HD)
        for s in range(B):
            for t in range(ctx[s]):
                p, o = tables[s, t // PT], t % PT
                assert np.array_equal(got[p, o * W:(o + 1) * W], want[p, o * W:(o + 1) * W]), (turn, s, t)
                assert np.array_equal(got[p, PT * W + 4 * o:][:4], want[p, PT * W + 4 * o:][:4])
                assert np.array_equal(got_k[p * PT + o], want_k[p * PT + o])
    assert moved > 0 and (ctx > ctx0 + 3).any()
