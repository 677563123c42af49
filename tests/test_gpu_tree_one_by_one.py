"""A node's attention in a tree against the same token's alone: as the last of a chain of one behind the rows of its ancestors, and by the attention of
single queries (rivoli_mla_attend_paged), which takes q and gives results in f32."""
import numpy as np
import pytest

from rivoli_amd import hip
from tests.draft_cases import ancestors, bf16_rows, pack_masks, random_parents, random_pool
from tests.gpu_util import back, dev, dzeros
from tests.tree_precision import FLOOR, HALF, bf16_of
from tests.util import bf16_to_f32, shuffled_block_tables

pytestmark = pytest.mark.gpu

PAGE, W = 64, 576


def tree(qabs, qrope, pool, tables, ctx, cu, masks, max_nodes, scale):
    n, H = qabs.shape[:2]
    floats = hip.mla_attend_tree_paged_scratch_floats(len(ctx), H, n, max_nodes, int(max(ctx)))
    out = dzeros(n * H * 1024, 0xEE)
    hip.launch_mla_attend_tree_paged(dev(qabs), dev(qrope), dev(pool), dev(tables), dev(np.array(ctx, np.int32)), dev(cu), None if masks is None else dev(masks), len(ctx), H,
                                     n, max_nodes, int(max(ctx)), tables.shape[1], 512, 64, PAGE, len(pool), scale, out, None, dzeros(max(floats, 4) * 4, 0xFF))
    return bf16_to_f32(back(out, np.uint16)).reshape(n, H, 512).astype(np.float64)


@pytest.mark.parametrize("ctx,nodes,H", [([0, 61, 700], 9, 16), ([2500], 17, 8), ([127, 5000], 5, 64)])
def test_a_node_in_a_tree_is_the_token_alone(ctx, nodes, H):
    rng = np.random.default_rng(len(ctx) + H)
    seqs, scale = len(ctx), float(np.float32(192 ** -0.5))
    blocks = -(-(max(ctx) + nodes) // PAGE)
    tables = shuffled_block_tables(seqs, blocks, seqs * blocks + 1, 3)
    pool = random_pool(rng, seqs * blocks + 1, PAGE, W)
    qabs, qrope = bf16_rows(rng, (seqs * nodes, H, 512), 2.0), bf16_rows(rng, (seqs * nodes, H, 64), 2.0)
    cu = np.arange(0, seqs * nodes + 1, nodes, dtype=np.int32)
    seen = [ancestors(random_parents(rng, nodes)) for _ in range(seqs)]
    got = tree(qabs, qrope, pool, tables, ctx, cu, pack_masks(np.concatenate(seen), nodes), nodes, scale)
    for i in range(nodes):
        # every sequence's node i, its ancestors' rows behind the prefix in order, as a commit leaves them
        alone, depth = pool.copy(), np.array([s[i].sum() - 1 for s in seen])
        for s in range(seqs):
            for k, j in enumerate(np.flatnonzero(seen[s][i])):
                (a, o), (b, p) = divmod(ctx[s] + j, PAGE), divmod(ctx[s] + k, PAGE)
                alone[tables[s, b], p * W:(p + 1) * W] = pool[tables[s, a], o * W:(o + 1) * W]
                alone[tables[s, b], PAGE * W + 4 * p:][:4] = pool[tables[s, a], PAGE * W + 4 * o:][:4]
        at = np.array(ctx) + depth
        of = cu[:-1] + i
        one = tree(qabs[of], qrope[of], alone, tables, at, np.arange(seqs + 1, dtype=np.int32), None, 1, scale)
        # the same number to 2 (2^-11 + 2^-13), rounded: an element comes out a step (2^-7 of it at most) away with a likelihood of its error in steps
        assert np.linalg.norm(got[of] - one) <= 1.2 * np.sqrt(2 * (HALF + FLOOR) * 2.0 ** -7) * np.linalg.norm(one), i
        wide, lens = dzeros(seqs * H * 2048), dev((at + 1).astype(np.int32))
        floats = hip.lib().rivoli_mla_attend_paged_scratch_floats(seqs, H, int(at.max()) + 1)
        hip.launch_mla_attend_paged(dev(bf16_to_f32(qabs[of])), dev(bf16_to_f32(qrope[of])), dev(alone), dev(tables), lens, None, None, seqs, H, int(at.max()) + 1,
                                    tables.shape[1], 512, 64, PAGE, len(pool), scale, 2, wide, dzeros(max(floats, 4) * 4))
        # (its weights are bf16 pairs, of some 17 bits: nothing beside a rounding to bf16)
        want = back(wide, np.float32).reshape(seqs, H, 512).astype(np.float64)
        own = np.linalg.norm(bf16_of(want) - want)
        assert np.linalg.norm(got[of] - want) <= 1.1 * np.hypot(own, HALF * np.linalg.norm(want)) + FLOOR * np.linalg.norm(want), i
