"""What the calls of a step behind shared prompts refuse, before anything is launched (no GPU: a refused call touches
nothing), and their sizing functions."""
import torch

from rivoli_amd import hip
from tests.test_draft_guards import refused

B = torch.zeros(4096)  # an aligned address; refused calls never read it
INF, NAN = float("inf"), float("nan")


def test_norm_rope_refusals():
    good = dict(x=B, out=B, weight=B, bias=B, table=B, positions=B, slots=B, n_tokens=1, n_heads=1, width=128, norm_n=128, rope_at=64, rd=64,
                n_positions=4, n_slots=4, x_token_stride=128, x_head_stride=128, out_token_stride=128, out_head_stride=128, weight_head_stride=0,
                eps=1e-6, center=False, half=False, x_bf16=True, out_bf16=True)
    changes = [(dict([(name, None)]), 1001) for name in ("x", "out", "table", "positions")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_tokens", "n_heads", "width", "norm_n", "n_positions", "n_slots")]
    changes += [(dict([(name, -2)]), 1001) for name in ("rope_at", "rd", "weight_head_stride")]
    changes += [(dict(eps=-1e-6), 1001), (dict(eps=INF), 1001), (dict(eps=NAN), 1001), (dict(width=1032), 1002), (dict(norm_n=129), 1002),
                (dict(rope_at=65), 1002), (dict(rope_at=2 ** 31 - 2), 1002), (dict(n_tokens=2 ** 31 - 1, n_heads=64), 1002),
                (dict(n_tokens=2 ** 31 - 1, n_heads=64, rd=62), 1002), (dict(rd=63), 1004), (dict(x=B.data_ptr() + 1), 1004),
                (dict(out=B.data_ptr() + 2, out_bf16=False), 1004), (dict(table=B.data_ptr() + 4), 1004), (dict(weight=B.data_ptr() + 2), 1004),
                (dict(bias=B.data_ptr() + 1), 1004)]
    refused(hip.launch_norm_rope_rows, good, changes)


def test_norm_append_refusals():
    good = dict(x=B, slot_mapping=B, weight=B, table=B, positions=B, pool=B, n_tokens=1, x_stride=576, kvl=512, rope=64, n_positions=4, page_tokens=64,
                n_pages=1, eps=1e-6, half=False, bf16=True)
    changes = [(dict([(name, None)]), 1001) for name in ("x", "slot_mapping", "table", "positions", "pool")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_tokens", "kvl", "rope", "n_positions", "page_tokens", "n_pages")]
    changes += [(dict(eps=NAN), 1001), (dict(kvl=1024), 1002), (dict(kvl=2 ** 31 - 16), 1002), (dict(n_tokens=2 ** 26), 1002), (dict(kvl=520), 1004),
                (dict(kvl=508, rope=68), 1004), (dict(kvl=520, rope=56, half=True), 1004), (dict(page_tokens=6), 1004), (dict(x_stride=580), 1004),
                (dict(x_stride=578, bf16=False), 1004), (dict(x=B.data_ptr() + 8), 1004), (dict(pool=B.data_ptr() + 8), 1004),
                (dict(table=B.data_ptr() + 4), 1004), (dict(weight=B.data_ptr() + 2), 1004)]
    refused(hip.launch_kv_norm_append_paged, good, changes)


def test_sample_refusals():
    good = dict(logits=B, temperatures=None, top_ks=None, top_ps=None, min_ps=None, uniforms=B, n_rows=1, vocab=32, stride=32, bf16=False, tokens=B,
                n_kept=None, logprobs=None, probs=B, probs_stride=32, workspace=B)
    changes = [(dict([(name, None)]), 1001) for name in ("logits", "uniforms", "tokens", "workspace")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_rows", "vocab")]
    changes += [(dict(n_rows=2 ** 22), 1002), (dict(vocab=2 ** 21 + 1, stride=2 ** 22, probs_stride=2 ** 22), 1002), (dict(stride=31), 1002),
                (dict(stride=-32), 1002), (dict(probs_stride=31), 1002), (dict(n_rows=2 ** 22 - 1, vocab=2 ** 21, stride=2 ** 21, probs_stride=2 ** 21), 1002),
                (dict(logits=B.data_ptr() + 2), 1004), (dict(logits=B.data_ptr() + 1, bf16=True), 1004), (dict(probs=B.data_ptr() + 2), 1004),
                (dict(workspace=B.data_ptr() + 8), 1004)]
    refused(hip.launch_sample_rows, good, changes)
    assert hip.sample_rows_workspace_bytes(0, 32) == hip.sample_rows_workspace_bytes(4, 0) == hip.sample_rows_workspace_bytes(4, 2 ** 21 + 1) == 0
    assert hip.sample_rows_workspace_bytes(4, 32) >= 4 * hip.sample_rows_workspace_bytes(1, 1) > 0


def test_shared_attention_refusals():
    good = dict(qabs=B, qrope=B, pool=B, block_table=B, ctx_lens=B, cu_nodes=B, masks=None, cu_groups=B, prefix_lens=B, n_seqs=1, n_groups=1, H=16,
                n_nodes=4, max_nodes=4, max_prefix=64, max_ctx=128, max_blocks_per_seq=3, kvl=512, rope=64, page_tokens=64, n_pages=3, scale=1.0, clat=B,
                lse=None, partial=B)
    changes = [(dict([(name, None)]), 1001) for name in ("qabs", "qrope", "pool", "block_table", "ctx_lens", "cu_nodes", "cu_groups", "prefix_lens", "clat",
                                                        "partial")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_seqs", "n_groups", "H", "n_nodes", "max_nodes", "max_blocks_per_seq", "kvl", "rope",
                                                      "page_tokens", "n_pages")]
    changes += [(dict(max_ctx=-1), 1001), (dict(max_prefix=-1), 1001), (dict(n_groups=65536), 1002), (dict(n_seqs=65536), 1002), (dict(max_nodes=4097), 1002),
                (dict(max_ctx=2 ** 31 - 8192), 1002), (dict(n_nodes=2 ** 27), 1002), (dict(n_nodes=2 ** 26, max_ctx=0, max_prefix=0, max_nodes=4096, n_seqs=65535), 1002), (dict(page_tokens=2 ** 22 + 4), 1002), (dict(kvl=640), 1004),
                (dict(kvl=192), 1004), (dict(rope=12), 1004), (dict(page_tokens=6), 1004)]
    changes += [(dict([(name, B.data_ptr() + 8)]), 1004) for name in ("qabs", "qrope", "pool", "clat", "partial")]
    refused(hip.launch_mla_attend_tree_shared_paged, good, changes)
    sizes = hip.mla_attend_tree_shared_paged_scratch_floats
    record = 64 * (512 + 2)
    assert sizes(0, 1, 16, 4, 4, 64, 128) == sizes(1, 0, 16, 4, 4, 64, 128) == 0
    # two records a workgroup, one a block (one of the sequence's own, two that the group's rows may fill), eight numbers for each of these, the group and the call
    assert sizes(1, 1, 16, 4, 4, 64, 125) == (2 * 5 + 1 + 2) * record + 8 * (1 + 2 + 1 + 1)
    # past 31 bits of tiles: what the call without groups asks for
    assert sizes(65535, 1, 128, 2 ** 23, 128, 0, 2 ** 31 - 8193) == hip.mla_attend_tree_paged_scratch_floats(65535, 128, 2 ** 23, 128, 2 ** 31 - 8193)
