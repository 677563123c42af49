"""Calls of a drafted step that a launch does not hold (2^32 threads) are refused by their guard, before anything is launched. (No GPU: a refused call touches nothing.)"""
import torch

from rivoli_amd import hip
from tests.test_draft_guards import refused

B = torch.zeros(4096)


def test_rotation_tables_past_a_launch():
    # 16 positions a thread: 2^27 runs of 512 pairs are 2^36 threads; 2^27 of 32 pairs 2^32
    good = dict(table=B, first=0, n_positions=2 ** 31 - 2, rd=1024, base=1e4)
    refused(hip.launch_rope_table, good, [(dict(), 1002), (dict(rd=64), 1002), (dict(rd=66, n_positions=2 ** 31 - 64), 1002)])


def test_tree_attention_past_a_launch():
    good = dict(qabs=B, qrope=B, pool=B, block_table=B, ctx_lens=B, cu_nodes=B, masks=None, n_seqs=8192, H=1, n_nodes=2 ** 24, max_nodes=4096,
                max_ctx=0, max_blocks_per_seq=64, kvl=256, rope=64, page_tokens=64, n_pages=3, scale=1.0, clat=B, lse=None, partial=B)
    refused(hip.launch_mla_attend_tree_paged, good, [
        (dict(), 1002),                                                               # a workgroup of 256 a node
        (dict(kvl=512, H=64, n_nodes=2 ** 24, max_nodes=1024, n_seqs=65535, max_ctx=2 ** 20), 1002)])  # and a whole block of 64 rows


def test_verification_past_a_launch():
    good = dict(target_probs=B, draft_probs=None, tokens=B, parents=B, cu_nodes=B, uniforms=B, final_uniforms=B, n_seqs=2 ** 22, n_nodes=4, max_nodes=4,
                vocab=32, target_stride=32, draft_stride=32, bf16=False, path=B, n_path=B, next_token=B, workspace=B)
    refused(hip.launch_draft_verify, good, [(dict(), 1002), (dict(n_seqs=2 ** 31 - 1), 1002)])


def test_commits_past_a_launch():
    good = dict(block_table=B, ctx_lens=B, path=B, n_path=B, n_seqs=1, max_path=4, max_blocks_per_seq=2, page_tokens=64, n_pages=2, n_layers=65536)
    refused(hip.launch_kv_commit_paged, dict(good, pool=B, width=576, layer_bytes=2 * 37120), [(dict(), 1002), (dict(n_layers=2 ** 31 - 1), 1002)])
    refused(hip.launch_index_commit_paged, dict(good, kpool=B, hd=128, layer_keys=128), [(dict(), 1002), (dict(n_layers=2 ** 31 - 1), 1002)])


def test_pools_whose_bytes_pass_64_bits():
    """2^30 tokens of 1 028 bytes in 2^23 pages are past 2^63: no distance between layers holds them."""
    good = dict(pool=B, block_table=B, ctx_lens=B, path=B, n_path=B, n_seqs=1, max_path=4, max_blocks_per_seq=2, width=1024, page_tokens=2 ** 30, n_pages=2 ** 23,
                n_layers=2, layer_bytes=2 ** 62)
    refused(hip.launch_kv_commit_paged, good, [(dict(), 1002), (dict(n_pages=2 ** 24), 1002), (dict(layer_bytes=-16), 1002)])
