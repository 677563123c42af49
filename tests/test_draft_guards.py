"""What the calls of a drafted step refuse, before anything is launched (no GPU: a refused call touches nothing), and
their sizing functions."""
import pytest
import torch

from rivoli_amd import hip

B = torch.zeros(4096)  # an aligned address; refused calls never read it


def refused(call, good, changes):
    for change, code in changes:
        args = dict(good)
        args.update(change)
        with pytest.raises(hip.LaunchError) as e:
            call(**args)
        assert e.value.code == code, change


def test_rope_table_refusals():
    good = dict(table=B, first=0, n_positions=8, rd=64, base=1e4)
    inf, nan = float("inf"), float("nan")
    refused(hip.launch_rope_table, good, [
        (dict(table=None), 1001), (dict(first=-1), 1001), (dict(n_positions=0), 1001), (dict(rd=0), 1001), (dict(base=1.0), 1001),
        (dict(base=nan), 1001), (dict(base=inf), 1001), (dict(factor=0.0), 1001), (dict(factor=nan), 1001), (dict(mscale=inf), 1001),
        (dict(orig_ctx=-1), 1001), (dict(orig_ctx=4096, beta_slow=0.0), 1001), (dict(orig_ctx=4096, beta_fast=1.0), 1001),
        (dict(orig_ctx=4096, beta_fast=nan), 1001), (dict(rd=1026), 1002), (dict(first=2 ** 31 - 4), 1002), (dict(rd=63), 1004),
        (dict(table=B.data_ptr() + 4), 1004)])


def test_rope_rows_refusals():
    good = dict(x=B, out=B, table=B, positions=B, n_tokens=1, n_heads=1, rd=64, n_positions=4, x_token_stride=64, x_head_stride=64,
                out_token_stride=64, out_head_stride=64, half=False, bf16=True)
    refused(hip.launch_rope_rows, good, [
        (dict(x=None), 1001), (dict(out=None), 1001), (dict(table=None), 1001), (dict(positions=None), 1001), (dict(n_tokens=0), 1001),
        (dict(n_heads=0), 1001), (dict(rd=-2), 1001), (dict(n_positions=0), 1001), (dict(rd=1026), 1002),
        (dict(n_tokens=2 ** 31 - 1, n_heads=64), 1002), (dict(rd=63), 1004), (dict(x=B.data_ptr() + 1), 1004),
        (dict(out=B.data_ptr() + 2, bf16=False), 1004), (dict(table=B.data_ptr() + 4), 1004)])


def test_tree_attention_refusals():
    good = dict(qabs=B, qrope=B, pool=B, block_table=B, ctx_lens=B, cu_nodes=B, masks=None, n_seqs=1, H=16, n_nodes=4, max_nodes=4,
                max_ctx=128, max_blocks_per_seq=3, kvl=512, rope=64, page_tokens=64, n_pages=3, scale=1.0, clat=B, lse=None, partial=B)
    changes = [(dict([(name, None)]), 1001) for name in ("qabs", "qrope", "pool", "block_table", "ctx_lens", "cu_nodes", "clat")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_seqs", "H", "n_nodes", "max_nodes", "max_blocks_per_seq", "kvl", "rope",
                                                      "page_tokens", "n_pages")]
    changes += [(dict(max_ctx=-1), 1001), (dict(n_seqs=65536), 1002), (dict(max_nodes=4097), 1002), (dict(max_ctx=2 ** 31 - 8192), 1002),
                (dict(n_nodes=2 ** 27), 1002), (dict(page_tokens=2 ** 22 + 4), 1002), (dict(kvl=640), 1004), (dict(kvl=192), 1004), (dict(rope=12), 1004), (dict(rope=72), 1004),
                (dict(page_tokens=6), 1004)]
    changes += [(dict([(name, B.data_ptr() + 8)]), 1004) for name in ("qabs", "qrope", "pool", "clat", "partial")]
    refused(hip.launch_mla_attend_tree_paged, good, changes)
    # where partial records are needed a call without room for them is refused
    if hip.mla_attend_tree_paged_scratch_floats(4, 64, 32, 8, 32768):
        refused(hip.launch_mla_attend_tree_paged, dict(good, n_seqs=4, H=64, n_nodes=32, max_nodes=8, max_ctx=32768), [(dict(partial=None), 1001)])
    assert hip.mla_attend_tree_paged_scratch_floats(0, 64, 32, 8, 32768) == 0


def test_verify_refusals():
    good = dict(target_probs=B, draft_probs=B, tokens=B, parents=B, cu_nodes=B, uniforms=B, final_uniforms=B, n_seqs=1, n_nodes=4, max_nodes=4,
                vocab=32, target_stride=32, draft_stride=32, bf16=False, path=B, n_path=B, next_token=B, workspace=B)
    changes = [(dict([(name, None)]), 1001) for name in ("target_probs", "tokens", "parents", "cu_nodes", "uniforms", "final_uniforms", "path",
                                                        "n_path", "next_token")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_seqs", "n_nodes", "max_nodes", "vocab")]
    changes += [(dict(max_nodes=1025), 1002), (dict(vocab=2 ** 21 + 1, target_stride=2 ** 22, draft_stride=2 ** 22), 1002),
                (dict(target_stride=31), 1002), (dict(draft_stride=31), 1002), (dict(target_probs=B.data_ptr() + 2), 1004),
                (dict(draft_probs=B.data_ptr() + 1, bf16=True), 1004), (dict(workspace=B.data_ptr() + 8), 1004)]
    refused(hip.launch_draft_verify, good, changes)
    # where rows are shared among workgroups a call without room for their sums is refused
    wide = dict(n_seqs=2, max_nodes=4, vocab=131072)
    assert hip.draft_verify_workspace_bytes(**wide) > 0
    refused(hip.launch_draft_verify, dict(good, target_stride=131072, draft_stride=131072, **wide), [(dict(workspace=None), 1001)])
    assert hip.draft_verify_workspace_bytes(1, 4, 32) == hip.draft_verify_workspace_bytes(0, 4, 131072) == 0


@pytest.mark.parametrize("call,width,stride", [(hip.launch_kv_commit_paged, "width", "layer_bytes"),
                                               (hip.launch_index_commit_paged, "hd", "layer_keys")])
def test_commit_refusals(call, width, stride):
    pool = "pool" if width == "width" else "kpool"
    good = dict(block_table=B, ctx_lens=B, path=B, n_path=B, n_seqs=1, max_path=4, max_blocks_per_seq=2, page_tokens=64, n_pages=2)
    good.update({pool: B, width: 576 if width == "width" else 128})
    changes = [(dict([(name, None)]), 1001) for name in (pool, "block_table", "ctx_lens", "path", "n_path")]
    changes += [(dict([(name, 0)]), 1001) for name in ("n_seqs", "max_path", "max_blocks_per_seq", width, "page_tokens", "n_pages", "n_layers")]
    changes += [(dict(new_lens=B), 1001), (dict(n_seqs=65536), 1002), (dict([(width, 2048)]), 1002), (dict([("n_layers", 2), (stride, 16)]), 1002),
                (dict([(width, 100)]), 1004), (dict([(pool, B.data_ptr() + 8)]), 1004)]
    if width == "width":
        changes += [(dict(page_tokens=6), 1004), (dict(n_layers=2, layer_bytes=2 * 37120 + 8), 1004)]
    refused(call, good, changes)
