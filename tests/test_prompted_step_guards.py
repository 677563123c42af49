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
    changes += [(dict(eps=NAN), 1001), (dict(kvl=1024), 1002), (dict(kvl=2 ** 31 - 16), 1002), (dict(n_tokens=2 ** 28 + 1), 1002), (dict(kvl=520), 1004),
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
