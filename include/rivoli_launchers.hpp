// C++ mirror of the reference's host-side launcher layer for this path: one `launch_*`
// function per exported symbol, generated by a macro in the manner of `launchers!`
// (crates/backend/src/hip.rs:196-221), every call ending in `ensure_hip_status`
// (hip.rs:328-336, same wording: 0 ok, positive = argument guard, negative = -(hipError_t)).
// Names follow the Rust rows (crates/backend/src/hip_attn.rs); rows that exist only in this
// library keep the same `launch_<op>` -> `rivoli_<op>` convention. Header-only; link the
// shared library built from rivoli_amd/csrc.
#ifndef RIVOLI_LAUNCHERS_HPP
#define RIVOLI_LAUNCHERS_HPP

#include <stdexcept>
#include <string>

#include "rivoli_kvcache.h"

namespace rivoli {

// What `anyhow::bail!` carries in the reference: the launcher's tag and the raw code.
struct LaunchError : std::runtime_error {
    int code;
    LaunchError(const std::string& what, int c) : std::runtime_error(what), code(c) {}
};

inline void ensure_hip_status(int r, const char* name) {
    if (r == 0) return;
    if (r > 0) throw LaunchError(std::string(name) + ": argument guard rejected (" + std::to_string(r) + ")", r);
    throw LaunchError(std::string(name) + ": HIP error " + std::to_string(-r), r);
}

#define RIVOLI_LAUNCHER(fn, sym, tag)                 \
    template <class... Args>                          \
    inline void fn(Args... args) {                    \
        ensure_hip_status(sym(args...), tag);         \
    }

// rows the reference has (same argument lists: crates/backend/src/hip_attn.rs)
RIVOLI_LAUNCHER(launch_append_kv, rivoli_append_kv, "append_kv")
RIVOLI_LAUNCHER(launch_index_append, rivoli_index_append, "index_append")
RIVOLI_LAUNCHER(launch_index_topk, rivoli_index_topk, "index_topk")
RIVOLI_LAUNCHER(launch_index_score, rivoli_index_score, "index_score")
RIVOLI_LAUNCHER(launch_attend, rivoli_mla_attend, "mla_attend")
RIVOLI_LAUNCHER(launch_hash_rows, rivoli_hash_rows, "hash_rows")
RIVOLI_LAUNCHER(launch_act_quant_f8_prefix, rivoli_act_quant_f8_prefix, "act_quant_f8_prefix")
RIVOLI_LAUNCHER(launch_kv_compress_deposit, rivoli_kv_compress_deposit, "kv_compress_deposit")
RIVOLI_LAUNCHER(launch_kv_compress_prefill, rivoli_kv_compress_prefill, "kv_compress_prefill")
RIVOLI_LAUNCHER(launch_kv_compress_decode, rivoli_kv_compress_decode, "kv_compress_decode")
RIVOLI_LAUNCHER(launch_gather_attn_shared_kv, rivoli_gather_attn_shared_kv, "gather_attn_shared_kv")
RIVOLI_LAUNCHER(launch_act_quant_f4_rotated, rivoli_act_quant_f4_rotated, "act_quant_f4_rotated")
RIVOLI_LAUNCHER(launch_index_score_blocks, rivoli_index_score_blocks, "index_score_blocks")
// rows this library adds
RIVOLI_LAUNCHER(launch_index_score_blocks_prefill, rivoli_index_score_blocks_prefill, "index_score_blocks_prefill")
RIVOLI_LAUNCHER(launch_append_kv_rows, rivoli_append_kv_rows, "append_kv_rows")
RIVOLI_LAUNCHER(launch_kv_append_paged, rivoli_kv_append_paged, "kv_append_paged")
RIVOLI_LAUNCHER(launch_kv_gather_paged, rivoli_kv_gather_paged, "kv_gather_paged")
RIVOLI_LAUNCHER(launch_kv_gather_paged_packed, rivoli_kv_gather_paged_packed, "kv_gather_paged_packed")
RIVOLI_LAUNCHER(launch_kv_append_gather_paged, rivoli_kv_append_gather_paged, "kv_append_gather_paged")
RIVOLI_LAUNCHER(launch_kv_gather_rows_paged, rivoli_kv_gather_rows_paged, "kv_gather_rows_paged")
RIVOLI_LAUNCHER(launch_index_topk_batched, rivoli_index_topk_batched, "index_topk_batched")
RIVOLI_LAUNCHER(launch_index_append_paged, rivoli_index_append_paged, "index_append_paged")
RIVOLI_LAUNCHER(launch_index_score_paged, rivoli_index_score_paged, "index_score_paged")
RIVOLI_LAUNCHER(launch_index_score_paged_hist, rivoli_index_score_paged_hist, "index_score_paged_hist")
RIVOLI_LAUNCHER(launch_dsa_select_gather_paged, rivoli_dsa_select_gather_paged, "dsa_select_gather_paged")
RIVOLI_LAUNCHER(launch_dsa_select_gather_paged_noalloc, rivoli_dsa_select_gather_paged_noalloc,
                "dsa_select_gather_paged_noalloc")
RIVOLI_LAUNCHER(launch_attend_paged, rivoli_mla_attend_paged, "mla_attend_paged")
RIVOLI_LAUNCHER(launch_index_select_blocks, rivoli_index_select_blocks, "index_select_blocks")
RIVOLI_LAUNCHER(launch_sel_gather, rivoli_sel_gather, "sel_gather")
RIVOLI_LAUNCHER(launch_sel_gather_scored, rivoli_sel_gather_scored, "sel_gather_scored")
RIVOLI_LAUNCHER(launch_kv_ring_write, rivoli_kv_ring_write, "kv_ring_write")
RIVOLI_LAUNCHER(launch_gather_attn_shared_kv_bounded, rivoli_gather_attn_shared_kv_bounded, "gather_attn_shared_kv")
RIVOLI_LAUNCHER(launch_gather_attn_shared_kv_split, rivoli_gather_attn_shared_kv_split, "gather_attn_shared_kv")
RIVOLI_LAUNCHER(launch_rope_table, rivoli_rope_table, "rope_table")
RIVOLI_LAUNCHER(launch_rope_rows, rivoli_rope_rows, "rope_rows")
RIVOLI_LAUNCHER(launch_attend_tree_paged, rivoli_mla_attend_tree_paged, "mla_attend_tree_paged")
RIVOLI_LAUNCHER(launch_draft_verify, rivoli_draft_verify, "draft_verify")
RIVOLI_LAUNCHER(launch_kv_commit_paged, rivoli_kv_commit_paged, "kv_commit_paged")
RIVOLI_LAUNCHER(launch_index_commit_paged, rivoli_index_commit_paged, "index_commit_paged")
RIVOLI_LAUNCHER(launch_norm_rope_rows, rivoli_norm_rope_rows, "norm_rope_rows")
RIVOLI_LAUNCHER(launch_kv_norm_append_paged, rivoli_kv_norm_append_paged, "kv_norm_append_paged")
RIVOLI_LAUNCHER(launch_sample_rows, rivoli_sample_rows, "sample_rows")
RIVOLI_LAUNCHER(launch_attend_tree_shared_paged, rivoli_mla_attend_tree_shared_paged, "mla_attend_tree_shared_paged")
RIVOLI_LAUNCHER(launch_codec_e4m3_encode, rivoli_codec_e4m3_encode, "codec_e4m3_encode")
RIVOLI_LAUNCHER(launch_codec_e4m3_dequant_bf16, rivoli_codec_e4m3_dequant_bf16, "codec_e4m3_dequant_bf16")
RIVOLI_LAUNCHER(launch_codec_bf16_encode, rivoli_codec_bf16_encode, "codec_bf16_encode")
#undef RIVOLI_LAUNCHER

// hip.rs:339-342
inline void device_sync() { ensure_hip_status(rivoli_device_sync(), "device_sync"); }

// Sel::shape (crates/engine/src/v4/select.rs:350-361): throws where the reference refuses.
struct SelShape {
    int rows, cols;
};
inline SelShape sel_shape(int win, int ratio, int index_topk, int seqlen, int start_pos) {
    SelShape s{0, 0};
    ensure_hip_status(rivoli_sel_shape(win, ratio, index_topk, seqlen, start_pos, &s.rows, &s.cols), "sel_shape");
    return s;
}

// pure sizing functions, as attend_scratch_floats (hip_attn.rs:113-128)
inline size_t kv_page_bytes(int page_tokens, int width) { return rivoli_kv_page_bytes(page_tokens, width); }
inline size_t attend_scratch_floats(int H, int kvl) { return rivoli_mla_attend_scratch_floats(H, kvl); }
inline size_t attend_paged_scratch_floats(int n_seqs, int H, int max_rows) {
    return rivoli_mla_attend_paged_scratch_floats(n_seqs, H, max_rows);
}
inline size_t index_topk_workspace_bytes(int n_queries, int nt) { return rivoli_index_topk_workspace_bytes(n_queries, nt); }
inline size_t gather_attn_scratch_floats(int m, int h, int d, int topk) {
    return rivoli_gather_attn_scratch_floats(m, h, d, topk);
}

inline size_t attend_tree_paged_scratch_floats(int n_seqs, int H, int n_nodes, int max_nodes, int max_ctx) {
    return rivoli_mla_attend_tree_paged_scratch_floats(n_seqs, H, n_nodes, max_nodes, max_ctx);
}
inline size_t attend_tree_shared_paged_scratch_floats(int n_seqs, int n_groups, int H, int n_nodes, int max_nodes, int max_prefix,
                                                      int max_ctx) {
    return rivoli_mla_attend_tree_shared_paged_scratch_floats(n_seqs, n_groups, H, n_nodes, max_nodes, max_prefix, max_ctx);
}
inline size_t draft_verify_workspace_bytes(int n_seqs, int max_nodes, int vocab) {
    return rivoli_draft_verify_workspace_bytes(n_seqs, max_nodes, vocab);
}
inline size_t sample_rows_workspace_bytes(int n_rows, int vocab) { return rivoli_sample_rows_workspace_bytes(n_rows, vocab); }

}  // namespace rivoli

#endif
