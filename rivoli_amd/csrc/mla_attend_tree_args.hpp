// What the kernels of tree attention take, and a sequence of a call's as they see it.
#pragma once
#include "attend_common.hpp"
#include "mla_attend_tree_plan.hpp"

namespace rk {

struct TreeArgs {
    const uint16_t *qabs, *qrope;  // [n_nodes][H][kvl], [n_nodes][H][rope], bf16
    const uint8_t* pool;
    const int *block_table, *ctx_lens, *cu_nodes;
    const uint32_t* masks;  // [n_nodes][mask_words]; null: node i sees drafted rows 0 .. i
    int n_seqs, H, n_nodes, max_nodes, mask_words, max_ctx, max_blocks;
    int kvl, rope, row_w, page_tokens, n_pages;
    size_t page_bytes;
    float qscale;           // softmax scale * log2(e), kept from zero: results are divided by it
    uint16_t* clat;
    float* lse;
    int groups;             // TreePlan's
    float* partial;
    unsigned int* bad_rows;
};

// A sequence's cached rows and its nodes, held to what the call says there is.
struct TreeSeq {
    int ctx, node0, nodes;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int seq) {
    TreeSeq s;
    s.ctx = min(max(a.ctx_lens[seq], 0), a.max_ctx);
    s.node0 = min(max(a.cu_nodes[seq], 0), a.n_nodes);
    const long long held = (long long)a.cu_nodes[seq + 1] - s.node0;
    s.nodes = (int)min(max(held, 0ll), (long long)min(a.max_nodes, a.n_nodes - s.node0));
    return s;
}

}  // namespace rk
