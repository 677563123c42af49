// How a tree attention call becomes work items: host arithmetic on the call's sizes alone (no length is known
// there), and the cut of the work by the device-side lengths that both of its kernels make.
#pragma once

namespace rk {

constexpr int kTreeRows = 64;             // of q (node, head) a workgroup
constexpr int kTreeTokens = 64;           // of a tile
constexpr int kTreeGroups = 256;          // workgroups, one per compute unit
constexpr int kTreeDies = 8;
constexpr int kTreeMinTiles = 4;          // a work item's least, but for what lengths leave
constexpr int kTreeWholeTiles = 8;        // up to these a block of rows is one workgroup's
constexpr int kTreeRecordFloats = kTreeRows * (512 + 2);

// `blocks`: most blocks of 64 rows. `groups` > 0: that many workgroups share the tiles of all blocks evenly, each leaving up to
// two partial records; 0: a workgroup has a whole block.
struct TreePlan {
    long long blocks;
    int groups;
};

static inline TreePlan tree_plan(int n_seqs, int H, int n_nodes, int max_nodes, int max_ctx) {
    TreePlan p{0, 0};
    if (n_seqs <= 0 || H <= 0 || n_nodes <= 0 || max_nodes <= 0 || max_ctx < 0) return p;
    const long long by_seq = ((long long)max_nodes * H + kTreeRows - 1) / kTreeRows * n_seqs;
    const long long by_node = (long long)n_nodes * H / kTreeRows + (n_seqs < n_nodes ? n_seqs : n_nodes);
    p.blocks = by_seq < by_node ? by_seq : by_node;
    const long long tiles = ((long long)max_ctx + max_nodes + kTreeTokens - 1) / kTreeTokens;
    if (tiles <= kTreeWholeTiles || p.blocks * tiles >= 1ll << 31) return p;  // (cut calls count their tiles in 32 bits)
    const long long groups = (p.blocks * tiles + kTreeMinTiles - 1) / kTreeMinTiles;
    p.groups = (int)(groups < kTreeGroups ? groups : kTreeGroups);
    return p;
}
static inline size_t tree_scratch_floats(const TreePlan& p) { return (size_t)p.groups * 2 * kTreeRecordFloats; }

}  // namespace rk
