// How a tree attention call becomes work items: host arithmetic on the call's sizes alone (no length is known
// there), and the cut of the work by the device-side lengths that both of its kernels make.
#pragma once

namespace rk {

constexpr int kTreeRows = 64;             // of q (node, head) a workgroup
constexpr int kTreeTokens = 64;           // of a tile
constexpr int kTreeGroups = 256;          // workgroups, one per compute unit
constexpr int kTreeDies = 8;
// A work item's least tiles, but for what the lengths leave. Fewer are not worth their records: 8 blocks of 32 tiles 19.6 us by two, 24.9 by
// one, 21.6 by four; 1 block of 126 tiles 27.6, 42.5, 26.8. Calls of up to kTreeFewTiles are cut to single tiles: 1 block of 4 or 9 tiles 14.3 us,
// by two 16.3.
constexpr int kTreeMinTiles = 2, kTreeFewTiles = 64;
// What a block costs a work item to begin with and end, in tiles: 13 ragged sequences of up to 79 tiles, 3 blocks each, 33.6 us, by three tiles 35.7, as
// nothing over 44; 8 of 63 tiles, 8 blocks each, 60.1 and 65.5; 1 of 513, 8 blocks, 61.7 and 65.8; but 64 ragged of up to 32, 4 blocks, 52.9 and 51.8. Seven or nine
// lose more there. Nothing in calls of less than a tile a workgroup: 8 blocks of 16 17.1 us, and 20.1.
constexpr unsigned kTreeBeginTiles = 5;
// Blocks of up to this many tiles are a workgroup's each, where there are kTreeWholeBlocks of them or two tiles at most: 32 blocks of 5 tiles 20.0 us,
// cut 24.6; 64 of 6 22.7 and 29.4; but 8 of 16 28.1 and 17.2, 1 of 9 25.0 and 14.3.
constexpr int kTreeWholeTiles = 8, kTreeWholeBlocks = 32;
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
    const long long most = p.blocks * tiles;
    if (tiles <= 2 || (tiles <= kTreeWholeTiles && p.blocks >= kTreeWholeBlocks)) return p;
    if (most >= 1ll << 29) return p;  // (cut calls count their tiles in 32 bits; nor is there anything to gain)
    const long long groups = most <= kTreeFewTiles ? most : most / kTreeMinTiles > kTreeFewTiles ? most / kTreeMinTiles : kTreeFewTiles;
    p.groups = (int)(groups < kTreeGroups ? groups : kTreeGroups);
    return p;
}
static inline size_t tree_scratch_floats(const TreePlan& p) { return (size_t)p.groups * 2 * kTreeRecordFloats; }

}  // namespace rk
