// Tree attention for sequences of which whole groups have the same first pages. Launch-only.
//
// A call is cut into the tiles of two kinds of parts: the rows (node, head) of a group's sequences, all together, over the pages that they share, and a sequence's rows over its
// cached rows behind those and its nodes. Rows of several sequences fill blocks of 64 where one's would not: of 16 heads four sequences go through a shared tile for what one would
// cost alone. Both kinds are tree_part()'s work, dealt as one line of units to the workgroups; each leaves records of its sums, which the merge puts together by row:
// a sequence's own in its blocks, its group's wherever the row is in the group's.
#include <climits>
#include <cmath>
#include <type_traits>
#include <utility>

#include "rivoli_kvcache.h"

#include "mla_attend_tree_args.hpp"
#include "mla_attend_tree.hpp"

namespace rk {

struct SharedArgs : TreeArgs {
    const int *cu_groups, *prefix_lens;
    int n_groups, max_prefix;
    long long records;           // that there is room for
};

// A part: rows of `s` over s.ctx cached rows from `first` on and, of a sequence, its nodes.
struct SharedPart {
    TreeSeq s;
    int seq, first;              // whose pages they are; 0: a group's part, or a sequence's that shares nothing
    int group;                   // of a sequence that shares
};
// A group's sequences, from lo to below hi.
struct SharedGroup {
    int lo, hi;
};
__device__ __forceinline__ SharedGroup shared_group(const SharedArgs& a, int g) {
    SharedGroup r;
    r.lo = min(max(a.cu_groups[g], 0), a.n_seqs), r.hi = min(max(a.cu_groups[g + 1], r.lo), a.n_seqs);
    return r;
}
// Its nodes, all of its sequences'.
__device__ __forceinline__ int2 shared_nodes(const SharedArgs& a, const SharedGroup& of) {
    const int node0 = min(max(a.cu_nodes[of.lo], 0), a.n_nodes);
    return int2{node0, min(max(a.cu_nodes[of.hi], node0), a.n_nodes) - node0};
}
// What is to be gained before a group's pages are attended apart, in tiles of a block: of each block of the group's rows, whose sums are written and read once more, and of a
// group. In us, shared and by sequence: 64 sequences of 16 heads behind 4 096 rows 48 and 60 (3 072 tiles saved, 16 blocks), 64 of 32 heads 55 and 62 (2 048; 32), 32 of 48
// heads in two groups behind 8 192 56 and 59 (512; 12 each), 64 of 16 heads behind 256 33 and 29 (192; 16), 2 behind 4 096 30 and 24 (64; 1), 32 of 64 heads behind 1 024 35
// and 31, 256 of 64 heads in 16 groups behind 512 106 and 56 (none saved).
constexpr long long kSharedBlockGain = 24, kSharedGroupGain = 256;
// The cached rows that a group shares: whole pages, where its rows fill enough fewer blocks together than sequence by sequence (as if its nodes were theirs evenly).
__device__ __forceinline__ int shared_rows(const SharedArgs& a, int g, const SharedGroup& of, int nodes) {
    int held = min(max(a.prefix_lens[g], 0), a.max_prefix);
    held -= held % a.page_tokens;
    const unsigned seqs = (unsigned)(of.hi - of.lo), rows = (unsigned)nodes * (unsigned)a.H;
    if (seqs < 2) return 0;
    const long long together = (rows + kTreeRows - 1) / kTreeRows, apart = (long long)seqs * (((rows + seqs - 1) / seqs + kTreeRows - 1) / kTreeRows);
    const long long tiles = ((long long)held + kTreeTokens - 1) / kTreeTokens;
    return (apart - together) * tiles > kSharedBlockGain * together + kSharedGroupGain ? held : 0;
}
__device__ __forceinline__ SharedPart shared_of_group(const SharedArgs& a, int g) {
    const SharedGroup of = shared_group(a, g);
    const int2 nodes = shared_nodes(a, of);
    SharedPart p;
    p.s.ctx = shared_rows(a, g, of, nodes.y);
    p.s.node0 = nodes.x, p.s.nodes = nodes.y;
    p.seq = min(of.lo, a.n_seqs - 1), p.first = 0, p.group = g;
    // the pages of the first that has so many rows: one that has not (an empty place in a batch) need not name them
    if (p.s.ctx > 0) {
        while (p.seq + 1 < of.hi && a.ctx_lens[p.seq] < p.s.ctx) ++p.seq;
        if (min(a.ctx_lens[p.seq], a.max_ctx) < p.s.ctx) p.s.ctx = 0;
    }
    return p;
}
// The groups. Up to 64 (FEW), a lane has one, which sequences and how many rows they share, so that no lookup waits for another.
template <bool FEW>
struct SharedGroups {
    SharedGroup of{};
    int rows = 0;
    __device__ __forceinline__ explicit SharedGroups(const SharedArgs& a) {
        if (!FEW) return;
        const int g = min((int)(threadIdx.x & 63), a.n_groups - 1);
        of = shared_group(a, g), rows = shared_rows(a, g, of, shared_nodes(a, of).y);
    }
    // The group that a sequence is of and what it shares there (nothing: of none): the number of those that end in front of it.
    __device__ __forceinline__ int find(const SharedArgs& a, int seq, int& shared) const {
        int g = 0;
        if constexpr (FEW) {
            for (int k = 0; k < a.n_groups; ++k) g += __builtin_amdgcn_readlane(of.hi, k) <= seq;
            const int lo = __shfl(of.lo, g, kWave), held = __shfl(rows, g, kWave);
            shared = g < a.n_groups && lo <= seq ? held : 0;
            return g;
        } else {
            int hi = a.n_groups;
            while (g < hi) {
                const int mid = (g + hi) >> 1;
                if (a.cu_groups[mid + 1] <= seq) g = mid + 1;
                else hi = mid;
            }
            shared = 0;
            if (g < a.n_groups && a.cu_groups[g] <= seq) {
                const SharedGroup in = shared_group(a, g);
                shared = shared_rows(a, g, in, shared_nodes(a, in).y);
            }
            return g;
        }
    }
};
// A sequence whose cached rows end within its group's is by itself: what the group makes of its rows is left out.
template <bool FEW>
__device__ __forceinline__ SharedPart shared_of_seq(const SharedArgs& a, const SharedGroups<FEW>& groups, int seq) {
    SharedPart p{tree_seq(a, seq), seq, 0, 0};
    int shared;
    p.group = groups.find(a, seq, shared);
    if (shared <= p.s.ctx) p.first = shared, p.s.ctx -= shared;
    return p;
}

// The parts are numbered, groups' first; a lane has those numbered lane, lane + 64, ... (as TreeWalk).
struct SharedLane {
    SharedPart p;
    unsigned blocks, tiles;
};
template <bool FEW>
__device__ __forceinline__ SharedLane shared_lane(const SharedArgs& a, const SharedGroups<FEW>& groups, int part) {
    SharedLane l{};
    // (every lane is here: groups are in lanes)
    const SharedPart as_seq = shared_of_seq(a, groups, min(max(part - a.n_groups, 0), a.n_seqs - 1));
    if (part >= a.n_groups + a.n_seqs) return l;
    const bool group = part < a.n_groups;
    l.p = group ? shared_of_group(a, part) : as_seq;
    l.blocks = ((unsigned)l.p.s.nodes * (unsigned)a.H + kTreeRows - 1) / kTreeRows;
    l.tiles = ((unsigned)l.p.s.ctx + (group ? 0u : (unsigned)l.p.s.nodes) + kTreeTokens - 1) / kTreeTokens;
    if (l.tiles == 0) l.blocks = 0;
    return l;
}
// A block: its part, its numbers in the part and in all, and the unit of its first tile.
struct SharedBlock {
    SharedPart p;
    int rb;
    unsigned blocks, tiles, number, first_tile;
    bool group;
};
template <bool FEW>
struct SharedWalk {
    const SharedArgs& a;
    const SharedGroups<FEW> groups;
    const SharedLane first;      // of the first 64 parts
    __device__ __forceinline__ explicit SharedWalk(const SharedArgs& args) : a(args), groups(args), first(shared_lane(args, groups, threadIdx.x & 63)) {}
    __device__ __forceinline__ SharedLane lane_of(int p0) const { return p0 == 0 ? first : shared_lane(a, groups, p0 + (int)(threadIdx.x & 63)); }
    unsigned begin = 0;          // what a block costs to begin with, in tiles
    __device__ __forceinline__ unsigned units(const SharedLane& l) const { return l.blocks * (l.tiles + begin); }
    // Units in all; sets `begin`, and the blocks of groups' parts and of all.
    __device__ __forceinline__ unsigned total(unsigned& of_groups, unsigned& blocks) {
        unsigned t = 0, b = 0, g = 0;
        for (int p0 = 0; p0 < a.n_groups + a.n_seqs; p0 += kWave) {
            const SharedLane l = lane_of(p0);
            t += l.blocks * l.tiles, b += l.blocks;
            if (p0 + (int)(threadIdx.x & 63) < a.n_groups) g += l.blocks;
        }
        t = wave_total(wave_inclusive_sum(t)), blocks = wave_total(wave_inclusive_sum(b)), of_groups = wave_total(wave_inclusive_sum(g));
        begin = t <= kTreeGroups ? 0u : kTreeBeginTiles;
        return t + begin * blocks;
    }
    // The one that unit u is of.
    __device__ __forceinline__ bool block(unsigned u, SharedBlock& b) const {
        unsigned run_units = 0, run_blocks = 0;
        for (int p0 = 0; p0 < a.n_groups + a.n_seqs; p0 += kWave) {
            const SharedLane l = lane_of(p0);
            const unsigned upto_units = wave_inclusive_sum(units(l)), upto_blocks = wave_inclusive_sum(l.blocks);
            if (u < run_units + wave_total(upto_units)) {
                const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(u < run_units + upto_units));
                auto of = [&](unsigned v) -> unsigned { return (unsigned)__builtin_amdgcn_readlane((int)v, at); };
                b.p.s.ctx = (int)of((unsigned)l.p.s.ctx), b.p.s.node0 = (int)of((unsigned)l.p.s.node0), b.p.s.nodes = (int)of((unsigned)l.p.s.nodes);
                b.p.seq = (int)of((unsigned)l.p.seq), b.p.first = (int)of((unsigned)l.p.first), b.p.group = (int)of((unsigned)l.p.group);
                b.blocks = of(l.blocks), b.tiles = of(l.tiles), b.group = p0 + at < a.n_groups;
                const unsigned units_before = run_units + of(upto_units - units(l)), blocks_before = run_blocks + of(upto_blocks - l.blocks);
                b.rb = (int)((u - units_before) / (b.tiles + begin));
                b.number = blocks_before + (unsigned)b.rb;
                b.first_tile = units_before + (unsigned)b.rb * (b.tiles + begin) + begin;
                return true;
            }
            run_units += wave_total(upto_units), run_blocks += wave_total(upto_blocks);
        }
        return false;
    }
};

// What the merge goes by, left behind the records by the workgroups that begin a block's or a group's work: looking the parts up again took most of a merge's time.
struct SharedHead {
    unsigned of_groups, blocks;  // blocks of groups' parts, and all
    unsigned items, each, more;  // TreeItems
    unsigned begin, pad[2];
};
struct SharedNote {              // of a block; of a group: its first one
    unsigned first_tile, tiles;
    int node0, nodes, rb, first, group;
    unsigned number;
};
static_assert(sizeof(SharedHead) == 32 && sizeof(SharedNote) == 4 * kSharedNoteFloats, "as the plan counts them");
struct SharedNotes {
    SharedHead* head;
    SharedNote *groups, *blocks;
    long long n_blocks;
    __device__ __forceinline__ explicit SharedNotes(const SharedArgs& a) {
        head = reinterpret_cast<SharedHead*>(a.partial + a.records * kTreeRecordFloats);
        groups = reinterpret_cast<SharedNote*>(head + 1), blocks = groups + a.n_groups;
        n_blocks = a.records - 2 * a.groups;
    }
};

// A tile is bound by the issue of its instructions as the tree kernel's is: 4 430 cycles a workgroup, 2 176 of them matrix cores'. Outside of its tiles a workgroup spends another 37 500: groups and
// parts looked up by dependent loads, again for a further block, q through LDS, the first tile's way, records (both counted, as the slope and the rest of 64 sequences of 16 heads behind
// 16 384, 32 768 and 65 536 rows: 117, 188 and 330 thousand cycles a wave for 18, 34 and 66 tiles). Of these 32 768 rows, 8 192 shared tiles in 16 blocks and 519 of the sequences' own, it is a fifth of the launch, 88 us in a
// run of such calls, matrix cores busy for 39 %; 128 of 32 heads behind four prompts of 65 536 470 us, 0.96 PFLOP/s, 204 tiles a workgroup, matrix cores 48 %. FEW: up to 64 groups in lanes, looked up without a
// chain of loads: the last of these calls 487 us with its merge, by bisection 498; one prompt 103.3 and 103.7.
template <bool RUNS, bool FEW>
__global__ __launch_bounds__(kTreeThreads, 1) void mla_attend_shared_kernel(const SharedArgs a) {
    __shared__ __attribute__((aligned(1024))) TreeShared shared;
    const lds_ptr<TreeShared> sh = (lds_ptr<TreeShared>)&shared;
    if (threadIdx.x == 0) sh->grown = sh->dirty = sh->holed[0] = sh->holed[1] = -1;
    unsigned item = blockIdx.x, u, end, begin;
    SharedBlock b;
    {
        SharedWalk<FEW> walk(a);
        unsigned of_groups, blocks;
        const unsigned total = walk.total(of_groups, blocks);
        begin = walk.begin;
        const TreeItems items(a, max(total, 1u));
        if (item == 0 && threadIdx.x == 0) *SharedNotes(a).head = SharedHead{of_groups, total == 0 ? 0u : blocks, items.items, items.each, items.more, begin, {0, 0}};
        if (total == 0 || item >= items.items) return;
        // an eighth of the items on each die: neighbours, which often read the same tokens
        if (items.items % kTreeDies == 0) item = (item % kTreeDies) * (items.items / kTreeDies) + item / kTreeDies;
        u = items.lo(item), end = items.lo(item + 1);
        if (!walk.block(u, b)) return;
    }
    for (int number = 0;;) {
        const int lo = max((int)(u - b.first_tile), 0), hi = min((int)b.tiles, (int)(end - b.first_tile));
        // an item's own two records, of blocks that go on in others, or the block's
        const bool all = lo == 0 && hi == (int)b.tiles;
        const size_t slot = all ? (size_t)2 * a.groups + b.number : (size_t)2 * item + (lo == 0 ? 1 : 0);
        if (hi > lo && lo == 0 && threadIdx.x == 0) {
            const SharedNotes notes(a);
            const SharedNote note{b.first_tile, b.tiles, b.p.s.node0, b.p.s.nodes, b.rb, b.p.first, b.p.group, b.number};
            if ((long long)b.number < notes.n_blocks) notes.blocks[b.number] = note;
            if (b.group && b.rb == 0) notes.groups[b.p.group] = note;
        }
        if (hi > lo && (long long)slot < a.records)  // (more blocks than there are nodes for: prefix sums that are none)
            tree_part<RUNS, true>(a, sh, b.p.s, b.p.seq, b.rb, b.rb == (int)b.blocks - 1, lo, hi, all && !b.group && b.p.first == 0,
                                  a.partial + slot * kTreeRecordFloats, number, b.p.first, b.group);
        const unsigned next = b.first_tile + b.tiles;
        if (next >= end || next <= u) return;  // (the second: prefix sums that are none, whose units pass 32 bits)
        u = next;
        SharedWalk<FEW> walk(a);  // (looked up again: what it has would keep registers through the tiles)
        walk.begin = begin;
        if (!walk.block(u, b)) return;
    }
}

// A row's sums out of the records of a block's tiles, under the largest reference so far.
struct SharedSums {
    float m = -INFINITY, l = 0.0f;
    f32x4 sum = {0, 0, 0, 0};
    // The block with its first tile's unit and tiles, `number` of all; the row in it and the piece of a record.
    __device__ __forceinline__ void add(const SharedArgs& a, const SharedHead& head, unsigned first_tile, unsigned tiles, unsigned number, int row, int at, bool is) {
        const auto item_of = [&](unsigned unit) -> unsigned {
            const unsigned large = head.more * (head.each + 1);
            return min(unit < large ? unit / (head.each + 1) : head.more + (unit - large) / max(head.each, 1u), head.items - 1);
        };
        const unsigned g0 = is ? item_of(first_tile) : 1u, g1 = is ? item_of(first_tile + tiles - 1) : 0u;
        constexpr int kBatch = 8;
        for (unsigned from = 0; __builtin_amdgcn_ballot_w64(is && g0 + from <= g1) != 0; from += kBatch) {
            f32x2 ml[kBatch];
            f32x4 v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {  // (a record past the last re-reads the last, and is left out)
                const unsigned g = min(g0 + from + k, g1);
                const long long slot = !is ? 0 : g0 == g1 ? 2ll * a.groups + number : 2ll * g + (g == g0 ? 1 : 0);
                const float* const rec = a.partial + min(slot, a.records - 1) * kTreeRecordFloats;
                ml[k] = *reinterpret_cast<const f32x2*>(rec + kTreeRows * 512 + 2 * row);
                v[k] = reinterpret_cast<const f32x4*>(rec)[at];
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) top = is && g0 + from + k <= g1 ? fmaxf(top, ml[k].x) : top;
            if (top == -INFINITY) continue;     // nothing yet that the row sees
            const float keep = __builtin_amdgcn_exp2f(m - top);
            m = top, l *= keep, sum *= keep;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (!is || g0 + from + k > g1 || ml[k].y == 0.0f) continue;
                const float by = __builtin_amdgcn_exp2f(ml[k].x - top);
                l += ml[k].y * by;
                sum += v[k] * by;
            }
        }
    }
};

// Bound by a chain of reads, the head, notes, then records: 64 sequences behind one prompt 14 us, 128 16. (Of the records, 34 and 46 MB as the launch before writes them, 17 and 23 MB are fetched, 1.2 and 1.4 TB/s;
// the rest is still in the dies' second level. Counted.) Blocks of the sequences' parts, a column of the launch each, that are not whole without others' records: their own, then those of their group's blocks that have their rows.
__global__ __launch_bounds__(256) void mla_attend_shared_merge_kernel(const SharedArgs a) {
    const SharedNotes notes(a);
    const SharedHead head = *notes.head;
    const long long block = (long long)head.of_groups + blockIdx.x;
    if (block >= head.blocks || block >= notes.n_blocks) return;
    const SharedNote own = notes.blocks[block];
    // (held to what the call says there is: a note of prefix sums that are none may be none)
    const int node0 = min(max(own.node0, 0), a.n_nodes), nodes = min(max(own.nodes, 0), a.n_nodes - node0);
    const int at = blockIdx.y * 256 + threadIdx.x, lane = at & 63, idx = at >> 6;
    const int i = idx & 3, b = (idx >> 2) & 1, c = (idx >> 3) & 3, wave = idx >> 5;
    const int row = 32 * b + (lane & 31), r = kTreeRows * own.rb + row;
    const bool live = r >= 0 && r < nodes * a.H;
    if (__builtin_amdgcn_ballot_w64(live) == 0) return;
    if (own.first == 0) {  // a whole one's results are there already
        const unsigned large = head.more * (head.each + 1);
        const auto item_of = [&](unsigned unit) -> unsigned { return unit < large ? unit / (head.each + 1) : head.more + (unit - large) / max(head.each, 1u); };
        if (item_of(own.first_tile) == item_of(own.first_tile + own.tiles - 1)) return;
    }
    SharedSums s;
    s.add(a, head, own.first_tile, own.tiles, own.number, live ? row : 0, live ? at : 0, live);
    if (own.first != 0) {
        const SharedNote part = notes.groups[min(max(own.group, 0), a.n_groups - 1)];
        const int of = (node0 - part.node0) * a.H + r;
        const bool is = live && of >= 0 && of < part.nodes * a.H;
        const unsigned rb = is ? (unsigned)of / kTreeRows : 0u;
        const int its_row = is ? of & (kTreeRows - 1) : 0;
        const int its_at = is ? ((idx & ~4) | (its_row >> 5) << 2) * kWave + (lane & 32) + (its_row & 31) : 0;
        s.add(a, head, part.first_tile + rb * (part.tiles + head.begin), part.tiles, part.number + rb, its_row, its_at, is);
    }
    if (!live) return;
    const float inv = s.l == 0.0f ? 0.0f : 1.0f / (s.l * a.qscale);
    const size_t out = (size_t)node0 * a.H + r;
    *reinterpret_cast<u32x2*>(a.clat + out * 512 + 128 * wave + 16 * c + 64 * (i >> 1) + 8 * (i & 1) + 4 * (lane >> 5)) =
        u32x2{pack_bf16x2(s.sum[0] * inv, s.sum[1] * inv), pack_bf16x2(s.sum[2] * inv, s.sum[3] * inv)};
    if (a.lse && idx == 4 * b && lane < 32) a.lse[out] = s.l == 0.0f ? -INFINITY : (s.m + __builtin_amdgcn_logf(s.l)) * 0.6931471805599453f;
}

}  // namespace rk

extern "C" size_t rivoli_mla_attend_tree_shared_paged_scratch_floats(int n_seqs, int n_groups, int H, int n_nodes, int max_nodes, int max_prefix, int max_ctx) {
    if (n_groups <= 0 || max_prefix < 0) return 0;
    const rk::SharedPlan plan = rk::shared_plan(n_seqs, n_groups, H, n_nodes, max_nodes, max_prefix, max_ctx);
    return plan.groups ? rk::shared_scratch_floats(plan, n_groups) : rivoli_mla_attend_tree_paged_scratch_floats(n_seqs, H, n_nodes, max_nodes, max_ctx);
}

extern "C" int rivoli_mla_attend_tree_shared_paged(const unsigned short* qabs, const unsigned short* qrope,
                                                   const unsigned char* pool, const int* block_table, const int* ctx_lens,
                                                   const int* cu_nodes, const unsigned int* masks, const int* cu_groups,
                                                   const int* prefix_lens, int n_seqs, int n_groups, int H, int n_nodes,
                                                   int max_nodes, int max_prefix, int max_ctx, int max_blocks_per_seq,
                                                   int kvl, int rope, int page_tokens, int n_pages, float scale,
                                                   unsigned short* clat, float* lse, float* partial,
                                                   unsigned int* bad_rows, void* stream) {
    if (!cu_groups || !prefix_lens || n_groups <= 0 || max_prefix < 0) return 1001;
    if (n_groups > 65535) return 1002;
    const rk::SharedPlan plan = rk::shared_plan(n_seqs, n_groups, H, n_nodes, max_nodes, max_prefix, max_ctx);
    // rows of other widths, and calls past what is counted: every sequence by itself, through its own pages
    if (kvl != 512 || rope != 64 || plan.groups == 0)
        return rivoli_mla_attend_tree_paged(qabs, qrope, pool, block_table, ctx_lens, cu_nodes, masks, n_seqs, H, n_nodes, max_nodes, max_ctx,
                                            max_blocks_per_seq, kvl, rope, page_tokens, n_pages, scale, clat, lse, partial, bad_rows, stream);
    if (!qabs || !qrope || !pool || !block_table || !ctx_lens || !cu_nodes || !clat || max_blocks_per_seq <= 0 || page_tokens <= 0 || n_pages <= 0)
        return 1001;
    if (n_seqs > 65535 || max_nodes > 4096 || max_ctx > INT_MAX - 8192 || (long long)n_nodes * H > 1 << 30 || H > 262140 ||
        page_tokens > 1 << 22)
        return 1002;
    if (page_tokens % 4 != 0) return 1004;
    if (!rk::aligned16(qabs) || !rk::aligned16(qrope) || !rk::aligned16(pool) || !rk::aligned16(clat) || !rk::aligned16(partial)) return 1004;
    if (!partial) return 1001;
    float qscale = scale * rk::kLog2e;
    if (std::fabs(qscale) < 1e-20f) qscale = std::copysign(1e-20f, qscale);  // as good as nothing to any softmax
    const rk::SharedArgs a{{qabs, qrope, pool, block_table, ctx_lens, cu_nodes, masks, n_seqs, H, n_nodes, max_nodes, (max_nodes + 31) / 32,
                            max_ctx, max_blocks_per_seq, kvl, rope, kvl + rope, page_tokens, n_pages,
                            (size_t)page_tokens * (size_t)(kvl + rope + 4), qscale, clat, lse, plan.groups, partial, bad_rows},
                           cu_groups, prefix_lens, n_groups, max_prefix, plan.records};
    if (plan.blocks > (long long)(rk::kLaunchThreads / 256)) return 1002;
    const hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();
    const bool runs = page_tokens % 16 == 0, few = n_groups <= rk::kWave;
    rk::launch_kernel(runs ? few ? rk::mla_attend_shared_kernel<true, true> : rk::mla_attend_shared_kernel<true, false>
                           : few ? rk::mla_attend_shared_kernel<false, true> : rk::mla_attend_shared_kernel<false, false>, dim3((unsigned)plan.groups), dim3(rk::kTreeThreads), 0, st, a);
    const int rc = rk::launch_status();
    if (rc != 0) return rc;
    rk::launch_kernel(rk::mla_attend_shared_merge_kernel, dim3((unsigned)plan.blocks, 32), dim3(256), 0, st, a);
    return rk::launch_status();
}
