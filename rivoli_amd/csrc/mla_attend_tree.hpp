// Tree attention for rows of 512 + 64 codes on the matrix cores, included by mla_attend_tree.hip and, for its tiles' work, mla_attend_shared.hip.
//
// What bounds it: of a tile of 64 tokens 64 rows of q need 64 * 64 * (576 + 512) multiply-adds, 2 176 cycles of a compute unit's four
// matrix cores at 512 a cycle, while its LDS moves 128 bytes a cycle. So no operand may pass through LDS more often than
// it must, and a fragment that is read has to serve many rows:
//   - a workgroup is 64 rows (any mixture of nodes and heads of one sequence) and four waves, one per SIMD on the whole register file;
//   - scores: wave (th, kh) has 32 tokens x all 64 rows over half of the dims, its q operands (144 registers) there for the whole
//     call; every byte of a key is read out of LDS once for the workgroup. The two halves' partial scores meet through LDS: each wave sends
//     32 rows and keeps the other 32, so that a score is handled once;
//   - values: a wave has 128 of the 512 columns for all 64 rows (128 accumulators); every byte of a value is read once, by the transposing
//     load, and only the weights (8 KB) are read by all four.
// Codes go from memory into LDS as they are, three tiles in rotation, and become bf16 for the scores and f16 for the values (both exact) when an
// operand is read, once for the workgroup. 32 x 32 matrix tiles: a fragment serves two of them.
// An iteration has two halves, a barrier behind each: the scores of tile i + 1, with tile i's softmax and the transfers of tile i + 2
// between their matrix instructions; then the values of tile i, with the partial scores of i + 1 meeting.
// A weight is its exponential times its token's scale, rounded once to f16, which codes are exact in as well. A row's reference makes the
// largest of these products 2^lift in its first tile; the row is rescaled only when some weight has grown to kTreeGrown, which every wave learns from a flag behind
// the first barrier (regrow). A weight below 2^-14 there is off by up to 2^-25, one below 2^-25 gone, so that the small weights of n tokens lose at most n 2^-25: where
// one early token outweighs a long flat rest that is a part of the result (with a lift of none 2^17 tokens of 2^-25 each lost 3.8e-3 of it). So the lift grows with a work
// item's tiles, floor(log2(tiles)) - 5, and n 2^-(25 + lift) stays below 2^-13 of that weight, a thirty-second of a result's half step; past 2^26 tokens, where the lift
// is held to 14 (2^15 is kTreeGrown), n 2^-39. Higher lifts leave less room to grow and rescale more often: 64 nodes of 128 heads over 131 072 tokens take 1 930 us by
// none, 1 954 by this one, 1 976 by two more; 32 sequences of 32 768 1 042, 1 031 and 1 067.
// Against 64 bits results are off by 1.6e-3 of the norm, their own rounding to bf16 (by bf16 weights 2.4e-3). The sum of the weights, and so lse, is of the unrounded ones, in f32.
// One wave a SIMD issues an instruction in four cycles at best and a matrix instruction of 32 cycles in sixteen, which leaves room for four
// others under each. So what counts beside the matrix instructions is how many others there are and what waits: fragments are asked for steps
// ahead of their use, control flow and a run's address are scalar, rare work sits behind flags. An iteration is 68 matrix instructions, 315 other vector and 55 LDS instructions a
// wave, 4 270 cycles (counted over 32 sequences of 32 768 tokens; 2 176 are of matrix instructions; with 70 more others 4 580).
// Measured: 32 sequences of 32 768 tokens, 8 nodes of 64 heads 1 030 to 1 085 us by the card, 1.13 to 1.08 PFLOP/s; 131 072 tokens, 64 nodes of 128 heads 1 955 to 2 040, 1.19 to 1.15, where
// a large bf16 product reaches 1.36. The clock follows the power: some 2.1 GHz here, 1.8 in a loop of nothing but these
// matrix instructions (1.86 PFLOP/s), so that an instruction saved gives about a quarter of its cycles. Short calls are bound by
// what a block costs to begin with and end (kTreeBeginTiles): 4 nodes of 16 heads over 200 tokens 13.4 us, 10 of them here (of some 20 000 cycles, 6 500 until the first tile and q are there, 2 000 until q is
// in its registers, 3 000 for the record).
#pragma once

namespace rk {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = kTreeWaves * kWave;
constexpr int kTreeBuffers = 3;
// A tile in LDS: eight rows after the other, 4 KB each: their latent codes in four groups of 128 bytes, a group's rows next to each
// other; then 1 KB of roped codes for each sixteen rows. A row's eight 16-byte pieces of a group change places by the row's number,
// (row >> 1) & 7, so that reads of one piece of sixteen rows meet in no bank; of the roped codes the first eight rows of
// sixteen have their four pieces in the lower 64 bytes then, the others in the upper.
constexpr int kTreeRopeAt = 8 * 4096;
constexpr int kTreeTileBytes = kTreeRopeAt + 4 * 1024;
constexpr int kTreeSteps = 18;            // of 16 dims a wave: 16 of its 256 latent dims, two of its 32 roped ones
// A row's largest weight of its first tile is 2^lift, later ones may grow to 2^15 (65 504 is the largest of 16 bits, 2^-14 the least with all of its bits).
constexpr uint16_t kTreeGrown = 0x7800;  // 2^15; a number with a sign bit counts as more (negative softmax scales)
constexpr int kTreeMostLift = 14;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
constexpr uint32_t kTreeHole = 0x80000000u;  // the scale of a token that is not there: -0

// A call's blocks of rows are numbered by sequence, and so are its work units: block after block what a block costs to begin with, counted in tiles,
// and its tiles; or the blocks themselves where a workgroup has a whole one. A lane has the lengths of the sequences lane, lane + 64, ...; counts fit 32 bits (tree_plan).
struct TreeLane {
    TreeSeq s;
    unsigned blocks, tiles;
};
__device__ __forceinline__ TreeLane tree_lane(const TreeArgs& a, int seq) {
    TreeLane l{tree_seq(a, min(seq, a.n_seqs - 1)), 0u, 0u};
    if (seq < a.n_seqs) {
        l.blocks = ((unsigned)l.s.nodes * (unsigned)a.H + kTreeRows - 1) / kTreeRows;
        l.tiles = ((unsigned)l.s.ctx + (unsigned)l.s.nodes + kTreeTokens - 1) / kTreeTokens;
    }
    return l;
}
struct TreeWalk {
    const TreeArgs& a;
    const TreeLane first;  // of the first 64 sequences
    __device__ __forceinline__ explicit TreeWalk(const TreeArgs& args) : a(args), first(tree_lane(args, threadIdx.x & 63)) {}
    __device__ __forceinline__ TreeLane lane_of(int s0) const { return s0 == 0 ? first : tree_lane(a, s0 + (int)(threadIdx.x & 63)); }
    unsigned begin = 0;    // what a block costs to begin with
    __device__ __forceinline__ unsigned units(const TreeLane& l, bool whole) const { return whole ? l.blocks : l.blocks * (l.tiles + begin); }
    // Units in all of a cut call; sets `begin`.
    __device__ __forceinline__ unsigned total() {
        unsigned tiles = 0, blocks = 0;
        for (int s0 = 0; s0 < a.n_seqs; s0 += kWave) {
            const TreeLane l = lane_of(s0);
            tiles += l.blocks * l.tiles, blocks += l.blocks;
        }
        tiles = wave_total(wave_inclusive_sum(tiles)), blocks = wave_total(wave_inclusive_sum(blocks));
        begin = tiles <= kTreeGroups ? 0u : kTreeBeginTiles;
        return tiles + begin * blocks;
    }
    // The block that unit u is of: its sequence, number and tiles in it, and the unit of its first tile in a cut call.
    struct Block {
        TreeSeq s;
        int seq, rb;
        unsigned blocks, tiles, first_tile;
    };
    __device__ __forceinline__ bool block(bool whole, unsigned u, Block& b) const {
        unsigned run = 0, cut_run = 0;
        for (int s0 = 0; s0 < a.n_seqs; s0 += kWave) {
            const TreeLane l = lane_of(s0);
            const unsigned mine = units(l, whole), upto = wave_inclusive_sum(mine), all = wave_total(upto);
            if (u < run + all) {
                const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(u < run + upto));
                auto of = [&](unsigned v) -> unsigned { return (unsigned)__builtin_amdgcn_readlane((int)v, at); };
                b.s.ctx = (int)of((unsigned)l.s.ctx), b.s.node0 = (int)of((unsigned)l.s.node0), b.s.nodes = (int)of((unsigned)l.s.nodes);
                b.seq = s0 + at, b.blocks = of(l.blocks), b.tiles = of(l.tiles);
                const unsigned rel = u - run - of(upto - mine);
                b.rb = (int)(whole ? rel : rel / (b.tiles + begin));
                const unsigned cut = units(l, false);
                b.first_tile = cut_run + of(wave_inclusive_sum(cut) - cut) + (unsigned)b.rb * (b.tiles + begin) + begin;
                return true;
            }
            run += all;
            cut_run += wave_total(wave_inclusive_sum(units(l, false)));
        }
        return false;
    }
};
// The work items of a cut call, the first `more` of them with a unit more than the others.
struct TreeItems {
    unsigned items, each, more;
    __device__ __forceinline__ TreeItems(const TreeArgs& a, unsigned total) {
        items = min(total <= kTreeFewTiles ? total : max(total / kTreeMinTiles, (unsigned)kTreeFewTiles), (unsigned)a.groups);
        if (items > kTreeDies) items = items / kTreeDies * kTreeDies;  // eighths of them stay on one die
        each = total / items, more = total - each * items;
    }
    __device__ __forceinline__ unsigned lo(unsigned item) const { return item * each + min(item, more); }
    __device__ __forceinline__ unsigned of(unsigned unit) const {
        const unsigned large = more * (each + 1);
        return unit < large ? unit / (each + 1) : more + (unit - large) / each;
    }
};

// f(0) .. f(N - 1), the numbers being constants of the compiler's.
template <int N, class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of<N>(static_cast<F&&>(f), std::make_integer_sequence<int, N>{});
}
// (Weights carry their token's scale times the softmax's: one number a token for both products; results are divided by the softmax's.)
struct TreeShared {
    uint8_t tiles[kTreeBuffers * kTreeTileBytes];
    f32x4 part[4][4][kWave];             // partial scores on their way to wave (th, kh)
    uint8_t weights[kTreeRows * kTreeTokens * 2];
    float scale[kTreeBuffers][kTreeTokens];  // of a tile's tokens, times the softmax's; kTreeHole: not there
    float spare[kWave];
    float top[2][kTreeRows], corr[kTreeRows], sum[2][kTreeRows], ref[kTreeRows];
    // numbers of the latest tile of which some row outgrew its reference, some score is no number, some token is not there
    int grown, dirty, holed[2];          // (the last by the tile's parity)
};
struct TreeFlags {
    int grown, dirty, holed;
};
static_assert(sizeof(TreeShared) <= 160 * 1024, "one workgroup per compute unit");

// A lane's sixteen bytes on their way to LDS, at `to` for the wave's first lane: from a scalar address and a lane's 32 bits, or (RUNS false) a lane's 64.
// PIECE: 128 bytes further in memory a piece (the instruction's offset, which counts in LDS as well) and 1024 in LDS. m0, the
// instruction's LDS base, is nobody else's here.
template <int PIECE, bool RUNS>
__device__ __forceinline__ void tree_dma(unsigned long long base, uint32_t off, const uint8_t* src, uint32_t to) {
    if constexpr (RUNS)
        asm volatile("s_add_i32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%4"
                     :: "v"(off), "s"(base), "s"(to), "n"((1024 - 128) * PIECE), "n"(128 * PIECE) : "memory", "m0", "scc");
    else
        asm volatile("s_add_i32 m0, %1, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:%3"
                     :: "v"(src), "s"(to), "n"((1024 - 128) * PIECE), "n"(128 * PIECE) : "memory", "m0", "scc");
}

// Four codes as f16, exact.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t c, uint32_t& lo, uint32_t& hi) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true));
}
__device__ __forceinline__ uint32_t pack_f16x2(float x, float y) {
    typedef float f32x2v __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v{x, y}), f16x2v));
}

// Codes that are no number as zeros.
__device__ __forceinline__ uint32_t numbers_only(uint32_t c) {
    const uint32_t nan = (((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
    return c & ~(nan * 0xffu);
}

// Tiles [tile_lo, tile_hi) of rows 64 rb .. of a sequence. `whole`: they are all it has, results go out; else its record.
// `number`: a count of the tiles the workgroup has had, for the flag. PARTS: the rows of `s` are cached from row `first` of the sequence on, whole pages in front of
// them; `cached`: they are those rows alone, and the nodes' own none of them.
template <bool RUNS, bool PARTS = false>
__device__ __forceinline__ void tree_part(const TreeArgs& a, const lds_ptr<TreeShared> sh, const TreeSeq& s, int seq, int rb, bool last_block,
                                          int tile_lo, int tile_hi, bool whole, float* rec, int& number, int first = 0, bool cached = false) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, n32 = lane & 31;
    const int th = wave & 1, kh = wave >> 1;  // its 32 tokens and its half of the dims, in the scores
    const lds_ptr<uint8_t> tiles = (lds_ptr<uint8_t>)&sh->tiles[0];
    const lds_ptr<uint8_t> weights = (lds_ptr<uint8_t>)&sh->weights[0];
    const int rows = s.nodes * a.H;           // of the sequence
    // what the block's last row may see: a chain's later nodes are nobody's business here
    const int last_row = min(kTreeRows * rb + kTreeRows, rows) - 1;
    const int len = PARTS && cached ? s.ctx : a.masks ? s.ctx + s.nodes : s.ctx + last_row / a.H + 1;
    const int n_tiles = min(tile_hi, (len + kTreeTokens - 1) / kTreeTokens) - tile_lo;
    const int lift = n_tiles < 64 ? 0 : min(26 - __builtin_clz((unsigned)n_tiles), kTreeMostLift);

    // ---- where a tile's rows are: eight lanes have rows 16 wave + 8 o + (lane >> 3) -----------------------------
    // Lookups and transfers have no branches, so that they go between the matrix instructions: tiles past the end are asked for too,
    // and a row's page and its place in it move on by a tile's tokens without a division. RUNS: pages are whole runs of 16 rows, so that the
    // wave's rows have one page and one place, which are scalar.
    const int l8 = lane & 7, r8 = lane >> 3;
    const int at_row = PARTS ? first : 0;
    const int end_row = at_row + min(len, tile_hi * kTreeTokens);
    const int* const table = a.block_table + (size_t)seq * a.max_blocks;
    const unsigned page_tokens = (unsigned)a.page_tokens, on_pages = kTreeTokens / page_tokens, on_rows = kTreeTokens % page_tokens;
    constexpr int kRuns = RUNS ? 1 : 2;
    int token[kRuns], page[kRuns];            // of the tile to be asked for
    unsigned block[kRuns], place[kRuns];      // of it; and of the next when that has been looked up
#pragma unroll
    for (int o = 0; o < kRuns; ++o) {
        token[o] = at_row + tile_lo * kTreeTokens + 16 * wave + (RUNS ? 0 : 8 * o + r8);
        block[o] = (unsigned)token[o] / page_tokens, place[o] = (unsigned)token[o] - block[o] * page_tokens;
    }
    int no_lane = 0;                          // (a vector zero: the page is a load of every lane, not a scalar one, which LDS reads would wait for)
    if (RUNS) asm volatile("" : "+v"(no_lane));
    auto look_up = [&](int o) { page[o] = table[min(block[o], (unsigned)a.max_blocks - 1) + no_lane]; };
    unsigned int missing = 0;                 // rows of the block's that have no page
    bool there[2];
    float raw_scale[2];
    auto swap_of = [&](int o) -> int { return (4 * o + (r8 >> 1)) & 7; };
    // of the roped codes a lane has the piece that its place asks for, of the first or the second eight rows
    const bool roped_second = (l8 ^ swap_of(0)) >= 4;
    const uint32_t page_bytes = (uint32_t)a.page_bytes, codes_bytes = page_tokens * 576u;
    const uint8_t* src[2] = {nullptr, nullptr};
    unsigned long long base = 0;              // RUNS: of the wave's rows
    const uint32_t lane_off[2] = {576u * (uint32_t)r8 + 16u * (uint32_t)(l8 ^ swap_of(0)), 576u * (uint32_t)(8 + r8) + 16u * (uint32_t)(l8 ^ swap_of(1))};
    const uint32_t roped_off = (roped_second ? lane_off[1] : lane_off[0]) + 512u;
    auto find = [&](int o) {  // the lane's row of a tile looked up: its address, and its scale asked for
        if constexpr (RUNS) {
            const unsigned at = (unsigned)__builtin_amdgcn_readfirstlane(page[0]);
            const bool has = block[0] < (unsigned)a.max_blocks && at < (unsigned)a.n_pages;
            const bool mine = token[0] + 8 * o + r8 < end_row;
            there[o] = mine & has;
            missing += mine & !has;
            const uint8_t* const run = a.pool + (unsigned long long)(has ? at : 0u) * page_bytes;
            raw_scale[o] = *reinterpret_cast<const float*>(run + codes_bytes + 4u * place[0] + 4u * (8u * o + r8));
            base = (unsigned long long)(uintptr_t)run + 576u * place[0];
        } else {
            const bool mine = token[o] < end_row;
            there[o] = mine & (block[o] < (unsigned)a.max_blocks) & ((unsigned)page[o] < (unsigned)a.n_pages);
            missing += mine & !there[o];
            const unsigned off = there[o] ? place[o] : 0u;
            const uint8_t* const from = a.pool + (unsigned long long)(there[o] ? (unsigned)page[o] : 0u) * page_bytes;
            raw_scale[o] = *reinterpret_cast<const float*>(from + (codes_bytes + 4u * off));
            src[o] = from + (off * 576u + 16u * (unsigned)(l8 ^ swap_of(o)));
        }
    };
    // Of the tile found: piece k of nine, four of either octet's latent codes and the roped ones.
    auto bring = [&](auto number_of, int buf) {
        constexpr int k = decltype(number_of)::value, o = k / 4;
        const uint32_t tile = (uint32_t)(uintptr_t)(tiles + buf * kTreeTileBytes);
        if constexpr (k < 8) tree_dma<k % 4, RUNS>(base, lane_off[o], src[o], tile + (2 * wave + o) * 4096);
        else tree_dma<0, RUNS>(base, roped_off, (roped_second ? src[1] : src[0]) + 512, tile + kTreeRopeAt + wave * 1024);
    };
    auto go_on = [&](int o) {
        if (o >= kRuns) return;
        token[o] += kTreeTokens;
        place[o] += on_rows;
        const bool over = place[o] >= page_tokens;
        place[o] -= over ? page_tokens : 0u;
        block[o] += on_pages + (over ? 1u : 0u);
        look_up(o);
    };
    auto ask = [&](int buf) {
        find(0), find(1);
        each<9>([&](auto k) { bring(k, buf); });
        go_on(0), go_on(1);
    };
    // The transfers asked for have landed: scales, and (holes) zeros for rows that are not there: codes must be finite, they meet a zero
    // weight. A scale that is not a positive number cannot come from the append: such a row is not there.
    bool ok[2];
    unsigned long long holes = 0;
    auto arrived = [&](int buf) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            ok[o] = there[o] & (raw_scale[o] > 0.0f);
            // (a row's eight lanes: the first has its place, the others a spare one, which costs less than a branch)
            const lds_ptr<float> to = l8 == 0 ? &sh->scale[buf][16 * wave + 8 * o + r8] : &sh->spare[lane];
            *to = ok[o] ? raw_scale[o] * a.qscale : __uint_as_float(kTreeHole);
        }
        holes = __builtin_amdgcn_ballot_w64(!(ok[0] & ok[1]));
    };
    auto fill_holes = [&](int buf, int of) {
        if (__builtin_expect(holes == 0, 1)) return;
        sh->holed[of & 1] = of;
#pragma unroll
        for (int o = 0; o < 2; ++o)
            if (!ok[o]) {
                const lds_ptr<uint8_t> to = tiles + buf * kTreeTileBytes + 16 * lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) *(lds_ptr<u32x4>)(to + (2 * wave + o) * 4096 + 1024 * i) = u32x4{0, 0, 0, 0};
                if ((l8 ^ swap_of(o)) < 4) *(lds_ptr<u32x4>)(to + kTreeRopeAt + wave * 1024) = u32x4{0, 0, 0, 0};
            }
    };

    f32x16 o[4][2];  // O^T: column tile c of 32, row block b: sixteen columns a lane, of row 32 b + n32
    float m_ref = -INFINITY, l_sum = 0.0f, l_before = 0.0f;  // of row 32 kh + n32: the lane's share of the sum
    const int own = 32 * kh + n32;
    const int own_row = kTreeRows * rb + own;
    const bool live = own_row < rows;
    const int own_node = (live ? own_row : 0) / a.H;

    if (n_tiles > 0) {
        // ---- the rows' operands: K-steps of 16 dims, eight a lane. Two K-steps share a 16-byte piece of codes. They live in the
        // accumulation half of the register file, which the matrix instructions read as well; the sums are in the other. They come through the
        // second and third tile's LDS, a row a transfer (a lane's own loads of 32 rows each took 9 600 cycles, this 3 700): a row's 16-byte pieces change
        // places by its number. The first page is asked for in front of them, where it can be by the scalar cache's way, which they are not waited for with.
        const lds_ptr<uint8_t> q_at = tiles + kTreeTileBytes;
        static_assert(kTreeRows * (1024 + 128) == 2 * kTreeTileBytes, "the rows fill two tiles");
        if constexpr (RUNS) page[0] = ((const __attribute__((address_space(4))) int*)(uintptr_t)table)[min(block[0], (unsigned)a.max_blocks - 1)];
        else look_up(0), look_up(1), ask(0);
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
            const int r = kTreeRows * rb + 16 * wave + i;
            dma16_from(reinterpret_cast<const uint8_t*>(a.qabs + ((size_t)s.node0 * a.H + (r < rows ? r : 0)) * 512), 16u * (uint32_t)(lane ^ i),
                       q_at + 1024 * (16 * wave + i));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = kTreeRows * rb + 16 * wave + 8 * i + r8;
            dma16(reinterpret_cast<const uint8_t*>(a.qrope + ((size_t)s.node0 * a.H + (r < rows ? r : 0)) * 64) + 16 * (l8 ^ r8),
                  (lds_ptr<uint8_t>)(uintptr_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(q_at + 1024 * kTreeRows + 128 * (16 * wave + 8 * i))));
        }
        if constexpr (RUNS) ask(0);
        arrived(0);
        lds_barrier();
        u32x4 q[kTreeSteps][2];  // of the rows that are the wave's in the softmax, and of the others
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int r = 32 * (b ^ kh) + n32;
            u32x4 raw[kTreeSteps];
#pragma unroll
            for (int j = 0; j < kTreeSteps; ++j)
                raw[j] = j < 16 ? *(lds_ptr<u32x4>)(q_at + 1024 * r + 16 * ((32 * kh + 4 * (j >> 1) + 2 * half + (j & 1)) ^ (r & 15)))
                                : *(lds_ptr<u32x4>)(q_at + 1024 * kTreeRows + 128 * r + 16 * ((4 * kh + 2 * half + (j & 1)) ^ (r & 7)));
#pragma unroll
            for (int j = 0; j < kTreeSteps; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t kept;
                    asm volatile("v_accvgpr_write_b32 %0, %1" : "=a"(kept) : "v"(raw[j][k]));
                    q[j][b][k] = kept;
                }
        }
        fill_holes(0, number);
        lds_barrier();  // (the next tile comes where they were)

        // ---- the lane's operands of a tile --------------------------------------------------------------------
        const int k_swap = (n32 >> 1) & 7, e8 = (lane & 15) >> 1;
        const int k_row = (4 * th + (n32 >> 3)) * 4096 + 2048 * kh + (n32 & 7) * 128;
        const int k_rope = kTreeRopeAt + (2 * th + (n32 >> 4)) * 1024 + (n32 & 7) * 128 + 16 * ((2 * kh + half) ^ k_swap);
        // values: of sixteen lanes, pair e addresses row 8 half + e of sixteen tokens; column tile c is piece c of group `wave` and, in
        // the other sixteen lanes, c + 4, which keeps the two in different banks
        const int v_swap = 4 * half + (e8 >> 1);
        const int v_row = half * 4096 + wave * 1024 + e8 * 128 + 8 * (lane & 1);
        const int v_piece = 4 * ((lane >> 4) & 1);
        auto as_bf16 = [](uint32_t x, uint32_t y) -> bf16x8 {
            uint32_t d0, d1, d2, d3;
            e4m3x4_to_bf16(x, d0, d1), e4m3x4_to_bf16(y, d2, d3);
            const u32x4 d = {d0, d1, d2, d3};
            return __builtin_bit_cast(bf16x8, d);
        };
        // Which of the wave's 32 tokens of a tile the lane's row sees, a bit a token.
        auto seen_of = [&](int i, int buf) -> uint32_t {
            const uint32_t is_there = (uint32_t)__builtin_amdgcn_ballot_w64(__float_as_uint(sh->scale[buf][32 * th + n32]) != kTreeHole);
            const int t0 = (tile_lo + i) * kTreeTokens + 32 * th;
            if (t0 + 32 <= s.ctx) return is_there;
            const int j0 = t0 - s.ctx;                  // drafted row of bit 0
            const int most = (a.masks ? s.nodes : min(s.nodes, own_node + 1)) - j0;
            uint32_t bits = most >= 32 ? ~0u : most > 0 ? (1u << most) - 1u : 0u;
            if (a.masks) {
                const uint32_t* const mask = a.masks + (size_t)(s.node0 + own_node) * a.mask_words;
                const int w = j0 >> 5, shift = j0 & 31;  // (floors below zero)
                const uint32_t lo = w < 0 ? ~0u : w < a.mask_words ? mask[w] : 0u;
                const uint32_t hi = w + 1 < 0 ? ~0u : w + 1 < a.mask_words ? mask[w + 1] : 0u;
                bits &= (uint32_t)((((unsigned long long)hi << 32) | lo) >> shift);
            }
            return bits & is_there;
        };
        f32x16 sc;               // a tile's scores: of token 8 (r >> 2) + 4 half + (r & 3) in register r
        uint32_t seen = ~0u, seen_half = ~0u;  // (the second from the lane's first token on)
        auto bit_of = [&](int r) -> bool { return (int)(seen_half << (31 - 8 * (r >> 2) - (r & 3))) < 0; };
        const lds_ptr<uint8_t> w_row = weights + own * (2 * kTreeTokens) + 8 * half;
        const int w_swap = (own >> 1) & 7;
        lds_ptr<float> scale_row = (lds_ptr<float>)&sh->scale[0][32 * th + 4 * half];
        asm volatile("" : "+v"(scale_row));  // (one address: its part of the layout is past an instruction's offset)
        auto scales_of = [&](int buf, int i) -> f32x4 { return *(lds_ptr<f32x4>)(scale_row + buf * kTreeTokens + 8 * i); };
        u16x2 high = {0, 0};     // the largest of a tile's weights
        auto put_weights = [&](int i, const float (&p)[4]) {
            const uint32_t lo = pack_f16x2(p[0], p[1]), hi = pack_f16x2(p[2], p[3]);
            high = __builtin_elementwise_max(high, __builtin_elementwise_max(__builtin_bit_cast(u16x2, lo), __builtin_bit_cast(u16x2, hi)));
            *(lds_ptr<u32x2>)(w_row + 16 * ((4 * th + i) ^ w_swap)) = u32x2{lo, hi};
        };
        // A tile's weights out of its scores, a token at a time; l_sum and the largest exponent go along. As if every row saw every token.
        f32x4 by;
        float mu = 0.0f, p[4];
        auto weigh_begin = [&](int buf) {
            mu = m_ref == -INFINITY ? 0.0f : m_ref, high.x = m_ref == -INFINITY ? kTreeGrown : (uint16_t)0, high.y = 0, l_before = l_sum;
            by = scales_of(buf, 0);
        };
        auto weigh = [&](int buf, int r) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], by[r & 3], -mu));
            l_sum += e;
            asm volatile("" : "+v"(l_sum));  // (here, under the matrix instructions, though weigh_seen() may replace it)
            p[r & 3] = e * by[r & 3];
            if ((r & 3) == 3) {
                put_weights(r >> 2, p);
                if (r < 15) by = scales_of(buf, (r >> 2) + 1);
            }
        };
        // The same of a tile with tokens that some row does not see, in place of what weigh() made of it. Whether a score is no number: then some code of
        // the tile may be none, and its product with a weight of zero would be none either (clean).
        auto weigh_seen = [&](int buf) -> bool {
            l_sum = l_before, high.x = m_ref == -INFINITY ? kTreeGrown : (uint16_t)0, high.y = 0;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 s4 = scales_of(buf, i);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    nan |= sc[4 * i + k] != sc[4 * i + k];
                    const float x = bit_of(4 * i + k) ? __builtin_fmaf(sc[4 * i + k], s4[k], -mu) : -INFINITY;
                    const float e = __builtin_amdgcn_exp2f(x);
                    l_sum += e;
                    p[k] = bit_of(4 * i + k) ? e * s4[k] : 0.0f;
                }
                put_weights(i, p);
            }
            return __builtin_amdgcn_ballot_w64(nan) != 0;
        };
        // New references for the rows of a tile (the workgroup's decision), and a factor for what came before. (A scale counts as 2^(lift - 90) at least, so
        // that an exponential is 2^90 at most and the sum of 2^31 of them a number.)
        auto refer = [&](int buf) -> float {
            float top = -INFINITY;
            const float least = (float)(lift - 90);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 s4 = scales_of(buf, i);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    top = fmaxf(top, bit_of(4 * i + k) ? __builtin_fmaf(sc[4 * i + k], s4[k], fmaxf(__builtin_amdgcn_logf(fabsf(s4[k])), least)) : -INFINITY);
            }
            const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1]));
            if (half == 0) sh->top[th][own] = top;
            lds_barrier();
            top = fmaxf(sh->top[0][own], sh->top[1][own]) - (float)lift;
            const bool grow = top > m_ref;
            const float corr = grow ? __builtin_amdgcn_exp2f(m_ref - top) : 1.0f;  // 2^-inf = 0 at first
            if (grow) m_ref = top;
            mu = m_ref == -INFINITY ? 0.0f : m_ref;
            return corr;
        };
        auto regrow = [&](int buf) {
            const float corr = refer(buf);
            if (th == 0 && half == 0) sh->corr[own] = corr;
            l_before *= corr;
            weigh_seen(buf);
            lds_barrier();
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float f = sh->corr[32 * b + n32];
#pragma unroll
                for (int c = 0; c < 4; ++c) o[c][b] *= f;
            }
        };
        // ---- the first half of an iteration: S^T[token][row] of the wave's tokens of a tile over its half of the dims, x[0] of the rows that are the
        // wave's, x[1] of the others on their way to the other half's wave. A piece of codes is out of LDS two steps and
        // converted one step before its matrix instructions; the fences keep that order. With MORE the tile before is weighed and the next
        // but one asked for in between.
        f32x16 x[2];
        auto scores = [&](int buf, auto more, int before, int third) {
            constexpr bool MORE = decltype(more)::value;
            const lds_ptr<uint8_t> codes = tiles + buf * kTreeTileBytes;
            u32x4 k[3];
            auto load = [&](int i) {
                k[i % 3] = *(lds_ptr<u32x4>)(codes + (i < 8 ? k_row + 1024 * (i >> 2) + 16 * ((2 * (i & 3) + half) ^ k_swap) : k_rope));
            };
            load(0), load(1);
            if (MORE) {
                weigh_begin(before);
                find(0), find(1);
                weigh(before, 0), weigh(before, 1);
            }
            x[0] = f32x16{}, x[1] = f32x16{};
            bf16x8 lo = as_bf16(k[0].x, k[0].y), hi = as_bf16(k[0].z, k[0].w);
            each<8>([&](auto step) {
                constexpr int i = decltype(step)::value;
                __builtin_amdgcn_sched_barrier(0);
                if (i + 2 < 9) load(i + 2);
                const u32x4 then = k[(i + 1) % 3];
                x[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, __builtin_bit_cast(bf16x8, q[2 * i][0]), x[0], 0, 0, 0);
                if (MORE && i < 7) weigh(before, 2 + 2 * i);
                __builtin_amdgcn_sched_barrier(0);
                x[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, __builtin_bit_cast(bf16x8, q[2 * i][1]), x[1], 0, 0, 0);
                lo = as_bf16(then.x, then.y);
                if constexpr (MORE) bring(std::integral_constant<int, i>{}, third);
                __builtin_amdgcn_sched_barrier(0);
                x[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, __builtin_bit_cast(bf16x8, q[2 * i + 1][0]), x[0], 0, 0, 0);
                if (MORE && i < 7) weigh(before, 3 + 2 * i);
                __builtin_amdgcn_sched_barrier(0);
                x[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, __builtin_bit_cast(bf16x8, q[2 * i + 1][1]), x[1], 0, 0, 0);
                hi = as_bf16(then.z, then.w);
            });
            // (the last step: the rows that are sent first, so that they go out while the others are made)
            __builtin_amdgcn_sched_barrier(0);
            x[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, __builtin_bit_cast(bf16x8, q[16][1]), x[1], 0, 0, 0);
            if constexpr (MORE) bring(std::integral_constant<int, 8>{}, third);
            __builtin_amdgcn_sched_barrier(0);
            x[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, __builtin_bit_cast(bf16x8, q[17][1]), x[1], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            x[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, __builtin_bit_cast(bf16x8, q[16][0]), x[0], 0, 0, 0);
            if constexpr (MORE) go_on(0), go_on(1);
            __builtin_amdgcn_sched_barrier(0);
            x[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, __builtin_bit_cast(bf16x8, q[17][0]), x[0], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) sh->part[2 * th + 1 - kh][i][lane] = f32x4{x[1][4 * i], x[1][4 * i + 1], x[1][4 * i + 2], x[1][4 * i + 3]};
        };
        // ---- the second half: O^T[column][row] += V^T . P^T of a tile, sixteen units of a K-step and a column tile each. With NEXT the
        // partial scores of the next tile meet and the transfers asked for arrive in between. A unit's codes are out of LDS three units and
        // converted one unit before its matrix instructions. `check` comes once every weight is there, and says whether it changed the
        // tile's codes.
        auto values = [&](auto more, int buf, int third, int number_of, auto check) {
            constexpr bool NEXT = decltype(more)::value;
            const lds_ptr<uint8_t> codes = tiles + buf * kTreeTileBytes + v_row;
            const lds_ptr<uint8_t> w_from = weights + n32 * (2 * kTreeTokens);
            i32x2 raw[4];
            f16x8 w[2][2];
            auto load = [&](int u) {
                raw[u % 4] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_ptr<i32x2>)(codes + 8192 * (u >> 2) + 16 * ((v_piece + (u & 3)) ^ v_swap)));
            };
            auto load_w = [&](int ks) {
#pragma unroll
                for (int b = 0; b < 2; ++b) w[ks & 1][b] = *(lds_ptr<f16x8>)(w_from + 32 * b * (2 * kTreeTokens) + 16 * ((2 * ks + half) ^ k_swap));
            };
            load(0), load(1), load(2);
            lds_barrier();  // partial scores and weights are there
            const TreeFlags flags{sh->grown, sh->dirty, sh->holed[(number_of + 1) & 1]};
            load_w(0);
            f32x4 part[4];
            if (NEXT) {
#pragma unroll
                for (int i = 0; i < 4; ++i) part[i] = sh->part[2 * th + kh][i][lane];
            }
            if (__builtin_expect(check(flags), 0)) load(0), load(1), load(2), load_w(0);
            u32x4 v[2];
            auto convert = [&](int u, int side) {
                uint32_t lo, hi;
                e4m3x4_to_f16((uint32_t)raw[u % 4][side], lo, hi);
                v[u & 1][2 * side] = lo, v[u & 1][2 * side + 1] = hi;
            };
            convert(0, 0), convert(0, 1);
            each<16>([&](auto unit) {
                constexpr int u = decltype(unit)::value, ks = u >> 2, c = u & 3;
                __builtin_amdgcn_sched_barrier(0);
                if (u + 3 < 16) load(u + 3);
                if (c == 1 && ks < 3) load_w(ks + 1);
                o[c][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[u & 1]), w[ks & 1][0], o[c][0], 0, 0, 0);
                if (u < 15) convert(u + 1, 0);
                if (NEXT && u == 12) arrived(third);
                __builtin_amdgcn_sched_barrier(0);
                o[c][1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[u & 1]), w[ks & 1][1], o[c][1], 0, 0, 0);
                if (u < 15) convert(u + 1, 1);
                if (NEXT && u >= 2 && u < 10) {
                    constexpr int r = 2 * (u - 2) & 15;
                    float s0 = x[0][r] + part[r >> 2][r & 3], s1 = x[0][r + 1] + part[r >> 2][(r & 3) + 1];
                    asm volatile("" : "+v"(s0), "+v"(s1));  // (here, under the matrix instructions, though a later tile's)
                    sc[r] = s0, sc[r + 1] = s1;
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        };
        // A tile whose keys have all been read, the wave's sixteen rows of it: codes that are no number become zeros. A row that does see such a
        // token has no number for its weight.
        auto clean = [&](int buf) {
            const lds_ptr<uint8_t> to = tiles + buf * kTreeTileBytes + 2 * wave * 4096 + 16 * lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const u32x4 c = *(lds_ptr<u32x4>)(to + 1024 * i);
                const u32x4 d = {numbers_only(c.x), numbers_only(c.y), numbers_only(c.z), numbers_only(c.w)};
                *(lds_ptr<u32x4>)(to + 1024 * i) = d;
            }
            lds_barrier();
        };
        auto drafted = [&](int i) -> bool { return (tile_lo + i + 1) * kTreeTokens > s.ctx; };

#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int b = 0; b < 2; ++b) o[c][b] = f32x16{};
        // ---- the first tile, which sets the references -----------------------------------------------------------
        if (n_tiles > 1) ask(1);
        scores(0, std::false_type{}, 0, 0);
        seen = seen_of(0, 0), seen_half = seen >> 4 * half;
        bool masked = __builtin_amdgcn_ballot_w64(seen != ~0u) != 0;  // some row may not see some token of tile i
        lds_barrier();
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = x[0][r] + sh->part[2 * th + kh][r >> 2][lane][r & 3];
        refer(0);
        if (n_tiles > 1) arrived(1), fill_holes(1, number + 1);
        lds_barrier();
        int buf = 0;  // of tile i
        for (int i = 0; i + 1 < n_tiles; ++i) {
            const int next = buf == 2 ? 0 : buf + 1, third = next == 2 ? 0 : next + 1;
            scores(next, std::true_type{}, buf, third);
            if (__builtin_expect(masked, 0) && weigh_seen(buf)) sh->dirty = number + i;
            if (__builtin_amdgcn_ballot_w64(max(high.x, high.y) >= kTreeGrown) != 0) sh->grown = number + i;
            bool holed = false;
            values(std::true_type{}, buf, third, number + i, [&](const TreeFlags& f) {
                const bool dirty = __builtin_amdgcn_readfirstlane(f.dirty) == number + i, grown = __builtin_amdgcn_readfirstlane(f.grown) == number + i;
                holed = __builtin_amdgcn_readfirstlane(f.holed) == number + i + 1;
                if (__builtin_expect(dirty, 0)) clean(buf);
                if (__builtin_expect(grown, 0)) regrow(buf);
                return dirty || grown;
            });
            fill_holes(third, number + i + 2);
            masked = drafted(i + 1) || holed;
            seen = seen_half = ~0u;
            if (__builtin_expect(masked, 0)) {
                seen = seen_of(i + 1, next), seen_half = seen >> 4 * half;
            }
            lds_barrier();
            buf = next;
        }
        weigh_begin(buf);
        seen = seen_of(n_tiles - 1, buf), seen_half = seen >> 4 * half;
        if (weigh_seen(buf)) sh->dirty = number + n_tiles - 1;
        if (__builtin_amdgcn_ballot_w64(max(high.x, high.y) >= kTreeGrown) != 0) sh->grown = number + n_tiles - 1;
        values(std::false_type{}, buf, 0, number + n_tiles - 1, [&](const TreeFlags& f) {
            const bool dirty = __builtin_amdgcn_readfirstlane(f.dirty) == number + n_tiles - 1, grown = __builtin_amdgcn_readfirstlane(f.grown) == number + n_tiles - 1;
            if (dirty) clean(buf);
            if (grown) regrow(buf);
            return dirty || grown;
        });
        if (a.bad_rows && last_block && l8 == 0 && missing) atomicAdd(a.bad_rows, missing);
        number += n_tiles + 2;  // (two tiles past the end were asked for)
    }

    if (n_tiles <= 0) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int b = 0; b < 2; ++b) o[c][b] = f32x16{};
    }

    // ---- results: of column tile c a lane's registers 4 i .. are columns of piece c, or four pieces further on (i >= 2), from
    // 8 (i & 1) + 4 half on
    const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_sum), __float_as_uint(l_sum), false, false);
    l_sum = __uint_as_float(other[0]) + __uint_as_float(other[1]);
    if (half == 0) {
        sh->sum[th][own] = l_sum;
        if (th == 0) sh->ref[own] = m_ref;
    }
    lds_barrier();
    if (!whole) {
        if (n_tiles > 0) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
                if (kTreeRows * rb + 32 * b + n32 < rows) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) reinterpret_cast<f32x4*>(rec)[(((wave * 4 + c) * 2 + b) * 4 + i) * kWave + lane] =
                            f32x4{o[c][b][4 * i], o[c][b][4 * i + 1], o[c][b][4 * i + 2], o[c][b][4 * i + 3]};
                }
        }
        if (tid < kTreeRows) {
            rec[kTreeRows * 512 + 2 * tid] = sh->ref[tid];
            rec[kTreeRows * 512 + 2 * tid + 1] = sh->sum[0][tid] + sh->sum[1][tid];
        }
    } else {
        // through LDS, a row a store: the same places as the rows' operands had
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int row = 32 * b + n32, r = kTreeRows * rb + row;
            const float l = sh->sum[0][row] + sh->sum[1][row];
            const float inv = l == 0.0f ? 0.0f : 1.0f / (l * a.qscale);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *(lds_ptr<u32x2>)(tiles + 1024 * row + 16 * ((16 * wave + c * 2 + 8 * (i >> 1) + (i & 1)) ^ (row & 15)) + 8 * half) =
                        u32x2{pack_bf16x2(o[c][b][4 * i] * inv, o[c][b][4 * i + 1] * inv), pack_bf16x2(o[c][b][4 * i + 2] * inv, o[c][b][4 * i + 3] * inv)};
            if (a.lse && wave == 0 && half == 0 && r < rows)
                a.lse[(size_t)s.node0 * a.H + r] = l == 0.0f ? -INFINITY : (sh->ref[row] + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
        }
        lds_barrier();
        const int first = kTreeRows * rb + 16 * wave;  // the wave's
        uint8_t* const out = reinterpret_cast<uint8_t*>(a.clat) + ((size_t)s.node0 * a.H + first) * 1024;
        const lds_ptr<uint8_t> from = tiles + 1024 * 16 * wave;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            u32x4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *(lds_ptr<u32x4>)(from + 1024 * (i + k) + 16 * (lane ^ (i + k)));
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (first + i + k < rows) *reinterpret_cast<u32x4*>(out + (1024u * (unsigned)(i + k) + 16u * (unsigned)lane)) = v[k];
        }
    }
    lds_barrier();
}

// RUNS: pages are whole runs of 16 rows, whose addresses are scalar. 32 sequences of 8 192 tokens, 8 nodes of 64 heads, in pages of 48 and 64 rows 269 us, of 4 and 60
// rows, by the form for any, 275; 64 nodes of 128 heads over 32 768 524 and 535.
template <bool RUNS>
__global__ __launch_bounds__(kTreeThreads, 1) void mla_attend_tree_kernel(const TreeArgs a) {
    __shared__ __attribute__((aligned(1024))) TreeShared shared;
    const lds_ptr<TreeShared> sh = (lds_ptr<TreeShared>)&shared;
    if (threadIdx.x == 0) sh->grown = sh->dirty = sh->holed[0] = sh->holed[1] = -1;
    const bool all = a.groups == 0;  // a block of rows is a work item
    unsigned item = blockIdx.x, u = item, end = u + 1, begin = 0;
    TreeWalk::Block b;
    {
        TreeWalk walk(a);
        if (!all) {
            const unsigned total = walk.total();
            begin = walk.begin;
            if (total == 0) return;
            const TreeItems items(a, total);
            if (item >= items.items) return;
            // an eighth of the items on each die: neighbours, which often read the same tokens
            if (items.items % kTreeDies == 0) item = (item % kTreeDies) * (items.items / kTreeDies) + item / kTreeDies;
            u = items.lo(item), end = items.lo(item + 1);
        }
        if (!walk.block(all, u, b)) return;
    }
    for (int number = 0;;) {
        const int lo = all ? 0 : max((int)(u - b.first_tile), 0), hi = all ? (int)b.tiles : min((int)b.tiles, (int)(end - b.first_tile));
        float* const rec = a.partial + (size_t)(2 * item + (lo == 0 ? 1 : 0)) * kTreeRecordFloats;
        if (hi > lo) tree_part<RUNS>(a, sh, b.s, b.seq, b.rb, b.rb == (int)b.blocks - 1, lo, hi, lo == 0 && hi == (int)b.tiles, rec, number);
        const unsigned next = all ? end : b.first_tile + b.tiles;
        if (next >= end || next <= u) return;  // (the second: prefix sums that are none, whose units pass 32 bits)
        u = next;
        TreeWalk walk(a);  // (looked up again: what it has would keep registers through the tiles)
        walk.begin = begin;
        if (!walk.block(false, u, b)) return;
    }
}

// Blocks that several work items had: their records, in order, under the largest reference. A workgroup's column of the launch has a block,
// or, where there are more blocks than work items (BY_ITEM), the block inside of which its work item begins, the first one of that
// block. Bound by memory's round trips where there are few: records go eight at a time, every load of a batch in front of the first use. 39 blocks of some 8 records
// 12 us, 3.2 TB/s; in an eighth of the workgroups with four pieces a thread, rows stored whole, 16.
template <bool BY_ITEM>
__global__ __launch_bounds__(256) void mla_attend_tree_merge_kernel(const TreeArgs a) {
    TreeWalk walk(a);
    const unsigned total = walk.total();
    if (total == 0) return;
    const TreeItems items(a, total);
    TreeWalk::Block block;
    unsigned g0;
    if (BY_ITEM) {
        const unsigned g = blockIdx.x + 1;
        if (g >= items.items) return;
        const unsigned u = items.lo(g);
        g0 = g - 1;
        if (!walk.block(false, u, block) || u <= block.first_tile || items.lo(g0) > block.first_tile) return;
    } else {
        if (!walk.block(true, blockIdx.x, block)) return;
        g0 = items.of(block.first_tile);
    }
    const unsigned g1 = items.of(block.first_tile + block.tiles - 1);
    if (g0 == g1) return;
    const int at = blockIdx.y * 256 + threadIdx.x, lane = at & 63, idx = at >> 6;
    const int i = idx & 3, b = (idx >> 2) & 1, c = (idx >> 3) & 3, wave = idx >> 5;
    const int row = 32 * b + (lane & 31), r = kTreeRows * block.rb + row;
    if (r >= block.s.nodes * a.H) return;
    float m = -INFINITY, l = 0.0f;
    f32x4 sum = {0, 0, 0, 0};
    constexpr int kBatch = 8;
    for (unsigned from = g0; from <= g1; from += kBatch) {
        f32x2 ml[kBatch];
        f32x4 v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {  // (a record past the last re-reads the last, and is left out)
            const unsigned rec_of = min(from + k, g1);
            const float* const rec = a.partial + (size_t)(2 * rec_of + (rec_of == g0 ? 1 : 0)) * kTreeRecordFloats;
            ml[k] = *reinterpret_cast<const f32x2*>(rec + kTreeRows * 512 + 2 * row);
            v[k] = reinterpret_cast<const f32x4*>(rec)[at];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) top = fmaxf(top, ml[k].x);
        if (top == -INFINITY) continue;         // nothing yet that the row sees
        const float keep = __builtin_amdgcn_exp2f(m - top);
        m = top, l *= keep, sum *= keep;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (from + k > g1 || ml[k].y == 0.0f) continue;
            const float by = __builtin_amdgcn_exp2f(ml[k].x - top);
            l += ml[k].y * by;
            sum += v[k] * by;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / (l * a.qscale);
    const size_t out = (size_t)block.s.node0 * a.H + r;
    *reinterpret_cast<u32x2*>(a.clat + out * 512 + 128 * wave + 16 * c + 64 * (i >> 1) + 8 * (i & 1) + 4 * (lane >> 5)) =
        u32x2{pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv)};
    if (a.lse && idx == 4 * b && lane < 32) a.lse[out] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

}  // namespace rk
