// The rows of accepted drafts, moved to where the next step expects them: of a sequence with ctx cached rows and its
// drafted nodes behind them, row ctx + path[k] becomes row ctx + k. One launch for every layer. Launch-only.
//
// Bound by memory's round trip: a row is 580 bytes, a step keeps a handful of them in each layer. A wave has a sequence's
// rows of one layer and a 16-byte piece of them a lane, 16 rows in flight. In place without a copy:
// path[k] >= k, so what a batch reads lies behind everything that earlier batches wrote, and a batch has read all
// of its rows before it writes one (a lane's piece of a row is nobody else's). Entries that break the rule are left out.
// 6 rows of 64 sequences in each of 48 layers 5.9 us (18 MB at most, 3.6 us of a copy), 4 rows of one sequence 2.6.
#include "codec.hpp"

namespace rk {

struct CommitArgs {
    uint8_t* pool;
    const int *block_table, *ctx_lens, *path, *n_path;
    int max_path, max_blocks, page_tokens, n_pages;
    int row_bytes, scaled;  // scaled: a page's rows are followed by an f32 for each
    unsigned long long page_bytes;
    long long layer_bytes;
    int* new_lens;
    unsigned int* bad;
};
constexpr int kCommitRows = 16;

__global__ __launch_bounds__(64) void kv_commit_kernel(const CommitArgs a) {
    const int layer = blockIdx.x, seq = blockIdx.y, lane = threadIdx.x;
    const int ctx = max(a.ctx_lens[seq], 0), n = min(max(a.n_path[seq], 0), a.max_path);
    if (layer == 0 && lane == 0 && a.new_lens) a.new_lens[seq] = ctx + n;
    uint8_t* const pool = a.pool + layer * a.layer_bytes;
    const int* const table = a.block_table + (size_t)seq * a.max_blocks;
    const int* const path = a.path + (size_t)seq * a.max_path;
    const int pieces = a.row_bytes / 16;
    // byte offset of a row's page and its place in it; false: the table has no page for it
    auto find = [&](long long t, unsigned long long& page_at, unsigned int& off) -> bool {
        const unsigned long long blk = (unsigned long long)t / (unsigned)a.page_tokens;
        off = (unsigned int)((unsigned long long)t - blk * (unsigned)a.page_tokens);
        const int page = blk < (unsigned long long)a.max_blocks ? table[blk] : -1;
        page_at = (unsigned long long)(unsigned)page * a.page_bytes;
        return (unsigned)page < (unsigned)a.n_pages;
    };
    for (int k0 = 0; k0 < n; k0 += kCommitRows) {
        // lane k & 15 resolves row k
        const int k = k0 + (lane & (kCommitRows - 1));
        unsigned long long src = 0, dst = 0, src_scale = 0, dst_scale = 0;
        bool moves = false;
        if (k < n) {
            const int node = path[k];
            unsigned long long page_at;
            unsigned int off;
            if (node == k) {  // stays; looked up for the count alone
                if (a.bad && layer == 0 && lane < kCommitRows && !find((long long)ctx + k, page_at, off)) atomicAdd(a.bad, 1u);
            } else {
                bool ok = node > k && find((long long)ctx + node, page_at, off);
                src = page_at + (unsigned long long)off * (unsigned)a.row_bytes;
                src_scale = page_at + (unsigned long long)a.page_tokens * (unsigned)a.row_bytes + 4ull * off;
                ok = ok && find((long long)ctx + k, page_at, off);
                dst = page_at + (unsigned long long)off * (unsigned)a.row_bytes;
                dst_scale = page_at + (unsigned long long)a.page_tokens * (unsigned)a.row_bytes + 4ull * off;
                moves = ok;
                if (!ok && a.bad && layer == 0 && lane < kCommitRows) atomicAdd(a.bad, 1u);
            }
        }
        const unsigned int todo = (unsigned int)(__builtin_amdgcn_ballot_w64(moves) & 0xffffu);
        if (todo == 0) continue;
        float scale = 0.0f;
        const bool my_scale = a.scaled && moves && lane < kCommitRows;
        if (my_scale) scale = *reinterpret_cast<const float*>(pool + src_scale);
        auto row_of = [&](unsigned long long v, int r) -> unsigned long long {
            return ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), r) << 32) |
                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, r);
        };
        u32x4 row[kCommitRows];
#pragma unroll
        for (int r = 0; r < kCommitRows; ++r)
            if ((todo >> r & 1) && lane < pieces) row[r] = *reinterpret_cast<const u32x4*>(pool + row_of(src, r) + 16 * lane);
#pragma unroll
        for (int r = 0; r < kCommitRows; ++r)
            if ((todo >> r & 1) && lane < pieces) *reinterpret_cast<u32x4*>(pool + row_of(dst, r) + 16 * lane) = row[r];
        if (my_scale) *reinterpret_cast<float*>(pool + dst_scale) = scale;
    }
}

static int kv_commit(const CommitArgs& a, int n_seqs, int n_layers, hipStream_t st) {
    (void)hipGetLastError();
    launch_kernel(kv_commit_kernel, dim3((unsigned)n_layers, (unsigned)n_seqs), dim3(64), 0, st, a);
    return launch_status();
}

}  // namespace rk

extern "C" int rivoli_kv_commit_paged(unsigned char* pool, const int* block_table, const int* ctx_lens,
                                      const int* path, const int* n_path, int n_seqs, int max_path,
                                      int max_blocks_per_seq, int width, int page_tokens, int n_pages, int n_layers,
                                      long long layer_bytes, int* new_lens, unsigned int* bad_rows, void* stream) {
    if (!pool || !block_table || !ctx_lens || !path || !n_path || n_seqs <= 0 || max_path <= 0 ||
        max_blocks_per_seq <= 0 || width <= 0 || page_tokens <= 0 || n_pages <= 0 || n_layers <= 0)
        return 1001;
    if (new_lens == ctx_lens) return 1001;  // layers read it while the first one writes
    if (width > 1024 || n_seqs > 65535 || n_layers > 65535) return 1002;
    if (width % 16 != 0 || page_tokens % 4 != 0 || !rk::aligned16(pool) || (n_layers > 1 && layer_bytes % 16 != 0)) return 1004;
    const unsigned long long page_bytes = (unsigned long long)page_tokens * (unsigned)(width + 4);
    if (n_layers > 1 && (layer_bytes < 0 || (unsigned long long)layer_bytes / page_bytes < (unsigned)n_pages)) return 1002;
    const rk::CommitArgs a{pool, block_table, ctx_lens, path, n_path, max_path, max_blocks_per_seq, page_tokens, n_pages, width, 1,
                           page_bytes, layer_bytes, new_lens, bad_rows};
    return rk::kv_commit(a, n_seqs, n_layers, (hipStream_t)stream);
}

extern "C" int rivoli_index_commit_paged(unsigned short* kpool, const int* block_table, const int* ctx_lens,
                                         const int* path, const int* n_path, int n_seqs, int max_path,
                                         int max_blocks_per_seq, int hd, int page_tokens, int n_pages, int n_layers,
                                         long long layer_keys, int* new_lens, unsigned int* bad_rows, void* stream) {
    if (!kpool || !block_table || !ctx_lens || !path || !n_path || n_seqs <= 0 || max_path <= 0 ||
        max_blocks_per_seq <= 0 || hd <= 0 || page_tokens <= 0 || n_pages <= 0 || n_layers <= 0)
        return 1001;
    if (new_lens == ctx_lens) return 1001;
    if (hd > 512 || n_seqs > 65535 || n_layers > 65535) return 1002;
    if (hd % 8 != 0 || !rk::aligned16(kpool)) return 1004;
    if (n_layers > 1 && layer_keys < (long long)page_tokens * n_pages) return 1002;
    const rk::CommitArgs a{reinterpret_cast<unsigned char*>(kpool), block_table, ctx_lens, path, n_path, max_path, max_blocks_per_seq,
                           page_tokens, n_pages, 2 * hd, 0, (unsigned long long)page_tokens * (unsigned)(2 * hd),
                           n_layers > 1 ? layer_keys * 2 * hd : 0, new_lens, bad_rows};
    return rk::kv_commit(a, n_seqs, n_layers, (hipStream_t)stream);
}
