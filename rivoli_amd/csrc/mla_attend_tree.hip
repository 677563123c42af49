// Attention of a tree of drafted tokens over the paged latent cache: node i of a sequence attends its ctx cached rows
// and, of the drafted rows behind them, those its mask names. Launch-only.
#include <climits>
#include <cmath>
#include <type_traits>
#include <utility>

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
// Whether node `node` of `s` attends cached row `t`.
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, const TreeSeq& s, int node, int t) {
    const int j = t - s.ctx;
    if (j < 0) return true;
    if (j >= s.nodes) return false;
    if (!a.masks) return j <= node;
    return a.masks[(size_t)(s.node0 + node) * a.mask_words + (j >> 5)] >> (j & 31) & 1;
}

// The plain form, for any row width: a wave has one node's one head, 64 rows at a time; a lane a row's score, then
// a share of the columns.
constexpr int kTreeRowWaves = 4;
constexpr int kTreeMaxRow = 576;

__global__ __launch_bounds__(kTreeRowWaves* kWave) void mla_attend_tree_rowwise_kernel(const TreeArgs a) {
    __shared__ float q_smem[kTreeRowWaves][kTreeMaxRow];
    __shared__ float w_smem[kTreeRowWaves][kWave];
    __shared__ unsigned long long at_smem[kTreeRowWaves][kWave];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int node_all = blockIdx.x, head = blockIdx.y * kTreeRowWaves + wave;
    // the sequence: the last one that starts at or before the node
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu_nodes[mid] <= node_all) lo = mid;
        else hi = mid - 1;
    }
    const TreeSeq s = tree_seq(a, lo);
    const int node = node_all - s.node0;
    if (node < 0 || node >= s.nodes || head >= a.H) return;
    const size_t row = (size_t)node_all * a.H + head;
    float* const q = q_smem[wave];
    for (int i = lane; i < a.kvl; i += kWave) q[i] = bf16_lo_to_f32(a.qabs[row * a.kvl + i]);
    for (int i = lane; i < a.rope; i += kWave) q[a.kvl + i] = bf16_lo_to_f32(a.qrope[row * a.rope + i]);
    const int* const table = a.block_table + (size_t)lo * a.max_blocks;
    const int len = s.ctx + s.nodes;
    const bool counts = a.bad_rows && head == a.H - 1 && node == s.nodes - 1;
    float m = -INFINITY, l = 0.0f;  // l: the lane's own
    float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int t0 = 0; t0 < len; t0 += kWave) {
        const int t = t0 + lane;
        unsigned long long at = 0;
        float scale = 0.0f, x = -INFINITY;
        bool seen = false;
        if (t < len) {
            const int blk = t / a.page_tokens, off = t - blk * a.page_tokens;
            const int page = blk < a.max_blocks ? table[blk] : -1;
            if ((unsigned)page < (unsigned)a.n_pages) {
                at = (unsigned long long)page * a.page_bytes;
                scale = *reinterpret_cast<const float*>(a.pool + at + (size_t)a.page_tokens * a.row_w + 4ull * off);
                at += (unsigned long long)off * a.row_w;
                // a scale that is not a positive number cannot come from the append: left out like a row that is not there
                seen = scale > 0.0f && tree_sees(a, s, node, t);
            } else if (counts) {
                atomicAdd(a.bad_rows, 1u);
            }
        }
        if (seen) {
            float dot = 0.0f;
            for (int i = 0; i < a.row_w; i += 8) {
                const u32x2 c = *reinterpret_cast<const u32x2*>(a.pool + at + i);
                float v[4], w[4];
                e4m3x4_to_f32(c.x, v), e4m3x4_to_f32(c.y, w);
#pragma unroll
                for (int j = 0; j < 4; ++j) dot = __builtin_fmaf(q[i + j], v[j], dot);
#pragma unroll
                for (int j = 0; j < 4; ++j) dot = __builtin_fmaf(q[i + 4 + j], w[j], dot);
            }
            x = dot * scale * a.qscale;
        }
        const float top = fmaxf(m, wave_max(x));
        if (__builtin_amdgcn_ballot_w64(seen) == 0) continue;
        const float mu = top == -INFINITY ? 0.0f : top, keep = __builtin_amdgcn_exp2f(m - mu);
        m = top;
        const float e = seen ? __builtin_amdgcn_exp2f(x - mu) : 0.0f;
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= keep;
        w_smem[wave][lane] = seen ? e * scale : 0.0f, at_smem[wave][lane] = at;
        __builtin_amdgcn_wave_barrier();
        const int n = min(kWave, len - t0);
        unsigned long long live = __builtin_amdgcn_ballot_w64(seen);
        for (int j = 0; j < n; ++j) {
            if (!(live >> j & 1)) continue;
            const float w = w_smem[wave][j];
            const uint16_t* const codes = reinterpret_cast<const uint16_t*>(a.pool + at_smem[wave][j]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (128 * i < a.kvl) {
                    const f32x2 v = __builtin_amdgcn_cvt_pk_f32_fp8((uint32_t)codes[lane + 64 * i], false);
                    o[2 * i] = __builtin_fmaf(w, v.x, o[2 * i]), o[2 * i + 1] = __builtin_fmaf(w, v.y, o[2 * i + 1]);
                }
        }
        __builtin_amdgcn_wave_barrier();
    }
    for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, kWave);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // nothing attended: zeros
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (128 * i < a.kvl)
            reinterpret_cast<uint32_t*>(a.clat + row * a.kvl)[lane + 64 * i] = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
    if (a.lse && lane == 0) a.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

}  // namespace rk

#include "mla_attend_tree.hpp"

extern "C" size_t rivoli_mla_attend_tree_paged_scratch_floats(int n_seqs, int H, int n_nodes, int max_nodes, int max_ctx) {
    return rk::tree_scratch_floats(rk::tree_plan(n_seqs, H, n_nodes, max_nodes, max_ctx));
}

extern "C" int rivoli_mla_attend_tree_paged(const unsigned short* qabs, const unsigned short* qrope,
                                            const unsigned char* pool, const int* block_table, const int* ctx_lens,
                                            const int* cu_nodes, const unsigned int* masks, int n_seqs, int H,
                                            int n_nodes, int max_nodes, int max_ctx, int max_blocks_per_seq, int kvl,
                                            int rope, int page_tokens, int n_pages, float scale,
                                            unsigned short* clat, float* lse, float* partial, unsigned int* bad_rows,
                                            void* stream) {
    if (!qabs || !qrope || !pool || !block_table || !ctx_lens || !cu_nodes || !clat || n_seqs <= 0 || H <= 0 ||
        n_nodes <= 0 || max_nodes <= 0 || max_ctx < 0 || max_blocks_per_seq <= 0 || kvl <= 0 || rope <= 0 ||
        page_tokens <= 0 || n_pages <= 0)
        return 1001;
    if (n_seqs > 65535 || max_nodes > 4096 || max_ctx > INT_MAX - 8192 || (long long)n_nodes * H > 1 << 30 || H > 65535 * rk::kTreeRowWaves ||
        page_tokens > 1 << 22)
        return 1002;
    if (kvl % 128 != 0 || kvl > 512 || rope % 8 != 0 || rope > 64 || page_tokens % 4 != 0) return 1004;
    if (!rk::aligned16(qabs) || !rk::aligned16(qrope) || !rk::aligned16(pool) || !rk::aligned16(clat) || !rk::aligned16(partial)) return 1004;
    const bool plain = kvl != 512 || rope != 64;
    const rk::TreePlan plan = rk::tree_plan(n_seqs, H, n_nodes, max_nodes, max_ctx);
    if (!plain && plan.groups && !partial) return 1001;
    const long long grid = plain ? n_nodes : plan.groups ? plan.groups : plan.blocks;
    if (grid * rk::kTreeThreads > (long long)rk::kLaunchThreads) return 1002;
    float qscale = scale * rk::kLog2e;
    if (std::fabs(qscale) < 1e-20f) qscale = std::copysign(1e-20f, qscale);  // as good as nothing to any softmax
    const rk::TreeArgs a{qabs, qrope, pool, block_table, ctx_lens, cu_nodes, masks, n_seqs, H, n_nodes, max_nodes, (max_nodes + 31) / 32,
                         max_ctx, max_blocks_per_seq, kvl, rope, kvl + rope, page_tokens, n_pages,
                         (size_t)page_tokens * (size_t)(kvl + rope + 4), qscale, clat, lse, plan.groups, partial, bad_rows};
    const hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();
    if (plain) {
        rk::launch_kernel(rk::mla_attend_tree_rowwise_kernel, dim3((unsigned)grid, (unsigned)((H + rk::kTreeRowWaves - 1) / rk::kTreeRowWaves)),
                          dim3(rk::kTreeRowWaves * rk::kWave), 0, st, a);
        return rk::launch_status();
    }
    rk::launch_kernel(page_tokens % 16 == 0 ? rk::mla_attend_tree_kernel<true> : rk::mla_attend_tree_kernel<false>, dim3((unsigned)grid), dim3(rk::kTreeThreads), 0, st, a);
    const int rc = rk::launch_status();
    if (rc != 0 || plan.groups < 2) return rc;
    if (plan.blocks < plan.groups) rk::launch_kernel(rk::mla_attend_tree_merge_kernel<false>, dim3((unsigned)plan.blocks, 32), dim3(256), 0, st, a);
    else rk::launch_kernel(rk::mla_attend_tree_merge_kernel<true>, dim3((unsigned)plan.groups - 1, 32), dim3(256), 0, st, a);
    return rk::launch_status();
}
