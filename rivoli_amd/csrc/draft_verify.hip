// Which drafted tokens stand, decided by the target's probabilities and given random numbers, and the token that
// follows them. Launch-only.
//
// A sequence's nodes are a tree in index order (a node's parent comes before it), node 0 the last token that is certain. From
// there: cur = 0, and for cur's children in index order, with w_0 = the target's row after cur, c_0 = 1 and q the draft's row
// after cur, child i of token x is accepted when u_i q(x) c_k < w_k(x); cur becomes i. A rejection leaves
//     w_{k+1} = max(w_k - c_k q, 0),   c_{k+1} = sum of w_{k+1},
// the residual that makes the accepted or drawn token the target's own, here without its division: w_k / c_k is the
// normalised row. Where drafts were picked and not drawn q is one at x: w_{k+1} is w_k without x, c_{k+1} = c_k - w_k(x), no sum needed.
// Past the last child the next token is drawn from w: the first v whose running sum exceeds u_final times the whole.
// All of it in 64 bits from the given f32 or bf16 values, so that a decision does not depend on the order of a sum: over 131 072 tokens the
// orders differ by some 10^-16 of the whole where two tokens' borders are 10^-5 apart; in f32 a draw in a thousand would move.
#include <cfloat>

#include "codec.hpp"

namespace rk {

//
// What bounds it. The walk is a chain of short steps in LDS by one wave, some 7 us with the launch and the nodes' scattered loads; a row's sum reads it once,
// and a rejected draft whose sibling is still to be judged reads target and draft rows once more, by the sequence's own workgroup: 131 072 tokens
// of f32 and a draft are 1 MB, some 16 us for a compute unit, as much its conversions and sums in 64 bits as its loads. 256 sequences of 8 drawn nodes
// of that size take 98 us where one read of two rows each is 54, the rest being second and third siblings; 32 of 16 picked nodes 11 us; one of 4 over 32 001 tokens 8.2.
// A wave's loads of a block are all on their way before the first is used, and picked tokens that were rejected are looked for once a block:
// testing each weight against each of them took 28 us where one launch now takes 16.
constexpr int kVerifyThreads = 1024, kVerifyWaves = kVerifyThreads / kWave;
constexpr int kVerifyNodes = 1024;             // of a sequence, held in LDS
constexpr int kVerifyChunk = 8 * kWave;        // tokens a wave's loads bring at once: eight a lane
constexpr int kVerifyChunks = 2;               // of a block: four of them spill in a workgroup of 16 waves, and are no faster
constexpr int kVerifyBlock = kVerifyChunks * kVerifyChunk;
constexpr int kVerifyBlocks = 2048;            // block sums in LDS: up to 2^21 tokens
// Calls of few sequences and long rows have the last pass over a row, the only one that most have, by many workgroups, and the draw in a launch of its
// own. Picked drafts' walk takes no sums, so that every workgroup makes it for itself: two launches. In us, in one launch and in two: 1 sequence of 131 072
// bf16 tokens 15.6 and 9.3, 32 of them 16.0 and 9.9, 64 16.3 and 14.6, 128 16.9 and 21.3; 64 of 65 536 11.4 and 10.1, 32 of 32 768 9.3 and 9.5. Drawn drafts have the
// walk in front in a launch of its own, three launches, of f32 tokens: 1 sequence of 49 152 8.1 and 9.6, of 65 536 9.0 and 9.5, of 98 304 11.1 and 10.0, of 131 072 12.7 and 10.0; 16 of
// 49 152 37.1 and 37.6, of 65 536 20.6 and 18.5, of 98 304 40.4 and 33.8; 32 of 131 072 50.8 and 42.4; 48 of 98 304 41.2 and 37.3, 64 of 49 152 24.7 and 24.7, of 131 072 43.9 and 47.6 (what
// is judged on the way, the same in both, makes most of these times).
constexpr int kVerifySplitSeqs = 32, kVerifySplitVocab = 98304;
constexpr int kPickedSplitSeqs = 64, kPickedSplitVocab = 49152;
constexpr int kVerifySumThreads = 256, kVerifySumBlocks = 4;  // a workgroup of the split form: a block a wave

struct VerifyArgs {
    const void *target, *draft;
    const int *tokens, *parents, *cu;
    const float *u, *u_final;
    int n_nodes, max_nodes, vocab;
    long long target_stride, draft_stride;  // in elements
    int *path, *n_path, *next;
    // the split form's, by sequence: the walk's end (node and rejections), its levels and rejected tokens, the blocks' sums
    int* end;
    double* levels;
    int* gone;
    double* sums;
    unsigned int* bad;
};

// A probability as it counts: what is no number, or negative, as zero, infinity as the largest. (The median of three with a quiet NaN among
// them is the least of the others; a signalling one it would pass on.)
__device__ __forceinline__ float counted(float x) { return __builtin_amdgcn_fmed3f(__builtin_canonicalizef(x), 0.0f, FLT_MAX); }

template <bool BF16>
__device__ __forceinline__ float prob(const void* rows, long long at) {
    if constexpr (BF16) return counted(__uint_as_float((uint32_t) static_cast<const uint16_t*>(rows)[at] << 16));
    else return counted(static_cast<const float*>(rows)[at]);
}
// Eight of a row from `at`, as loaded, and as they count. A row starts where its stride puts it: on an element.
template <bool BF16>
struct Eight;
template <>
struct Eight<true> {
    u32x4 v;
    __device__ __forceinline__ void load(const void* rows, long long at) {
        typedef u32x4 words __attribute__((aligned(2)));
        v = *reinterpret_cast<const words*>(static_cast<const uint16_t*>(rows) + at);
    }
    __device__ __forceinline__ float operator[](int i) const { return counted(i & 1 ? bf16_hi_to_f32(v[i >> 1]) : bf16_lo_to_f32(v[i >> 1])); }
};
template <>
struct Eight<false> {
    typedef float f32x4v __attribute__((ext_vector_type(4)));
    f32x4v lo, hi;
    __device__ __forceinline__ void load(const void* rows, long long at) {
        typedef f32x4v words __attribute__((aligned(4)));
        const words* const src = reinterpret_cast<const words*>(static_cast<const float*>(rows) + at);
        lo = src[0], hi = src[1];
    }
    __device__ __forceinline__ float operator[](int i) const { return counted(i < 4 ? lo[i] : hi[i - 4]); }
};

// The same with `left` tokens from there on, of which some may not be (they count as zero).
template <bool BF16>
__device__ __forceinline__ void load_some(Eight<BF16>& x, const void* rows, long long at, int left) {
    x = Eight<BF16>{};
    if (left >= 8) {
        x.load(rows, at);
    } else if (left > 0) {
        for (int i = 0; i < left; ++i) {
            if constexpr (BF16) {
                const uint32_t v = static_cast<const uint16_t*>(rows)[at + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) x.v[j] |= j == i >> 1 ? v << (16 * (i & 1)) : 0u;
            } else {
                const float v = static_cast<const float*>(rows)[at + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) x.lo[j] = j == i ? v : x.lo[j], x.hi[j] = j + 4 == i ? v : x.hi[j];
            }
        }
    }
}

// Sum over the lanes before, and over all of them.
__device__ __forceinline__ double lanes_before(double x, double& total) {
    double sum = x;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const double y = __shfl_up(sum, off, kWave);
        if ((int)(threadIdx.x & 63) >= off) sum += y;
    }
    total = __shfl(sum, kWave - 1, kWave);
    return sum - x;
}
// The same over all of them alone, by rotations within sixteen lanes and swaps of those rows: no trip through LDS, which a shuffle is.
template <int CTRL>
__device__ __forceinline__ double rotated(double x) {
    const long long v = __builtin_bit_cast(long long, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true), hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(v >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double lanes_sum(double x) {
    x += rotated<0x128>(x), x += rotated<0x124>(x), x += rotated<0x122>(x), x += rotated<0x121>(x);
    const auto both = [](uint32_t lo, uint32_t hi) -> double { return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo); };
    unsigned long long v = __builtin_bit_cast(unsigned long long, x);
    auto l = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
    x = both(l[0], h[0]) + both(l[1], h[1]);
    v = __builtin_bit_cast(unsigned long long, x);
    l = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    h = __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
    return both(l[0], h[0]) + both(l[1], h[1]);
}

// A node's row after k rejections.
template <bool BF16>
struct Row {
    const VerifyArgs& a;
    long long p_at, q_at;
    int k;
    const double* level;  // in LDS, as is gone
    const int* gone;
    __device__ __forceinline__ Row(const VerifyArgs& args, int node, int rejections, const double* levels, const int* tokens)
        : a(args), p_at(node * args.target_stride), q_at(node * args.draft_stride), k(rejections), level(levels), gone(tokens) {}
    static __device__ __forceinline__ double eights(const double (&w)[8]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); }
    // Calls f(first token, weights of eight) for this lane's part of each of block b's chunks, whose loads are on their way before the first is used.
    template <class F>
    __device__ __forceinline__ void chunks(int b, F f) const {
        const int v = b * kVerifyBlock + 8 * (int)(threadIdx.x & 63);
        const bool drafted = a.draft && k > 0;
        bool less = false;  // whether picked tokens that were rejected lie here: they are few
        if (!a.draft) {
            for (int j = 0; j < k; j += kWave)
                less |= __builtin_amdgcn_ballot_w64((unsigned)(gone[min(j + (int)(threadIdx.x & 63), k - 1)] - b * kVerifyBlock) < (unsigned)kVerifyBlock) != 0;
        }
        Eight<BF16> p[kVerifyChunks], q[kVerifyChunks];
        if ((b + 1) * kVerifyBlock <= a.vocab) {
#pragma unroll
            for (int c = 0; c < kVerifyChunks; ++c) p[c].load(a.target, p_at + v + c * kVerifyChunk);
            if (drafted) {
#pragma unroll
                for (int c = 0; c < kVerifyChunks; ++c) q[c].load(a.draft, q_at + v + c * kVerifyChunk);
            }
        } else {
#pragma unroll
            for (int c = 0; c < kVerifyChunks; ++c) load_some<BF16>(p[c], a.target, p_at + v + c * kVerifyChunk, a.vocab - v - c * kVerifyChunk);
            if (drafted) {
#pragma unroll
                for (int c = 0; c < kVerifyChunks; ++c) load_some<BF16>(q[c], a.draft, q_at + v + c * kVerifyChunk, a.vocab - v - c * kVerifyChunk);
            }
        }
        double w[kVerifyChunks][8];
#pragma unroll
        for (int i = 0; i < 8 * kVerifyChunks; ++i) w[i / 8][i % 8] = (double)p[i / 8][i % 8];
        if (drafted) {
            for (int j = 0; j < k; ++j) {
                const double c = level[j];
#pragma unroll
                for (int i = 0; i < 8 * kVerifyChunks; ++i) w[i / 8][i % 8] = fmax(w[i / 8][i % 8] - c * (double)q[i / 8][i % 8], 0.0);
            }
        } else if (less) {
            for (int j = 0; j < k; ++j) {
                const int x = gone[j] - v;
#pragma unroll
                for (int i = 0; i < 8 * kVerifyChunks; ++i) w[i / 8][i % 8] = x == i / 8 * kVerifyChunk + i % 8 ? 0.0 : w[i / 8][i % 8];
            }
        }
#pragma unroll
        for (int c = 0; c < kVerifyChunks; ++c) f(v + c * kVerifyChunk, w[c]);
    }
    // The sum of block b, by a wave.
    __device__ __forceinline__ double block(int b) const {
        double sum = 0.0;
        chunks(b, [&](int, const double(&w)[8]) { sum += eights(w); });
        return lanes_sum(sum);
    }
};

// The sums of every block of a row by a workgroup, and of all of them.
template <class R>
__device__ __forceinline__ void sum_row(const R& row, int blocks, double* sums, double* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = wave; b < blocks; b += kVerifyWaves) {
        const double s = row.block(b);
        if (lane == 0) sums[b] = s;
    }
    __syncthreads();
    if (wave == 0) {
        double s = 0.0;
        for (int b = lane; b < blocks; b += kWave) s += sums[b];
        s = lanes_sum(s);
        if (lane == 0) *all = s;
    }
    __syncthreads();
}

// The first token whose running sum is past `goal`, by a wave, from the blocks' sums, some of which is positive.
template <class R>
__device__ __forceinline__ int drawn(const R& row, int blocks, const double* sums, double goal) {
    const int lane = threadIdx.x & 63;
    // the block: a lane has `each` of them in a row
    const int each = (blocks + kWave - 1) / kWave;
    double mine = 0.0, total;
    int some = -1;  // the lane's last block with anything in it
    for (int i = 0; i < each; ++i) {
        const int b = lane * each + i;
        if (b < blocks && sums[b] > 0.0) mine += sums[b], some = b;
    }
    double run = lanes_before(mine, total);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(run + mine > goal && some >= 0);
    const unsigned long long any = __builtin_amdgcn_ballot_w64(some >= 0);
    const int holder = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
    run = __shfl(run, holder, kWave), some = __shfl(some, holder, kWave);
    int block = holder * each;
    for (; block < some; ++block) {
        if (sums[block] > 0.0 && run + sums[block] > goal) break;
        run += sums[block];
    }
    // and in it: the first past the goal, or the last with anything in it where the sums' roundings leave none
    int answer = -1, found = -1;
    row.chunks(block, [&](int v, const double(&w)[8]) {
        double upto = run + lanes_before(R::eights(w), total);
        int first = -1, held = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            upto += w[i];
            if (w[i] > 0.0) {
                held = v + i;
                if (first < 0 && upto > goal) first = v + i;
            }
        }
        const unsigned long long past = __builtin_amdgcn_ballot_w64(first >= 0), left = __builtin_amdgcn_ballot_w64(held >= 0);
        if (left) answer = __shfl(held, 63 - __builtin_clzll(left), kWave);
        if (past && found < 0) found = __shfl(first, __builtin_ctzll(past), kWave);
        run += total;
    });
    return found >= 0 ? found : answer;
}

// The walk of a sequence's tree, a workgroup each, and the next token (kWhole); of the split forms the walk alone (kWalk), or (kPicked) the walk of picked
// drafts, which takes no sums, by every workgroup of a sequence, and then the sums of the blocks that are the workgroup's, a wave each.
enum VerifyForm { kWhole, kWalk, kPicked };
template <bool BF16, VerifyForm FORM>
__global__ __launch_bounds__(FORM == kPicked ? kVerifySumThreads : kVerifyThreads) void draft_verify_kernel(const VerifyArgs a) {
    constexpr int kThreads = FORM == kPicked ? kVerifySumThreads : kVerifyThreads;
    const bool drawn_drafts = FORM != kPicked && a.draft;
    const bool writes = FORM != kPicked || blockIdx.x == 0;
    __shared__ int parent[kVerifyNodes], token[kVerifyNodes], gone[kVerifyNodes];  // gone: tokens rejected at cur
    __shared__ float share[kVerifyNodes], p_of[kVerifyNodes], q_of[kVerifyNodes];
    __shared__ double level[kVerifyNodes];  // c_0 .. c_k at cur
    __shared__ double sums[kVerifyBlocks];
    __shared__ int state[3];
    __shared__ double all;
    const int seq = FORM == kPicked ? blockIdx.y : blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int node0 = min(max(a.cu[seq], 0), a.n_nodes);
    const int n = min(max(a.cu[seq + 1] - node0, 0), min(a.max_nodes, a.n_nodes - node0));
    int* const path = a.path + (size_t)seq * a.max_nodes;
    if (n == 0) {
        if (!writes) return;
        for (int i = tid; i < a.max_nodes; i += kThreads) path[i] = -1;
        if (tid == 0) a.n_path[seq] = 0, a.next[seq] = -1;
        if (FORM != kWhole && tid == 0) a.end[2 * seq] = -1;
        return;
    }
    for (int i = tid; i < n; i += kThreads) {
        int up = i > 0 ? a.parents[node0 + i] : -1;
        const int x = a.tokens[node0 + i];
        if (i > 0 && !((unsigned)up < (unsigned)i && (unsigned)x < (unsigned)a.vocab)) {
            up = -1;  // no node's child
            if (a.bad && writes) atomicAdd(a.bad, 1u);
        }
        parent[i] = up, token[i] = x, share[i] = a.u[node0 + i];
        const bool there = up >= 0;
        p_of[i] = there ? prob<BF16>(a.target, (long long)(node0 + up) * a.target_stride + x) : 0.0f;
        q_of[i] = there && drawn_drafts ? prob<BF16>(a.draft, (long long)(node0 + up) * a.draft_stride + x) : 1.0f;
    }
    const int blocks = (a.vocab + kVerifyBlock - 1) / kVerifyBlock;

    // ---- the walk: wave 0 goes on until it is done or needs the sum of a residual ------------------------------
    auto child_after = [&](int cur, int last) -> int {
        for (int b = last + 1; b < n; b += kWave) {
            const unsigned long long m = __builtin_amdgcn_ballot_w64(b + lane < n && parent[min(b + lane, n - 1)] == cur);
            if (m) return b + __builtin_ctzll(m);
        }
        return -1;
    };
    int cur = 0, last = 0, k = 0, count = 1;
    if (tid == 0 && writes) path[0] = 0;
    if (tid == 0) level[0] = 1.0;
    __syncthreads();
    for (;;) {
        if (wave == 0) {
            int need = 0;
            for (;;) {
                const int child = child_after(cur, last);
                if (child < 0) break;
                last = child;
                const int x = token[child];
                const double c = level[k], q = (double)q_of[child];
                double w = (double)p_of[child];
                if (drawn_drafts) {
                    for (int j = 0; j < k; ++j) w = fmax(w - level[j] * q, 0.0);
                } else {
                    for (int j = 0; j < k; j += kWave)
                        if (__builtin_amdgcn_ballot_w64(j + lane < k && gone[min(j + lane, k - 1)] == x)) w = 0.0;
                }
                if ((double)share[child] * q * c < w) {
                    cur = child, k = 0;
                    if (lane == 0 && writes) path[count] = child;
                    ++count;
                    continue;
                }
                if (lane == 0) gone[k] = x;
                if (lane == 0 && !drawn_drafts && k + 1 < kVerifyNodes) level[k + 1] = c - w;
                __builtin_amdgcn_wave_barrier();
                ++k;
                if (drawn_drafts && child_after(cur, last) >= 0) {  // (the sum is for a sibling's test)
                    need = 1;
                    break;
                }
            }
            if (lane == 0) state[0] = cur, state[1] = k, state[2] = need;
        }
        __syncthreads();
        const int at = state[0], after = state[1], need = state[2];
        if (FORM == kPicked || !need) break;
        sum_row(Row<BF16>(a, node0 + at, after, level, gone), blocks, sums, &all);
        if (tid == 0) level[after] = all;
        __syncthreads();
    }
    cur = state[0], k = state[1];
    if (wave == 0 && writes) {
        for (int i = count + lane; i < a.max_nodes; i += kWave) path[i] = -1;
        if (lane == 0) a.n_path[seq] = count;
    }
    if (FORM != kWhole) {
        if (tid == 0 && writes) a.end[2 * seq] = node0 + cur, a.end[2 * seq + 1] = k;
        if (writes)
            for (int j = tid; j < k; j += kThreads) {
                a.levels[(size_t)seq * a.max_nodes + j] = drawn_drafts ? level[j] : 0.0;
                a.gone[(size_t)seq * a.max_nodes + j] = gone[j];
            }
        if (FORM == kPicked) {
            const int b = blockIdx.x * kVerifySumBlocks + wave;
            if (b >= blocks) return;
            const double s = Row<BF16>(a, node0 + cur, k, level, gone).block(b);
            if (lane == 0) a.sums[(size_t)seq * blocks + b] = s;
        }
        return;
    }
    sum_row(Row<BF16>(a, node0 + cur, k, level, gone), blocks, sums, &all);
    if (!(all > 0.0) && k > 0) {  // nothing is left of it: the node's own row
        k = 0;
        __syncthreads();
        sum_row(Row<BF16>(a, node0 + cur, 0, level, gone), blocks, sums, &all);
    }
    if (wave != 0) return;
    const int next = all > 0.0 ? drawn(Row<BF16>(a, node0 + cur, k, level, gone), blocks, sums, (double)a.u_final[seq] * all) : -1;
    if (lane == 0) a.next[seq] = next;
}

// The split form's second launch after kWalk, a wave a block of the row that a sequence's walk ended with; and the last one, which draws from their sums.
template <bool BF16>
__global__ __launch_bounds__(kVerifySumThreads) void draft_sums_kernel(const VerifyArgs a) {
    __shared__ double level[kVerifyNodes];
    __shared__ int gone[kVerifyNodes];
    const int seq = blockIdx.y, node = a.end[2 * seq], k = a.end[2 * seq + 1];
    if (node < 0) return;
    for (int j = threadIdx.x; j < k; j += kVerifySumThreads)
        level[j] = a.levels[(size_t)seq * a.max_nodes + j], gone[j] = a.gone[(size_t)seq * a.max_nodes + j];
    __syncthreads();
    const int blocks = (a.vocab + kVerifyBlock - 1) / kVerifyBlock, b = blockIdx.x * kVerifySumBlocks + (int)(threadIdx.x >> 6);
    if (b >= blocks) return;
    const double s = Row<BF16>(a, node, k, level, gone).block(b);
    if ((threadIdx.x & 63) == 0) a.sums[(size_t)seq * blocks + b] = s;
}

template <bool BF16>
__global__ __launch_bounds__(kVerifyThreads) void draft_draw_kernel(const VerifyArgs a) {
    __shared__ double level[kVerifyNodes];
    __shared__ int gone[kVerifyNodes];
    __shared__ double sums[kVerifyBlocks];
    __shared__ double all;
    const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, node = a.end[2 * seq];
    int k = a.end[2 * seq + 1];
    if (node < 0) return;
    const int blocks = (a.vocab + kVerifyBlock - 1) / kVerifyBlock;
    for (int j = threadIdx.x; j < k; j += kVerifyThreads)
        level[j] = a.levels[(size_t)seq * a.max_nodes + j], gone[j] = a.gone[(size_t)seq * a.max_nodes + j];
    for (int b = threadIdx.x; b < blocks; b += kVerifyThreads) sums[b] = a.sums[(size_t)seq * blocks + b];
    __syncthreads();
    if (wave == 0) {
        double s = 0.0;
        for (int b = lane; b < blocks; b += kWave) s += sums[b];
        s = lanes_sum(s);
        if (lane == 0) all = s;
    }
    __syncthreads();
    if (!(all > 0.0) && k > 0) {
        k = 0;
        __syncthreads();
        sum_row(Row<BF16>(a, node, 0, level, gone), blocks, sums, &all);
    }
    if (wave != 0) return;
    const int next = all > 0.0 ? drawn(Row<BF16>(a, node, k, level, gone), blocks, sums, (double)a.u_final[seq] * all) : -1;
    if (lane == 0) a.next[seq] = next;
}

// Whether a call of picked or drawn drafts takes a split form, and the pieces of its workspace (from 16-byte boundaries on).
struct VerifySplit {
    bool picked, drawn;
    size_t levels, sums, gone, end, bytes;
};
static VerifySplit verify_split(int n_seqs, int max_nodes, int vocab) {
    const bool some = n_seqs > 0 && max_nodes > 0;
    VerifySplit s{some && n_seqs <= kPickedSplitSeqs && vocab >= kPickedSplitVocab, some && n_seqs <= kVerifySplitSeqs && vocab >= kVerifySplitVocab,
                  0, 0, 0, 0, 0};
    if (!s.picked && !s.drawn) return s;
    const size_t blocks = ((size_t)vocab + kVerifyBlock - 1) / kVerifyBlock, n = (size_t)n_seqs;
    s.sums = n * max_nodes * 8;
    s.gone = s.sums + n * blocks * 8;
    s.end = s.gone + n * max_nodes * 4;
    s.bytes = (s.end + n * 8 + 15) / 16 * 16;
    return s;
}

template <bool BF16>
static int draft_verify(const VerifyArgs& a, bool split, int n_seqs, hipStream_t st) {
    (void)hipGetLastError();
    const dim3 grid((unsigned)n_seqs), block(kVerifyThreads);
    if (!split) {
        launch_kernel(draft_verify_kernel<BF16, kWhole>, grid, block, 0, st, a);
        return launch_status();
    }
    const unsigned blocks = (unsigned)((a.vocab + kVerifyBlock - 1) / kVerifyBlock);
    const dim3 shares((blocks + kVerifySumBlocks - 1) / kVerifySumBlocks, (unsigned)n_seqs), some(kVerifySumThreads);
    if (a.draft) {
        launch_kernel(draft_verify_kernel<BF16, kWalk>, grid, block, 0, st, a);
        launch_kernel(draft_sums_kernel<BF16>, shares, some, 0, st, a);
    } else {
        launch_kernel(draft_verify_kernel<BF16, kPicked>, shares, some, 0, st, a);
    }
    launch_kernel(draft_draw_kernel<BF16>, grid, block, 0, st, a);
    return launch_status();
}

}  // namespace rk

extern "C" size_t rivoli_draft_verify_workspace_bytes(int n_seqs, int max_nodes, int vocab) {
    return rk::verify_split(n_seqs, max_nodes, vocab).bytes;
}

extern "C" int rivoli_draft_verify(const void* target_probs, const void* draft_probs, const int* tokens,
                                   const int* parents, const int* cu_nodes, const float* uniforms,
                                   const float* final_uniforms, int n_seqs, int n_nodes, int max_nodes, int vocab,
                                   long long target_stride, long long draft_stride, int bf16, int* path, int* n_path,
                                   int* next_token, void* workspace, unsigned int* bad_nodes, void* stream) {
    if (!target_probs || !tokens || !parents || !cu_nodes || !uniforms || !final_uniforms || !path || !n_path ||
        !next_token || n_seqs <= 0 || n_nodes <= 0 || max_nodes <= 0 || vocab <= 0)
        return 1001;
    if (n_seqs > (int)(rk::kLaunchThreads / rk::kVerifyThreads) || max_nodes > rk::kVerifyNodes || vocab > rk::kVerifyBlocks * rk::kVerifyBlock || target_stride < vocab ||
        (draft_probs && draft_stride < vocab))
        return 1002;
    const rk::VerifySplit split = rk::verify_split(n_seqs, max_nodes, vocab);
    const bool shared = draft_probs ? split.drawn : split.picked;
    if (shared && !workspace) return 1001;
    const uintptr_t size = bf16 ? 2 : 4;
    if ((uintptr_t)target_probs % size != 0 || (uintptr_t)draft_probs % size != 0 || !rk::aligned16(workspace)) return 1004;
    unsigned char* const work = static_cast<unsigned char*>(workspace);
    const rk::VerifyArgs a{target_probs, draft_probs, tokens, parents, cu_nodes, uniforms, final_uniforms, n_nodes, max_nodes, vocab,
                           target_stride, draft_stride, path, n_path, next_token, reinterpret_cast<int*>(work + split.end),
                           reinterpret_cast<double*>(work + split.levels), reinterpret_cast<int*>(work + split.gone),
                           reinterpret_cast<double*>(work + split.sums), bad_nodes};
    return bf16 ? rk::draft_verify<true>(a, shared, n_seqs, (hipStream_t)stream) : rk::draft_verify<false>(a, shared, n_seqs, (hipStream_t)stream);
}
