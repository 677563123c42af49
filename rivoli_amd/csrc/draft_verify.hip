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

constexpr int kVerifyThreads = 1024, kVerifyWaves = kVerifyThreads / kWave;
constexpr int kVerifyNodes = 1024;             // of a sequence, held in LDS
constexpr int kVerifyBlock = 8 * kWave;        // tokens of a block: eight a lane
constexpr int kVerifyBlocks = 4096;            // block sums in LDS: up to 2^21 tokens

struct VerifyArgs {
    const void *target, *draft;
    const int *tokens, *parents, *cu;
    const float *u, *u_final;
    int n_nodes, max_nodes, vocab;
    long long target_stride, draft_stride;  // in elements
    int *path, *n_path, *next;
    unsigned int* bad;
};

// A probability as it counts: what is no number, or negative, as zero.
__device__ __forceinline__ float counted(float x) { return x > 0.0f ? fminf(x, FLT_MAX) : 0.0f; }

template <bool BF16>
__device__ __forceinline__ float prob(const void* rows, long long at) {
    if constexpr (BF16) return counted(__uint_as_float((uint32_t) static_cast<const uint16_t*>(rows)[at] << 16));
    else return counted(static_cast<const float*>(rows)[at]);
}
// Eight of a row from `at`, of which `n` are there.
template <bool BF16>
__device__ __forceinline__ void prob8(const void* rows, long long at, int n, float (&p)[8]) {
    if (n >= 8) {  // (a row starts where its stride puts it: on an element)
        if constexpr (BF16) {
            typedef u32x4 words __attribute__((aligned(2)));
            const u32x4 v = *reinterpret_cast<const words*>(static_cast<const uint16_t*>(rows) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) p[2 * i] = counted(bf16_lo_to_f32(v[i])), p[2 * i + 1] = counted(bf16_hi_to_f32(v[i]));
        } else {
            typedef float f32x4v __attribute__((ext_vector_type(4)));
            typedef f32x4v words __attribute__((aligned(4)));
            const words* src = reinterpret_cast<const words*>(static_cast<const float*>(rows) + at);
            const f32x4v lo = src[0], hi = src[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = counted(lo[i]), p[4 + i] = counted(hi[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = i < n ? prob<BF16>(rows, at + i) : 0.0f;
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
__device__ __forceinline__ double lanes_sum(double x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
    return x;
}

template <bool BF16>
__global__ __launch_bounds__(kVerifyThreads) void draft_verify_kernel(const VerifyArgs a) {
    __shared__ int parent[kVerifyNodes], token[kVerifyNodes], gone[kVerifyNodes];  // gone: tokens rejected at cur
    __shared__ float share[kVerifyNodes], p_of[kVerifyNodes], q_of[kVerifyNodes];
    __shared__ double level[kVerifyNodes];  // c_0 .. c_k at cur
    __shared__ double sums[kVerifyBlocks];
    __shared__ int state[4];
    __shared__ double all;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int node0 = min(max(a.cu[seq], 0), a.n_nodes);
    const int n = min(max(a.cu[seq + 1] - node0, 0), min(a.max_nodes, a.n_nodes - node0));
    int* const path = a.path + (size_t)seq * a.max_nodes;
    if (n == 0) {
        for (int i = tid; i < a.max_nodes; i += kVerifyThreads) path[i] = -1;
        if (tid == 0) a.n_path[seq] = 0, a.next[seq] = -1;
        return;
    }
    for (int i = tid; i < n; i += kVerifyThreads) {
        int up = i > 0 ? a.parents[node0 + i] : -1;
        const int x = a.tokens[node0 + i];
        if (i > 0 && !((unsigned)up < (unsigned)i && (unsigned)x < (unsigned)a.vocab)) {
            up = -1;  // no node's child
            if (a.bad) atomicAdd(a.bad, 1u);
        }
        parent[i] = up, token[i] = x, share[i] = a.u[node0 + i];
        const bool there = up >= 0;
        p_of[i] = there ? prob<BF16>(a.target, (long long)(node0 + up) * a.target_stride + x) : 0.0f;
        q_of[i] = there && a.draft ? prob<BF16>(a.draft, (long long)(node0 + up) * a.draft_stride + x) : 1.0f;
    }
    __syncthreads();

    const int blocks = (a.vocab + kVerifyBlock - 1) / kVerifyBlock;
    // w of eight tokens from v on, after `k` rejections at `cur`
    auto weights = [&](int cur, int k, int v, double (&w)[8]) {
        float p[8], q[8];
        prob8<BF16>(a.target, (long long)(node0 + cur) * a.target_stride + v, a.vocab - v, p);
        if (a.draft && k > 0) prob8<BF16>(a.draft, (long long)(node0 + cur) * a.draft_stride + v, a.vocab - v, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (double)p[i];
        if (a.draft) {
            for (int j = 0; j < k; ++j) {
                const double c = level[j];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = fmax(w[i] - c * (double)q[i], 0.0);
            }
        } else {
            for (int j = 0; j < k; ++j) {
                const int x = gone[j] - v;
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = x == i ? 0.0 : w[i];
            }
        }
    };
    // The sums of every block, and of all of them.
    auto sum_row = [&](int cur, int k) {
        for (int b = wave; b < blocks; b += kVerifyWaves) {
            double w[8];
            weights(cur, k, b * kVerifyBlock + 8 * lane, w);
            const double s = lanes_sum(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
            if (lane == 0) sums[b] = s;
        }
        __syncthreads();
        if (wave == 0) {
            double s = 0.0;
            for (int b = lane; b < blocks; b += kWave) s += sums[b];
            s = lanes_sum(s);
            if (lane == 0) all = s;
        }
        __syncthreads();
    };

    // ---- the walk: wave 0 goes on until it is done or needs the sum of a residual ------------------------------
    auto child_after = [&](int cur, int last) -> int {
        for (int b = last + 1; b < n; b += kWave) {
            const unsigned long long m = __builtin_amdgcn_ballot_w64(b + lane < n && parent[min(b + lane, n - 1)] == cur);
            if (m) return b + __builtin_ctzll(m);
        }
        return -1;
    };
    int cur = 0, last = 0, k = 0, count = 1;
    if (tid == 0) path[0] = 0, level[0] = 1.0;
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
                if (a.draft) {
                    for (int j = 0; j < k; ++j) w = fmax(w - level[j] * q, 0.0);
                } else {
                    for (int j = 0; j < k; j += kWave)
                        if (__builtin_amdgcn_ballot_w64(j + lane < k && gone[min(j + lane, k - 1)] == x)) w = 0.0;
                }
                if ((double)share[child] * q * c < w) {
                    cur = child, k = 0;
                    if (lane == 0) path[count] = child;
                    ++count;
                    continue;
                }
                if (lane == 0) gone[k] = x;
                if (lane == 0 && !a.draft && k + 1 < kVerifyNodes) level[k + 1] = c - w;
                __builtin_amdgcn_wave_barrier();
                ++k;
                if (a.draft && child_after(cur, last) >= 0) {  // (the sum is for a sibling's test)
                    need = 1;
                    break;
                }
            }
            if (lane == 0) state[0] = cur, state[1] = k, state[2] = need;
        }
        __syncthreads();
        const int at = state[0], after = state[1], need = state[2];
        if (!need) break;
        sum_row(at, after);
        if (tid == 0) level[after] = all;
        __syncthreads();
    }
    cur = state[0], k = state[1];
    if (wave == 0) {
        for (int i = count + lane; i < a.max_nodes; i += kWave) path[i] = -1;
        if (lane == 0) a.n_path[seq] = count;
    }

    // ---- the next token ----------------------------------------------------------------------------------------
    sum_row(cur, k);
    if (!(all > 0.0) && k > 0) {  // nothing is left of it: the node's own row
        k = 0;
        __syncthreads();
        sum_row(cur, 0);
    }
    if (wave != 0) return;
    if (!(all > 0.0)) {
        if (lane == 0) a.next[seq] = -1;
        return;
    }
    // the block: a lane has `each` of them in a row
    const double goal = (double)a.u_final[seq] * all;
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
    int block = some;
    for (int i = 0; i < each; ++i) {
        const int b = holder * each + i;
        if (b >= blocks || b >= some) break;
        if (run + sums[b] > goal) {
            block = b;
            break;
        }
        run += sums[b];
    }
    // and in it: the first past the goal, or the last with anything in it where the sums' roundings leave none
    double w[8];
    const int v = block * kVerifyBlock + 8 * lane;
    weights(cur, k, v, w);
    double upto = run + lanes_before(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])), total);
    int first = -1, held = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        upto += w[i];
        if (w[i] > 0.0) {
            held = v + i;
            if (first < 0 && upto > goal) first = v + i;
        }
    }
    const unsigned long long found = __builtin_amdgcn_ballot_w64(first >= 0), left = __builtin_amdgcn_ballot_w64(held >= 0);
    const int answer = found ? __shfl(first, __builtin_ctzll(found), kWave) : __shfl(held, 63 - __builtin_clzll(left), kWave);
    if (lane == 0) a.next[seq] = answer;
}

}  // namespace rk

extern "C" size_t rivoli_draft_verify_workspace_bytes(int n_seqs, int max_nodes, int vocab) {
    (void)n_seqs, (void)max_nodes, (void)vocab;
    return 0;
}

extern "C" int rivoli_draft_verify(const void* target_probs, const void* draft_probs, const int* tokens,
                                   const int* parents, const int* cu_nodes, const float* uniforms,
                                   const float* final_uniforms, int n_seqs, int n_nodes, int max_nodes, int vocab,
                                   long long target_stride, long long draft_stride, int bf16, int* path, int* n_path,
                                   int* next_token, void* workspace, unsigned int* bad_nodes, void* stream) {
    (void)workspace;
    if (!target_probs || !tokens || !parents || !cu_nodes || !uniforms || !final_uniforms || !path || !n_path ||
        !next_token || n_seqs <= 0 || n_nodes <= 0 || max_nodes <= 0 || vocab <= 0)
        return 1001;
    if (max_nodes > rk::kVerifyNodes || vocab > rk::kVerifyBlocks * rk::kVerifyBlock || target_stride < vocab ||
        (draft_probs && draft_stride < vocab))
        return 1002;
    const uintptr_t size = bf16 ? 2 : 4;
    if ((uintptr_t)target_probs % size != 0 || (uintptr_t)draft_probs % size != 0) return 1004;
    const rk::VerifyArgs a{target_probs, draft_probs, tokens, parents, cu_nodes, uniforms, final_uniforms, n_nodes, max_nodes, vocab,
                           target_stride, draft_stride, path, n_path, next_token, bad_nodes};
    (void)hipGetLastError();
    const dim3 grid((unsigned)n_seqs), block(rk::kVerifyThreads);
    if (bf16) rk::launch_kernel(rk::draft_verify_kernel<true>, grid, block, 0, (hipStream_t)stream, a);
    else rk::launch_kernel(rk::draft_verify_kernel<false>, grid, block, 0, (hipStream_t)stream, a);
    return rk::launch_status();
}
