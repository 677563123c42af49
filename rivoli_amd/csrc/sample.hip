// Tokens drawn from logits by given random numbers, after temperature, top-k, top-p and min-p, and the distributions that
// they are drawn from. Launch-only.
//
// A row's tokens in order of their logits, equal ones by their index; token v weighs w_v = exp((x_v - max) / T). Kept are the first k of them; of
// those the shortest beginning that weighs p of their whole; of those the ones with w_v >= m. All three keep a beginning of the same order, so
// what is kept is known by its last token, the cut. The token drawn is the first, by index, whose running weight exceeds u times the whole of what is kept.
//
// Which tokens are kept and which one is drawn are decided by sums of up to 2^21 weights next to a border, so that weights and sums have more than 32 bits: over 131 072 tokens
// sums in f32 would move a draw in some hundred. A weight is made in 64 bits to 10^-14 and summed as a whole number of 2^-42 of the largest (in a histogram 2^-36 of
// its bin's least), so that no sum depends on its order and equal calls give equal tokens.
#include <cfloat>

#include "codec.hpp"

namespace rk {

// Bins of a logit: of a power of two's width h, 16 to 32 of them to T, numbered on one grid for all of a row: x / h and the place in a bin are exact. Below a
// chunk's largest logit's bin are kSampleBins of them in its histogram; what lies lower (e^-16 of it and less) is a tail, counted as a whole.
constexpr int kSampleBins = 512;
constexpr int kSampleThreads = 256, kSampleItems = 32;
constexpr int kSampleChunk = kSampleThreads * kSampleItems;  // tokens a workgroup of the first launch
constexpr int kSampleMaxVocab = 1 << 21, kSampleMaxChunks = kSampleMaxVocab / kSampleChunk;
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / kWave;
constexpr int kPickList = 8192;            // tokens in LDS
constexpr int kPickSubs = 2048, kPickFew = 256;
constexpr double kMassOne = 4398046511104.0;       // 2^42
constexpr double kBinOne = 68719476736.0;          // 2^36
constexpr double kWhole = 4503599627370496.0;      // 2^52: a number below it added to it is a whole number in its low bits
constexpr unsigned long long kWholeBits = 0x4330000000000000ull;
constexpr int kCountShift = 50;            // of a histogram's word: tokens above, their weight below (2^13 tokens of 2^36.1 at most)

typedef unsigned long long u64;

struct SampleChunk {
    double top;                  // its largest logit's bin
    u64 mass;                    // of all of its tokens, or, where there is a histogram, of the tail, in 2^-42 of the weight at that bin's beginning
    float most;                  // its largest logit
    int first;                   // that one's token
    unsigned count, tail;        // tokens that may be drawn, and of the tail
};
struct SampleEnd {               // what the third launch writes a row's probabilities by
    double top, inv;             // the row's top bin, 1 / the whole of what is kept
    u64 cut;                     // the last kept token's place in the order
    int token, kind;             // kind: 0 nothing may be drawn, 1 one token, 2 by weight
};
struct SampleArgs {
    const void* logits;
    const float *temperatures, *top_ps, *min_ps, *uniforms;
    const int* top_ks;
    int n_rows, vocab, chunks;
    long long stride, probs_stride;
    int *tokens, *n_kept;
    float *logprobs, *probs;
    SampleChunk* chunk;
    u64* hist;                   // [rows][chunks][kSampleBins]
    SampleEnd* end;
};

struct SampleRow {
    bool greedy, k_on, p_on, m_on;
    int k;
    double inv_h, a, p, m;       // a = h / T
    __device__ __forceinline__ bool filtered() const { return k_on || p_on || m_on; }
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int row) {
    SampleRow r;
    const float t = a.temperatures ? a.temperatures[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    const double td = r.greedy ? 1.0 : (double)fminf(t, FLT_MAX);
    const int e = ilogb(td) - 4;
    r.inv_h = ldexp(1.0, -e), r.a = ldexp(1.0, e) / td;
    r.k = a.top_ks ? a.top_ks[row] : 0;
    r.p = a.top_ps ? (double)a.top_ps[row] : 1.0;
    r.m = a.min_ps ? fmin((double)a.min_ps[row], 1.0) : 0.0;
    if (r.p <= 0.0 || (a.min_ps && a.min_ps[row] > 1.0f)) r.k = 1;  // (the first token alone)
    r.k_on = r.k > 0 && r.k < a.vocab;
    r.p_on = r.p > 0.0 && r.p < 1.0;
    r.m_on = r.m > 0.0;
    return r;
}

// A logit as it counts: what is no number as -inf, which is never drawn; infinity as the largest number; one zero.
__device__ __forceinline__ float logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX) + 0.0f; }

// The bin, and the weight over that of the bin's beginning: exp(y), 0 <= y < 1/16, to 6e-15 by its series.
__device__ __forceinline__ double bin_of(const SampleRow& r, float x, double& weight) {
    const double t = (double)x * r.inv_h, b = floor(t), y = (t - b) * r.a;
    double s = 1.0 / 5040;
    s = __builtin_fma(s, y, 1.0 / 720), s = __builtin_fma(s, y, 1.0 / 120), s = __builtin_fma(s, y, 1.0 / 24);
    s = __builtin_fma(s, y, 1.0 / 6), s = __builtin_fma(s, y, 0.5), s = __builtin_fma(s, y, 1.0);
    weight = __builtin_fma(s, y, 1.0);
    return b;
}
// What a bin's beginning weighs, `down` bins below the top: exp(-a down) by two tables of 64.
struct SampleTable {
    double fine[64], coarse[64];
    __device__ __forceinline__ double of(double down) const {
        const int g = (int)fmin(down, 4096.0);
        return g >= 4096 ? 0.0 : fine[g & 63] * coarse[g >> 6];
    }
};
__device__ __forceinline__ void make_table(SampleTable& t, const SampleRow& r) {
    if (threadIdx.x < 64) t.fine[threadIdx.x] = exp(-r.a * (double)threadIdx.x);
    else if (threadIdx.x < 128) t.coarse[threadIdx.x - 64] = exp(-r.a * 64.0 * (double)(threadIdx.x - 64));
}
__device__ __forceinline__ u64 whole(double x) { return __builtin_bit_cast(u64, x + kWhole) - kWholeBits; }  // x < 2^51
__device__ __forceinline__ u64 mass_of(double weight) { return whole(weight * kMassOne); }
// The same of a sum's product with a weight: up to 2^63.
__device__ __forceinline__ u64 scaled(u64 mass, double by) { return (u64)((double)mass * by + 0.5); }

// A token's place in the order, larger first: its logit's bits in order, then the lower index.
__device__ __forceinline__ u64 place_of(float x, unsigned index) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t key = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return ((u64)key << 21) | (kSampleMaxVocab - 1 - index);
}
__device__ __forceinline__ unsigned index_of(u64 place) { return kSampleMaxVocab - 1 - (unsigned)(place & (kSampleMaxVocab - 1)); }

// N tokens of a row from `at` on (bf16: eight, f32: four), those at `end` and past it as -inf. A row starts on an element.
template <bool BF16>
struct Logits;
template <>
struct Logits<true> {
    static constexpr int N = 8;
    u32x4 v;
    __device__ __forceinline__ void load(const void* rows, long long row, int at, int end) {
        typedef u32x4 words __attribute__((aligned(2)));
        const uint16_t* const src = static_cast<const uint16_t*>(rows) + row + at;
        v = u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
        if (at + 8 <= end) {
            v = *reinterpret_cast<const words*>(src);
        } else {
            for (int i = 0; i < end - at; ++i) {
                const uint32_t one = src[i], shift = 16 * (i & 1);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = j == i >> 1 ? (v[j] & ~(0xffffu << shift)) | (one << shift) : v[j];
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return logit(i & 1 ? bf16_hi_to_f32(v[i >> 1]) : bf16_lo_to_f32(v[i >> 1])); }
};
template <>
struct Logits<false> {
    static constexpr int N = 4;
    typedef float f32x4v __attribute__((ext_vector_type(4)));
    f32x4v v;
    __device__ __forceinline__ void load(const void* rows, long long row, int at, int end) {
        typedef f32x4v words __attribute__((aligned(4)));
        const float* const src = static_cast<const float*>(rows) + row + at;
        v = f32x4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (at + 4 <= end) {
            v = *reinterpret_cast<const words*>(src);
        } else {
            for (int i = 0; i < end - at; ++i) {
                const float one = src[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = j == i ? one : v[j];
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return logit(v[i]); }
};

__device__ __forceinline__ u64 wave_sum(u64 x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
    return x;
}
__device__ __forceinline__ u64 wave_most(u64 x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = max(x, (u64)__shfl_xor(x, off, kWave));
    return x;
}
__device__ __forceinline__ u64 wave_upto(u64 x) {  // the lane's and those before
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const u64 y = __shfl_up(x, off, kWave);
        if ((int)(threadIdx.x & 63) >= off) x += y;
    }
    return x;
}
// Of a whole workgroup, in every thread.
template <int WAVES>
__device__ __forceinline__ u64 all_sum(u64 x, u64* room) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x += room[i];
    return x;
}
template <int WAVES>
__device__ __forceinline__ u64 all_most(u64 x, u64* room) {
    x = wave_most(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x = max(x, room[i]);
    return x;
}

// ---- the first launch: a chunk of a row -----------------------------------------------------------------------
template <bool BF16>
__global__ __launch_bounds__(kSampleThreads) void sample_chunk_kernel(const SampleArgs a) {
    __shared__ u64 hist[kSampleBins];
    __shared__ SampleTable table;
    __shared__ u64 room[kSampleThreads / kWave];
    constexpr int N = Logits<BF16>::N, kLoads = kSampleItems / N;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks, tid = threadIdx.x;
    const int first = c * kSampleChunk;
    Logits<BF16> v[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) v[j].load(a.logits, (long long)row * a.stride, first + N * (tid + j * kSampleThreads), a.vocab);
    const SampleRow r = sample_row(a, row);
    for (int b = tid; b < kSampleBins; b += kSampleThreads) hist[b] = 0;
    make_table(table, r);
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) most = fmaxf(most, v[j][i]);
    // the largest and the first token that has it
    unsigned at = 0;
#pragma unroll
    for (int j = kLoads - 1; j >= 0; --j)
#pragma unroll
        for (int i = N - 1; i >= 0; --i)
            if (v[j][i] == most) at = first + N * (tid + j * kSampleThreads) + i;
    const u64 best = all_most<kSampleThreads / kWave>(place_of(most, at), room);
    at = index_of(best);
    const uint32_t key = (uint32_t)(best >> 21);
    most = __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
    SampleChunk* const out = a.chunk + (size_t)row * a.chunks + c;
    if (most == -INFINITY) {
        if (tid == 0) *out = SampleChunk{-INFINITY, 0, most, 0, 0, 0};
        return;
    }
    double weight;
    const double top = bin_of(r, most, weight);
    const bool filtered = r.filtered() && !r.greedy;
    unsigned count = 0, tail = 0;
    u64 mass = 0;
    if (!r.greedy) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = v[j][i];
                if (x == -INFINITY) continue;
                ++count;
                const double down = top - bin_of(r, x, weight);
                if (filtered && down < kSampleBins) {
                    atomicAdd(&hist[(int)down], whole(weight * kBinOne) + (1ull << kCountShift));
                } else {
                    ++tail;
                    mass += mass_of(weight * table.of(down));
                }
            }
    }
    mass = all_sum<kSampleThreads / kWave>(mass, room);
    const u64 counts = all_sum<kSampleThreads / kWave>((u64)count << 32 | tail, room);
    if (filtered)
        for (int b = tid; b < kSampleBins; b += kSampleThreads) a.hist[((size_t)row * a.chunks + c) * kSampleBins + b] = hist[b];
    if (tid == 0) *out = SampleChunk{top, mass, most, (int)at, r.greedy ? 1u : (unsigned)(counts >> 32), (unsigned)counts};
}

// ---- the second: a row -------------------------------------------------------------------------------------------
struct PickShared {
    SampleTable table;
    u64 room[kPickWaves];
    u64 chunk_mass[kSampleMaxChunks];
    int shift[kSampleMaxChunks];           // of a chunk's top bin below the row's
    unsigned count[kSampleBins + 1];       // of the bins, then of all up to them; the last is the tail
    u64 mass[kSampleBins + 1];
    unsigned sub_count[kPickSubs];
    u64 sub_mass[kPickSubs];
    u64 few[kPickFew], few_mass[kPickFew];
    float list_x[kPickList];
    unsigned list_at[kPickList];
    unsigned n, found;
    u64 lo, hi, cut, before;
    unsigned rank;
};

// A row as its kept tokens are asked for.
template <bool BF16>
struct Pick {
    const SampleArgs& a;
    const SampleRow r;
    PickShared& sh;
    const int row;
    double top, least;                     // the top bin; the least weight that min-p keeps
    // The weight of a logit, that of the top bin's beginning being one.
    __device__ __forceinline__ double weight_of(float x) const {
        double w;
        const double b = bin_of(r, x, w);
        return w * sh.table.of(top - b);
    }
    __device__ __forceinline__ int bin(float x) const { return (int)fmin(top - floor((double)x * r.inv_h), (double)kSampleBins); }
    // f(x, index) of the tokens in a bin, the tail being bin kSampleBins: those in the list, or all of the row's.
    template <class F>
    __device__ __forceinline__ void each(bool listed, int of, F f) const {
        if (listed) {
            for (unsigned i = threadIdx.x; i < sh.n; i += kPickThreads)
                if (bin(sh.list_x[i]) == of) f(sh.list_x[i], sh.list_at[i]);
        } else {
            row_each([&](float x, unsigned i) {
                if (x != -INFINITY && bin(x) == of) f(x, i);
            }, [](int) {});
        }
    }
    // f(x, index) of all of a row's; then done(first token) after every piece that the workgroup's threads have together: of one chunk.
    template <class F, class D>
    __device__ __forceinline__ void row_each(F f, D done) const {
        constexpr int N = Logits<BF16>::N, kLoads = 4;
        for (int from = 0; from < a.vocab; from += kLoads * N * kPickThreads) {
            Logits<BF16> v[kLoads];
#pragma unroll
            for (int j = 0; j < kLoads; ++j) v[j].load(a.logits, (long long)row * a.stride, from + N * ((int)threadIdx.x + j * kPickThreads), a.vocab);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
#pragma unroll
                for (int i = 0; i < N; ++i) f(v[j][i], (unsigned)(from + N * ((int)threadIdx.x + j * kPickThreads) + i));
                done(from + N * j * kPickThreads);
            }
        }
    }
    // The cut inside of a bin: the place of its rank-th token, or (by mass) of the last whose tokens before it weigh less than `left`; and what the bin's
    // tokens up to it weigh. Places are sorted out 2 048 at a time until few are left, which are compared with each other.
    __device__ void resolve(bool listed, int of, bool by_mass, unsigned rank, u64 left, u64& cut, u64& upto) const {
        const int tid = threadIdx.x;
        u64 most = 0, least_place = 0;  // (the second inverted)
        unsigned n = 0;
        each(listed, of, [&](float x, unsigned i) {
            const u64 p = place_of(x, i);
            most = max(most, p), least_place = max(least_place, ~p), ++n;
        });
        u64 hi = all_most<kPickWaves>(most, sh.room), lo = ~all_most<kPickWaves>(least_place, sh.room);
        n = (unsigned)all_sum<kPickWaves>(n, sh.room);
        u64 before = 0;
        unsigned ahead = 0;
        while (n > kPickFew) {
            const u64 span = hi - lo;
            const int bits = 64 - __builtin_clzll(span | 1), shift = bits > 11 ? bits - 11 : 0;
            __syncthreads();
            for (int i = tid; i < kPickSubs; i += kPickThreads) sh.sub_count[i] = 0, sh.sub_mass[i] = 0;
            __syncthreads();
            each(listed, of, [&](float x, unsigned i) {
                const u64 p = place_of(x, i);
                if (p < lo || p > hi) return;
                const int s = (int)((hi - p) >> shift);
                atomicAdd(&sh.sub_count[s], 1u);
                atomicAdd(&sh.sub_mass[s], mass_of(weight_of(x)));
            });
            __syncthreads();
            if (tid < kWave) {  // a lane has 32 of them
                constexpr int kEach = kPickSubs / kWave;
                u64 m = 0;
                unsigned k = 0;
                for (int i = 0; i < kEach; ++i) m += sh.sub_mass[kEach * tid + i], k += sh.sub_count[kEach * tid + i];
                u64 m_at = wave_upto(m) - m;
                unsigned k_at = (unsigned)(wave_upto(k) - k);
                // the sub-bin of the cut: the first up to which there is enough; the last that has a token where there never is
                int last = -1, hit = -1;
                u64 hit_m = 0, last_m = 0;
                unsigned hit_k = 0, last_k = 0;
                for (int i = 0; i < kEach; ++i) {
                    const int s = kEach * tid + i;
                    const u64 dm = sh.sub_mass[s];
                    const unsigned dk = sh.sub_count[s];
                    if (dk) {
                        last = s, last_m = m_at, last_k = k_at;
                        if (hit < 0 && (by_mass ? before + m_at + dm >= left : ahead + k_at + dk >= rank)) hit = s, hit_m = m_at, hit_k = k_at;
                    }
                    m_at += dm, k_at += dk;
                }
                const u64 hits = __builtin_amdgcn_ballot_w64(hit >= 0), lasts = __builtin_amdgcn_ballot_w64(last >= 0);
                const int lane = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(lasts);
                if (tid == lane) {
                    const int s = hits ? hit : last;
                    sh.hi = hi - ((u64)s << shift);
                    const u64 size = (1ull << shift) - 1;
                    sh.lo = sh.hi - lo > size ? sh.hi - size : lo;
                    sh.before = hits ? hit_m : last_m;
                    sh.rank = hits ? hit_k : last_k;
                    sh.found = sh.sub_count[s];
                }
            }
            __syncthreads();
            hi = sh.hi, lo = sh.lo, before += sh.before, ahead += sh.rank, n = sh.found;
        }
        __syncthreads();
        if (tid == 0) sh.found = 0, sh.cut = ~0ull;
        __syncthreads();
        each(listed, of, [&](float x, unsigned i) {
            const u64 p = place_of(x, i);
            if (p < lo || p > hi) return;
            const unsigned k = atomicAdd(&sh.found, 1u);
            if (k < kPickFew) sh.few[k] = p, sh.few_mass[k] = mass_of(weight_of(x));
        });
        __syncthreads();
        if (tid < (int)n) {
            const u64 p = sh.few[tid];
            u64 m = before;
            unsigned k = ahead;
            for (unsigned j = 0; j < n; ++j)
                if (sh.few[j] > p) m += sh.few_mass[j], ++k;
            // (the first is kept whatever it takes: it is in the bin of the cut)
            if (by_mass ? m < left || k == ahead : k < rank) {
                atomicMin(&sh.cut, p);
            }
        }
        __syncthreads();
        cut = sh.cut;
        u64 m = 0;
        if (tid < (int)n && sh.few[tid] >= cut) m = sh.few_mass[tid];
        upto = before + all_sum<kPickWaves>(m, sh.room);
    }
};

template <bool BF16>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(const SampleArgs a) {
    __shared__ PickShared sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    const SampleChunk* const chunks = a.chunk + (size_t)row * a.chunks;
    SampleChunk mine{-INFINITY, 0, -INFINITY, 0, 0, 0};
    if (tid < a.chunks) mine = chunks[tid];
    const SampleRow r = sample_row(a, row);
    const float u = a.uniforms[row];
    make_table(sh.table, r);
    const u64 best = all_most<kPickWaves>(mine.count ? place_of(mine.most, (unsigned)mine.first) : 0, sh.room);
    const unsigned candidates = (unsigned)all_sum<kPickWaves>(mine.count, sh.room);
    const auto finish = [&](int token, unsigned kept, float logprob, const SampleEnd& end) {
        a.tokens[row] = token;
        if (a.n_kept) a.n_kept[row] = (int)kept;
        if (a.logprobs) a.logprobs[row] = logprob;
        a.end[row] = end;
    };
    if (candidates == 0) {
        if (tid == 0) finish(-1, 0, -INFINITY, SampleEnd{0, 0, 0, -1, 0});
        return;
    }
    const int greedy = (int)index_of(best);
    if (r.greedy) {
        if (tid == 0) finish(greedy, 1, 0.0f, SampleEnd{0, 0, 0, greedy, 1});
        return;
    }
    const uint32_t key = (uint32_t)(best >> 21);
    const float most = __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
    double most_weight;
    const double top = bin_of(r, most, most_weight);
    Pick<BF16> pick{a, r, sh, row, top, r.m_on ? r.m * most_weight : 0.0};
    u64 cut = 0;
    unsigned kept = candidates;
    bool listed = false;
    if (tid < kSampleMaxChunks) sh.chunk_mass[tid] = 0;
    if (tid < a.chunks) {
        sh.shift[tid] = mine.count ? (int)fmin(top - mine.top, 4096.0) : 4096;
        if (!r.filtered() && mine.count) sh.chunk_mass[tid] = scaled(mine.mass, sh.table.of(top - mine.top));
    }
    if (r.filtered()) {
        // ---- the row's histogram
        if (tid <= kSampleBins) sh.count[tid] = 0, sh.mass[tid] = 0;
        __syncthreads();
        {
            const int b = tid & (kSampleBins - 1);
            constexpr int kAtOnce = 8;
            for (int c0 = tid / kSampleBins; c0 < a.chunks; c0 += 2 * kAtOnce) {
                u64 v[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int c = c0 + 2 * j;
                    v[j] = c < a.chunks && sh.shift[c] < 4096 ? a.hist[((size_t)row * a.chunks + c) * kSampleBins + b] : 0;
                }
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    if (v[j] == 0) continue;
                    const int g = b + sh.shift[c0 + 2 * j];
                    const u64 m = v[j] & ((1ull << kCountShift) - 1);
                    // (the tail's weights are rounded one by one)
                    atomicAdd(&sh.count[min(g, kSampleBins)], (unsigned)(v[j] >> kCountShift));
                    atomicAdd(&sh.mass[min(g, kSampleBins)], g < kSampleBins ? m : scaled(m, sh.table.of(g) * (kMassOne / kBinOne)));
                }
            }
            if (mine.count) {
                // a chunk far below the top has no histogram that is looked at: its tokens belong to the tail, and weigh nothing
                atomicAdd(&sh.count[kSampleBins], sh.shift[tid] < 4096 ? mine.tail : mine.count);
                atomicAdd(&sh.mass[kSampleBins], scaled(mine.mass, sh.table.of(top - mine.top)));
            }
        }
        __syncthreads();
        if (tid < kSampleBins) sh.mass[tid] = scaled(sh.mass[tid], sh.table.of(tid) * (kMassOne / kBinOne));
        __syncthreads();
        if (tid < kWave) {  // sums up to each bin: a lane has eight
            constexpr int kEach = kSampleBins / kWave;
            u64 m = 0;
            unsigned k = 0;
            for (int i = 0; i < kEach; ++i) m += sh.mass[kEach * tid + i], k += sh.count[kEach * tid + i];
            u64 m_at = wave_upto(m) - m;
            unsigned k_at = (unsigned)(wave_upto(k) - k);
            for (int i = 0; i < kEach; ++i) {
                sh.mass[kEach * tid + i] = m_at += sh.mass[kEach * tid + i];
                sh.count[kEach * tid + i] = k_at += sh.count[kEach * tid + i];
            }
            if (tid == kWave - 1) sh.mass[kSampleBins] += m_at, sh.count[kSampleBins] += k_at;
        }
        __syncthreads();
        // the first bin up to which there is enough, the tail if never: in every thread, by a search
        const auto bin_by_count = [&](unsigned want) {
            int lo = 0, hi = kSampleBins;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (sh.count[mid] >= want) hi = mid;
                else lo = mid + 1;
            }
            return lo;
        };
        const auto bin_by_mass = [&](u64 want) {
            int lo = 0, hi = kSampleBins;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (sh.mass[mid] >= want) hi = mid;
                else lo = mid + 1;
            }
            return lo;
        };
        const bool by_k = r.k_on && (unsigned)r.k < candidates;
        const auto share = [&](u64 mass) -> u64 { return max((u64)ceil(r.p * (double)mass), 1ull); };
        int last = kSampleBins;            // the lowest bin that may have a kept token
        const int k_bin = by_k ? bin_by_count((unsigned)r.k) : kSampleBins;
        if (by_k) last = k_bin;
        else if (r.p_on) last = bin_by_mass(share(sh.mass[kSampleBins]));
        if (r.m_on) {  // the first whose beginning is too light: bins past it hold nothing that is kept
            int lo = 0, hi = kSampleBins;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (sh.table.of(mid) < pick.least) hi = mid;
                else lo = mid + 1;
            }
            last = min(last, lo);
        }
        // ---- the tokens down to there (what the first k weigh is asked for by top-p, wherever min-p ends), where they are no more than the list has room for
        const int depth = by_k && r.p_on ? k_bin : last;
        listed = depth < kSampleBins && sh.count[depth] <= kPickList;
        if (tid == 0) sh.n = 0;
        __syncthreads();
        if (listed) {
            const double edge = (top - depth) / r.inv_h;  // exact: a whole number times a power of two
            pick.row_each([&](float x, unsigned i) {
                if (x != -INFINITY && (double)x >= edge) {
                    const unsigned at = atomicAdd(&sh.n, 1u);
                    if (at < kPickList) sh.list_x[at] = x, sh.list_at[at] = i;
                }
            }, [](int) {});
            __syncthreads();
            if (tid == 0) sh.n = min(sh.n, (unsigned)kPickList);
            __syncthreads();
        }
        // ---- the cut
        u64 whole_mass = sh.mass[kSampleBins];
        const auto count_before = [&](int b) { return b ? sh.count[b - 1] : 0u; };
        const auto mass_before = [&](int b) { return b ? sh.mass[b - 1] : 0ull; };
        if (by_k && (r.p_on || k_bin <= last)) {
            u64 upto;
            pick.resolve(listed, k_bin, false, (unsigned)r.k - count_before(k_bin), 0, cut, upto);
            whole_mass = mass_before(k_bin) + upto;
        }
        if (r.p_on) {
            const u64 want = share(whole_mass);
            const int p_bin = min(bin_by_mass(want), by_k ? k_bin : kSampleBins);
            if (p_bin <= last) {
                u64 upto, p_cut;
                const u64 ahead = mass_before(p_bin);
                pick.resolve(listed, p_bin, true, 0, want > ahead ? want - ahead : 1, p_cut, upto);
                cut = max(cut, p_cut);
            }
        }
        __syncthreads();
        // ---- what is kept, by chunk
        unsigned n = 0;
        u64 end = 0;                       // (inverted: the last kept token's place)
        const auto keep = [&](float x, unsigned i) -> u64 {
            const u64 p = place_of(x, i);
            if (p < cut) return 0;
            const double w = pick.weight_of(x);
            if (w < pick.least) return 0;
            ++n, end = max(end, ~p);
            return mass_of(w);
        };
        if (listed) {
            for (unsigned i = tid; i < sh.n; i += kPickThreads) {
                const u64 m = keep(sh.list_x[i], sh.list_at[i]);
                if (m) atomicAdd(&sh.chunk_mass[sh.list_at[i] / kSampleChunk], m);
            }
        } else {
            u64 piece = 0;
            pick.row_each([&](float x, unsigned i) {
                if (x != -INFINITY) piece += keep(x, i);
            }, [&](int from) {
                piece = wave_sum(piece);
                if (piece && (tid & 63) == 0) atomicAdd(&sh.chunk_mass[from / kSampleChunk], piece);
                piece = 0;
            });
        }
        kept = (unsigned)all_sum<kPickWaves>(n, sh.room);
        cut = ~all_most<kPickWaves>(end, sh.room);
    }
    // ---- the chunk that the draw falls into, and the token
    __syncthreads();
    u64 all = 0;
    int c = -1, last_c = 0;
    for (int i = 0; i < a.chunks; ++i) all += sh.chunk_mass[i];
    const double target = (double)u * (double)all;
    u64 run = 0, run_c = 0, run_last = 0;
    for (int i = 0; i < a.chunks; ++i) {
        const u64 m = sh.chunk_mass[i];
        if (m) {
            if (c < 0 && (double)(run + m) > target) c = i, run_c = run;
            last_c = i, run_last = run;
        }
        run += m;
    }
    if (c < 0) c = last_c, run_c = run_last;
    constexpr int kEach = kSampleChunk / kPickThreads;
    float x[kEach];
    u64 m[kEach], sum = 0;
    const int from = c * kSampleChunk + kEach * tid;
#pragma unroll
    for (int i = 0; i < kEach; i += Logits<BF16>::N) {
        Logits<BF16> v;
        v.load(a.logits, (long long)row * a.stride, min(from + i, a.vocab), a.vocab);
#pragma unroll
        for (int j = 0; j < Logits<BF16>::N; ++j) x[i + j] = v[j];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        m[i] = x[i] != -INFINITY && place_of(x[i], (unsigned)(from + i)) >= cut ? mass_of(pick.weight_of(x[i])) : 0;
        sum += m[i];
    }
    // the threads' sums in order
    const u64 upto = wave_upto(sum);
    __syncthreads();
    if ((tid & 63) == 63) sh.room[tid >> 6] = upto;
    if (tid == 0) sh.lo = ~0ull, sh.hi = 0;
    __syncthreads();
    u64 before = run_c + upto - sum;
    for (int w = 0; w < tid >> 6; ++w) before += sh.room[w];
    int hit = -1, last = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (m[i]) {
            if (hit < 0 && (double)(before + m[i]) > target) hit = i;
            last = i;
        }
        before += m[i];
    }
    if (hit >= 0) atomicMin(&sh.lo, (u64)(from + hit));
    if (last >= 0) atomicMax(&sh.hi, (u64)(from + last));
    __syncthreads();
    const int token = (int)(sh.lo != ~0ull ? sh.lo : sh.hi);
    if (token >= from && token < from + kEach) {
        float of = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) of = token - from == i ? x[i] : of;
        const double whole_weight = (double)all / kMassOne;
        finish(token, kept, (float)log(pick.weight_of(of) / whole_weight), SampleEnd{top, 1.0 / whole_weight, cut, token, 2});
    }
}

// ---- the third, where probabilities are asked for -------------------------------------------------------------------
template <bool BF16>
__global__ __launch_bounds__(kSampleThreads) void sample_probs_kernel(const SampleArgs a) {
    __shared__ SampleTable table;
    constexpr int N = Logits<BF16>::N, kLoads = kSampleItems / N;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks, tid = threadIdx.x;
    Logits<BF16> v[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) v[j].load(a.logits, (long long)row * a.stride, min(c * kSampleChunk + N * (tid + j * kSampleThreads), a.vocab), a.vocab);
    const SampleRow r = sample_row(a, row);
    const SampleEnd end = a.end[row];
    make_table(table, r);
    __syncthreads();
    float* const out = a.probs + (long long)row * a.probs_stride;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int at = c * kSampleChunk + N * (tid + j * kSampleThreads);
        float p[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p[i] = 0.0f;
            if (end.kind == 1) p[i] = at + i == end.token ? 1.0f : 0.0f;
            if (end.kind == 2 && v[j][i] != -INFINITY && place_of(v[j][i], (unsigned)(at + i)) >= end.cut) {
                double w;
                const double b = bin_of(r, v[j][i], w);
                p[i] = (float)(w * table.of(end.top - b) * end.inv);
            }
        }
        typedef float f32x4v __attribute__((ext_vector_type(4)));
        typedef f32x4v words __attribute__((aligned(4)));
        if (at + N <= a.vocab) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<words*>(out + at + i) = f32x4v{p[i], p[i + 1], p[i + 2], p[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < a.vocab) out[at + i] = p[i];
        }
    }
}

static size_t sample_chunks(int vocab) { return ((size_t)vocab + kSampleChunk - 1) / kSampleChunk; }
static size_t sample_bytes(int n_rows, int vocab) {
    if (n_rows <= 0 || vocab <= 0 || vocab > kSampleMaxVocab) return 0;
    const size_t chunks = (size_t)n_rows * sample_chunks(vocab);
    return chunks * (kSampleBins * sizeof(u64) + sizeof(SampleChunk)) + (size_t)n_rows * sizeof(SampleEnd);
}

template <bool BF16>
static int sample_rows(const SampleArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((size_t)a.n_rows * a.chunks)), block(kSampleThreads);
    (void)hipGetLastError();
    launch_kernel(sample_chunk_kernel<BF16>, grid, block, 0, st, a);
    int rc = launch_status();
    if (rc != 0) return rc;
    launch_kernel(sample_pick_kernel<BF16>, dim3((unsigned)a.n_rows), dim3(kPickThreads), 0, st, a);
    rc = launch_status();
    if (rc != 0 || !a.probs) return rc;
    launch_kernel(sample_probs_kernel<BF16>, grid, block, 0, st, a);
    return launch_status();
}

}  // namespace rk

extern "C" size_t rivoli_sample_rows_workspace_bytes(int n_rows, int vocab) { return rk::sample_bytes(n_rows, vocab); }

extern "C" int rivoli_sample_rows(const void* logits, const float* temperatures, const int* top_ks, const float* top_ps,
                                  const float* min_ps, const float* uniforms, int n_rows, int vocab, long long stride,
                                  int bf16, int* tokens, int* n_kept, float* logprobs, float* probs, long long probs_stride,
                                  void* workspace, void* stream) {
    if (!logits || !uniforms || !tokens || !workspace || n_rows <= 0 || vocab <= 0) return 1001;
    if (n_rows >= 1 << 22 || vocab > rk::kSampleMaxVocab || (stride != 0 && stride < vocab) || (probs && probs_stride < vocab)) return 1002;
    const uintptr_t size = bf16 ? 2 : 4;
    if ((uintptr_t)logits % size != 0 || (uintptr_t)probs % 4 != 0 || !rk::aligned16(workspace)) return 1004;
    const size_t chunks = rk::sample_chunks(vocab), all = (size_t)n_rows * chunks;
    if (all * rk::kSampleThreads > rk::kLaunchThreads || (size_t)n_rows * rk::kPickThreads > rk::kLaunchThreads) return 1002;
    rk::u64* const hist = static_cast<rk::u64*>(workspace);
    rk::SampleChunk* const chunk = reinterpret_cast<rk::SampleChunk*>(hist + all * rk::kSampleBins);
    rk::SampleEnd* const end = reinterpret_cast<rk::SampleEnd*>(chunk + all);
    const rk::SampleArgs a{logits, temperatures, top_ps, min_ps, uniforms, top_ks, n_rows, vocab, (int)chunks, stride, probs_stride, tokens, n_kept,
                           logprobs, probs, chunk, hist, end};
    return bf16 ? rk::sample_rows<true>(a, (hipStream_t)stream) : rk::sample_rows<false>(a, (hipStream_t)stream);
}
