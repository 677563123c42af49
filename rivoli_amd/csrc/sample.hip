// Tokens drawn from logits by given random numbers, after temperature, top-k, top-p and min-p, and the distributions that
// they are drawn from. Launch-only.
//
// A row's tokens in order of their logits, equal ones by their index; token v weighs w_v = exp((x_v - max) / T). Kept are the first k of them; of
// those the shortest beginning that weighs p of their whole; of those the ones with w_v >= m. All three keep a beginning of the same order, so
// what is kept is known by its last token, the cut. The token drawn is the first, by index, whose running weight exceeds u times the whole of what is kept.
//
// Which tokens are kept and which one is drawn are decided by sums of up to 2^21 weights next to a border, so that weights and sums have more than 32 bits: over 131 072 tokens
// sums in f32 would move a draw in some hundred. A weight is made in 64 bits and summed as a whole number of 2^-42 of the largest (in a histogram 2^-36 of
// its bin's least), so that no sum depends on its order and equal calls give equal tokens; within the chunk that the draw falls into they are summed as they are, in one order.
#include <cfloat>
#include <climits>

#include "codec.hpp"

namespace rk {

typedef unsigned long long u64;

// Logits are binned on one grid for all of a row: bins of a power of two's width h, 16 to 32 of them to T, so that x / h, its bin and its place in the bin are exact in f32, but for
// logits just below zero, whose place is right to 2^-25 of a bin, their weight to 2^-29 (bins have 31 bits: logits not above -2^25 T are never drawn, and a row that has some above 2^25 T, which lie
// two T apart and more, is read by itself, by its logits' distances from the largest). A histogram has some 250 bins from its top on (kFine; 8 T and more), then 256 of eight bins each, another 64 T; what lies
// deeper weighs less than 2^-92 of the top and is a tail that is only counted. Eights begin at multiples of eight, in every histogram of a row, so that histograms
// of unlike tops add up exactly: the finer ones' bins are parts of the coarser ones'.
constexpr int kFine = 256, kSampleBins = 512;
constexpr int kSampleThreads = 256, kSampleItems = 32;
constexpr int kSampleChunk = kSampleThreads * kSampleItems;  // tokens a workgroup of the first launch
constexpr int kSampleMaxVocab = 1 << 21, kSampleMaxChunks = kSampleMaxVocab / kSampleChunk;
// Of a chunk's largest logits that are listed: the first part is asked for by every row's workgroup, the second by those that need more.
constexpr int kSampleList = 128, kSampleMore = 512, kSampleListed = kSampleList + kSampleMore;
constexpr int kPickThreads = 512, kPickWaves = kPickThreads / kWave;
constexpr int kPickList = 8192;            // tokens in LDS
constexpr int kPickSubs = kPickThreads, kPickFew = 512;
// Down to so many tokens that may be kept they are put in order, past them the cut is looked for: 64 rows by k 300 32.1 and 36.6 us, 400 33.8 and 37.0, but 480 37.5 and 37.1; where min-p
// alone cuts, which needs no order, about 300 36.0 and 32.3. The lines lie there for one row and for 256 too: by k 400 26.6 and 30.6, 61.3 and 64.5, by k 480 28.7 and 29.7, 63.3 and 65.0; by min-p 200
// 21.8 and 22.8, 55.8 and 57.5, 300 25.5 and 22.9, 59.4 and 57.6 (bf16).
constexpr unsigned kPickInOrder = 448, kPickInOrderByM = 256;
// Up to this k a row's histogram has counts alone, and by min-p alone from this m on: 64 rows of 131 072 by k 50 25.5 us, with weights 31.9, by k 2 000 43.7 and 47.9, but by k 3 000
// 51.2 and 50.6; by m 0.05 30.4 and 36.7, 0.01 36.5 and 42.2, but by 0.002, where rows may keep more than the list holds, 118 and 54. One row: by k 50 18.7 and 20.8, 2 000 35.7 and 36.7, by m 0.01 18.9 and
// 21.0; 256 rows: 50.0 and 66.4, 71.8 and 87.5, 51.4 and 67.4 (bf16, a few dozen tokens far above the others: k 3 000 76.0 and 90.6 there).
constexpr int kCountedK = 2048;
constexpr double kCountedM = 1.0 / 128;
constexpr float kLeastTemperature = 1.0f / 65536;  // up to it the largest logit is taken
constexpr double kMassOne = 4398046511104.0;       // 2^42
constexpr double kBinOne = 68719476736.0;          // 2^36
constexpr double kWhole = 4503599627370496.0;      // 2^52: a number below it added to it is a whole number in its low bits
constexpr u64 kWholeBits = 0x4330000000000000ull;
constexpr int kCountShift = 50;            // of a histogram's word: tokens above, their weight below (2^13 tokens of 2^36.8 at most)
constexpr u64 kMassBits = (1ull << kCountShift) - 1;

struct SampleChunk {
    double weight;               // of a row without filters: all of its tokens', that of its top bin's beginning being one
    int top, cover[2];           // its largest logit's bin; its tokens of bins from cover on are listed, in the first part alone, in both
    float most;                  // its largest logit
    int first;                   // that one's token, in a row that takes the largest
    unsigned count, listed[2];   // tokens that may be drawn; that are listed in either part
};
struct SampleEnd {               // what the third launch writes a row's probabilities by
    double inv;                  // 1 / the whole of what is kept
    u64 cut;                     // the last kept token's place in the order
    int top;                     // the row's top bin
    int token, kind;             // kind: 0 nothing may be drawn, 1 one token, 2 by weight
    float base;                  // what its logits are taken from before they are binned: its largest in a row past the bins, else zero
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
    u64 *masses, *list;          // [rows][chunks][kSampleBins], where the histogram has weights; [kSampleListed] places
    unsigned* counts;            // [kSampleBins]
    SampleEnd* end;
};

struct SampleRow {
    bool greedy, k_on, p_on, m_on;
    int k;
    float inv_h, most, cap;      // 1 / h; logits up to minus `most` do not count at all, those above `cap` as that: as `most`, where there are bins
    double a, p, m;              // a = h / T
    double c[7];                 // a^k / k! in units of 2^-36, from the first on
    __device__ __forceinline__ bool filtered() const { return k_on || p_on || m_on; }
    // Whether the histogram has weights: not where they are asked for of few tokens alone.
    __device__ __forceinline__ bool weighed() const { return k_on ? k > kCountedK : p_on || !m_on || m < kCountedM; }
    // Whether more tokens than the lists' first parts may be asked for.
    __device__ __forceinline__ bool more() const { return !k_on || k > kSampleList; }
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int row) {
    SampleRow r;
    const float t = a.temperatures ? a.temperatures[row] : 1.0f;
    r.greedy = !(t > kLeastTemperature);
    const float tf = r.greedy ? 1.0f : fminf(t, FLT_MAX);
    const int e = (int)((__float_as_uint(tf) >> 23) & 0xff) - 127 - 4;  // (tf is a normal number)
    r.inv_h = __uint_as_float((uint32_t)(127 - e) << 23), r.most = fminf(tf * 33554432.0f, FLT_MAX);
    r.cap = r.greedy ? INFINITY : r.most;
    r.a = 1.0 / ((double)tf * (double)r.inv_h);
    r.c[0] = r.a * kBinOne;
#pragma unroll
    for (int k = 1; k < 7; ++k) r.c[k] = r.c[k - 1] * (r.a * (1.0 / (k + 1)));
    r.k = a.top_ks ? a.top_ks[row] : 0;
    r.p = a.top_ps ? (double)a.top_ps[row] : 1.0;
    r.m = a.min_ps ? (double)a.min_ps[row] : 0.0;
    if (r.p <= 0.0 || r.m > 1.0) r.k = 1;  // (the first token alone)
    r.k_on = r.k > 0 && r.k < a.vocab;
    r.p_on = r.p > 0.0 && r.p < 1.0;
    r.m_on = r.m > 0.0 && r.m <= 1.0;
    return r;
}
// A logit as it counts: what is no number, or further down than all that counts, as -inf, which is never drawn. (An infinite one past the bins: as the largest number.)
__device__ __forceinline__ float logit(const SampleRow& r, float x) { return x > -r.most ? fminf(x, r.cap) : -INFINITY; }

// The least logit of a bin's, or of one between it and the next that there is.
__device__ __forceinline__ float least_of(const SampleRow& r, int b) {
    float t = (float)b;
    if ((double)t < (double)b) t = __uint_as_float(__float_as_uint(t) + (t < 0.0f ? -1 : 1));
    return t / r.inv_h;
}
// A logit in bins from a row's base: near it exact, far below it, where all weigh nothing, held to the bins' range.
__device__ __forceinline__ float place_in(const SampleRow& r, float x, float base) { return fmaxf(x - base, -r.most) * r.inv_h; }
__device__ __forceinline__ int bin_of(const SampleRow& r, float x) { return (int)floorf(x * r.inv_h); }
// exp(place in the bin * a), or of a place in eight bins, in units of 2^-36 and rounded to a whole number, above 2^52: arguments up to 1/16 are right to 2^-47, up to 1/2 to 2^-23. Every
// weight is one of these, so that sums of either kind agree.
__device__ __forceinline__ double units_in(const SampleRow& r, float place) {
    const double y = (double)place;
    double s = r.c[6];
#pragma unroll
    for (int k = 5; k >= 0; --k) s = __builtin_fma(s, y, r.c[k]);
    return __builtin_fma(s, y, kWhole + kBinOne);
}
// A histogram by its top bin.
struct SampleGrid {
    int top, fine8;              // the least bin that is its own, an eighth of it
    __device__ __forceinline__ explicit SampleGrid(int t) : top(t), fine8((t - 248) >> 3) {}
    __device__ __forceinline__ int of(int b) const { return b >= 8 * fine8 ? top - b : kFine + fine8 - 1 - (b >> 3); }  // (kSampleBins and more: the tail; bin -2^31: what is never drawn)
    __device__ __forceinline__ int least(int i) const { return i < kFine ? max(top - i, 8 * fine8) : 8 * (fine8 - 1 - (i - kFine)); }  // of number i's bins (of some at the change, none)
};
// What a bin's beginning weighs, `down` bins below the top: exp(-a down) by two tables of 64.
struct SampleTable {
    double fine[64], coarse[64];
    __device__ __forceinline__ double of(int down) const { return (unsigned)down >= 4096u ? 0.0 : fine[down & 63] * coarse[down >> 6]; }
};
__device__ __forceinline__ void make_table(SampleTable& t, const SampleRow& r) {
    if (threadIdx.x < 128) {
        const double v = exp(-r.a * (double)(threadIdx.x < 64 ? threadIdx.x : 64 * (threadIdx.x - 64)));
        (threadIdx.x < 64 ? t.fine : t.coarse)[threadIdx.x & 63] = v;
    }
}
__device__ __forceinline__ double rounded_in(const SampleRow& r, float place) { return units_in(r, place) - kWhole; }
__device__ __forceinline__ u64 mass_of(double weight) { return __builtin_bit_cast(u64, __builtin_fma(weight, kMassOne, kWhole)) - kWholeBits; }
// A sum of such numbers times a weight: up to 2^63.
__device__ __forceinline__ u64 scaled(u64 mass, double by) { return (u64)((double)mass * by + 0.5); }

// A token's place in the order, larger first: its logit's bits in order, then the lower index.
__device__ __forceinline__ u64 place_of(float x, unsigned index) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // (one zero)
    const uint32_t key = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return ((u64)key << 21) | (kSampleMaxVocab - 1 - index);
}
__device__ __forceinline__ unsigned index_of(u64 place) { return kSampleMaxVocab - 1 - (unsigned)(place & (kSampleMaxVocab - 1)); }
__device__ __forceinline__ float logit_of(u64 place) {
    const uint32_t key = (uint32_t)(place >> 21);
    return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// N tokens of a row from `at` on (bf16: eight, f32: four). A row starts on an element. `some`: those at `end` and past it are -inf (one by one, the last there is again for those).
template <bool BF16>
struct Logits;
template <>
struct Logits<true> {
    static constexpr int N = 8;
    u32x4 v;
    __device__ __forceinline__ void load(const void* from, unsigned at) {
        typedef u32x4 words __attribute__((aligned(2)));
        v = *reinterpret_cast<const words*>(static_cast<const char*>(from) + 2u * at);
    }
    static __device__ __forceinline__ u32x4 none() { return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
    static __device__ __forceinline__ float one(const void* rows, long long at) { return __uint_as_float((uint32_t)static_cast<const uint16_t*>(rows)[at] << 16); }
    __device__ __forceinline__ void some(const void* rows, long long row, int at, int end) {
        uint32_t one[N];
#pragma unroll
        for (int i = 0; i < N; ++i) one[i] = static_cast<const uint16_t*>(rows)[row + min(at + i, end - 1)];
#pragma unroll
        for (int i = 0; i < N; ++i) one[i] = at + i < end ? one[i] : 0xff80u;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = one[2 * j] | one[2 * j + 1] << 16;
    }
    __device__ __forceinline__ float operator[](int i) const { return i & 1 ? bf16_hi_to_f32(v[i >> 1]) : bf16_lo_to_f32(v[i >> 1]); }
};
template <>
struct Logits<false> {
    static constexpr int N = 4;
    typedef float f32x4v __attribute__((ext_vector_type(4)));
    f32x4v v;
    __device__ __forceinline__ void load(const void* from, unsigned at) {
        typedef f32x4v words __attribute__((aligned(4)));
        v = *reinterpret_cast<const words*>(static_cast<const char*>(from) + 4u * at);
    }
    static __device__ __forceinline__ f32x4v none() { return f32x4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY}; }
    static __device__ __forceinline__ float one(const void* rows, long long at) { return static_cast<const float*>(rows)[at]; }
    __device__ __forceinline__ void some(const void* rows, long long row, int at, int end) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = static_cast<const float*>(rows)[row + min(at + i, end - 1)];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = at + i < end ? v[i] : -INFINITY;
    }
    __device__ __forceinline__ float operator[](int i) const { return v[i]; }
};
// A thread's K of them out of the tokens from `at` on, a piece of the workgroup's `step` tokens after the other, from its own on. Addresses are a scalar and the lane's, and branches
// are few: with one each, every load waited for the one before. Of the piece with the row's end a lane reads tokens one by one.
template <bool BF16, int K>
__device__ __forceinline__ void load_logits(Logits<BF16> (&v)[K], const void* rows, long long row, int at, int own, int step, int end) {
    const int whole = min((end - at) / step, K);  // pieces
    const auto load = [&](int j, int from) { v[j].load(static_cast<const char*>(rows) + (row + at + from * step) * (BF16 ? 2 : 4), (unsigned)own); };
    if (whole == K) {
#pragma unroll
        for (int j = 0; j < K; ++j) load(j, j);
        return;
    }
    Logits<BF16> last;
    last.some(rows, row, at + whole * step + own, end);
    if (whole > 0) {
#pragma unroll
        for (int j = 0; j < K; ++j) load(j, min(j, whole - 1));
    }
#pragma unroll
    for (int j = 0; j < K; ++j) v[j].v = j < whole ? v[j].v : j == whole ? last.v : Logits<BF16>::none();
}

// Sums and maxima over a wave, in every lane, by rotations within sixteen lanes and swaps of those rows: no trip through LDS, which a shuffle is.
template <int CTRL>
__device__ __forceinline__ u64 rotated64(u64 v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)v, CTRL, 0xf, 0xf, true), hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(v >> 32), CTRL, 0xf, 0xf, true);
    return ((u64)hi << 32) | lo;
}
template <class F>
__device__ __forceinline__ u64 wave_all(u64 x, F f) {
    x = f(x, rotated64<0x128>(x)), x = f(x, rotated64<0x124>(x)), x = f(x, rotated64<0x122>(x)), x = f(x, rotated64<0x121>(x));
    auto l = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(x >> 32), (uint32_t)(x >> 32), false, false);
    x = f(((u64)h[0] << 32) | l[0], ((u64)h[1] << 32) | l[1]);
    l = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    h = __builtin_amdgcn_permlane32_swap((uint32_t)(x >> 32), (uint32_t)(x >> 32), false, false);
    return f(((u64)h[0] << 32) | l[0], ((u64)h[1] << 32) | l[1]);
}
__device__ __forceinline__ u64 wave_sum64(u64 x) {
    return wave_all(x, [](u64 a, u64 b) { return a + b; });
}
__device__ __forceinline__ double wave_sum_f64(double x) {
    const auto f = [](u64 a, u64 b) { return __builtin_bit_cast(u64, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b)); };
    return __builtin_bit_cast(double, wave_all(__builtin_bit_cast(u64, x), f));
}
__device__ __forceinline__ u64 wave_most64(u64 x) {
    return wave_all(x, [](u64 a, u64 b) { return a > b ? a : b; });
}
template <int CTRL>
__device__ __forceinline__ float rotated32(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_top(float x) {
    x = fmaxf(x, rotated32<0x128>(x)), x = fmaxf(x, rotated32<0x124>(x)), x = fmaxf(x, rotated32<0x122>(x)), x = fmaxf(x, rotated32<0x121>(x));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// The lane's and those before, as wave_inclusive_sum.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ u64 before64(u64 v) {
    return ((u64)dpp_or_zero<CTRL, ROW_MASK>((uint32_t)(v >> 32)) << 32) | dpp_or_zero<CTRL, ROW_MASK>((uint32_t)v);
}
__device__ __forceinline__ u64 wave_upto(u64 v) {
    v += before64<0x111, 0xf>(v);
    v += before64<0x112, 0xf>(v);
    v += before64<0x114, 0xf>(v);
    v += before64<0x118, 0xf>(v);
    v += before64<0x142, 0xa>(v);
    v += before64<0x143, 0xc>(v);
    return v;
}
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double before_f64(double v) {
    return __builtin_bit_cast(double, before64<CTRL, ROW_MASK>(__builtin_bit_cast(u64, v)));  // (no bits are a zero)
}
__device__ __forceinline__ double wave_upto_f64(double v) {
    v += before_f64<0x111, 0xf>(v);
    v += before_f64<0x112, 0xf>(v);
    v += before_f64<0x114, 0xf>(v);
    v += before_f64<0x118, 0xf>(v);
    v += before_f64<0x142, 0xa>(v);
    v += before_f64<0x143, 0xc>(v);
    return v;
}
// Of a whole workgroup, in every thread.
template <int WAVES>
__device__ __forceinline__ u64 all_sum(u64 x, u64* room) {
    x = wave_sum64(x);
    lds_barrier();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
    lds_barrier();
    x = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x += room[i];
    return x;
}
template <int WAVES>
__device__ __forceinline__ u64 all_most(u64 x, u64* room) {
    x = wave_most64(x);
    lds_barrier();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
    lds_barrier();
    x = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x = max(x, room[i]);
    return x;
}

// ---- the first launch: a chunk of a row -----------------------------------------------------------------------
// Its largest logit, its histogram, and a list of its largest logits, bin by bin as many as there is room for.
// 64 rows of 131 072 in bf16 14.5 us: of a workgroup's 14 000 cycles loads are 2 000, the largest logit 1 500, the histogram 4 000 (with weights 7 000), the lists 5 500. 256 rows in f32
// 51 us, 2.6 TB/s, the vector units busy for 70 % of them (counted): 40 instructions a logit with weights, 7 of them the exponential's products in 64 bits.
template <bool BF16>
__global__ __launch_bounds__(kSampleThreads) void sample_chunk_kernel(const SampleArgs a) {
    __shared__ u64 hist[kSampleListed + kWave];    // its bins or the list, and a lane's spare place
    static_assert(kSampleBins <= kSampleListed, "room for either");
    __shared__ SampleTable table;
    __shared__ u64 room[kSampleThreads / kWave];
    __shared__ unsigned upto[kSampleThreads / kWave], n_listed[2], all_count;
    __shared__ int last_bin[2];
    constexpr int N = Logits<BF16>::N, kLoads = kSampleItems / N, kWaves = kSampleThreads / kWave;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks, tid = threadIdx.x;
    const int first = c * kSampleChunk + N * tid;
    Logits<BF16> raw[kLoads];
    load_logits(raw, a.logits, (long long)row * a.stride, c * kSampleChunk, N * tid, N * kSampleThreads, a.vocab);
    const SampleRow r = sample_row(a, row);
    for (int b = tid; b < kSampleBins; b += kSampleThreads) hist[b] = 0;
    if (tid == 0) n_listed[0] = n_listed[1] = all_count = 0, last_bin[0] = last_bin[1] = -1;
    float v[kSampleItems], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kSampleItems; ++i) v[i] = logit(r, raw[i / N][i % N]), most = fmaxf(most, v[i]);
    const auto index = [&](int i) { return (unsigned)(first + (i / N) * N * kSampleThreads + i % N); };
    SampleChunk* const out = a.chunk + (size_t)row * a.chunks + c;
    if (r.greedy) {
        unsigned at = 0;
#pragma unroll
        for (int i = kSampleItems - 1; i >= 0; --i)
            if (v[i] == most) at = index(i);
        const u64 best = all_most<kWaves>(place_of(most, at), room);
        if (tid == 0) *out = SampleChunk{0, 0, {0, 0}, logit_of(best), (int)index_of(best), logit_of(best) > -INFINITY ? 1u : 0u, {0, 0}};
        return;
    }
    most = wave_top(most);
    if ((tid & 63) == 0) room[tid >> 6] = __float_as_uint(most);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) most = fmaxf(most, __uint_as_float((uint32_t)room[i]));
    if (most == -INFINITY) {
        if (tid == 0) *out = SampleChunk{0, 0, {0, 0}, most, 0, 0, {0, 0}};
        return;
    }
    const SampleGrid grid(bin_of(r, most));
    unsigned* const counts = reinterpret_cast<unsigned*>(hist);
    // No branches: tokens without a bin go to spare ones, a lane's own, so that the elements' chains of dependent instructions run beside each other.
    const int spare = kSampleBins + (tid & 63);
    unsigned count = 0;                    // of the wave
    if (r.weighed()) {
#pragma unroll
        for (int i = 0; i < kSampleItems; ++i) {
            const float t = v[i] * r.inv_h, floor_t = floorf(t);
            const int b = (int)floor_t, at = grid.of(b);
            const float place = t - floor_t + (at < kFine ? 0.0f : (float)(b & 7));
            count += (unsigned)__builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] > -INFINITY));
            atomicAdd(&hist[at < kSampleBins ? at : spare],
                      __builtin_bit_cast(u64, units_in(r, place)) + ((1ull << kCountShift) - kWholeBits));
        }
    } else {
#pragma unroll
        for (int i = 0; i < kSampleItems; ++i) {
            const int at = grid.of(bin_of(r, v[i]));
            count += (unsigned)__builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] > -INFINITY));
            atomicAdd(&counts[at < kSampleBins ? at : spare], 1u);
        }
    }
    if ((tid & 63) == 0) atomicAdd(&all_count, count);
    double weight = 0.0;
    if (!r.filtered()) {
        make_table(table, r);
        lds_barrier();
        for (int i = tid; i < kSampleBins; i += kSampleThreads)
            weight += (double)(hist[i] & kMassBits) * (table.of(grid.top - grid.least(i)) * (1 / kBinOne));
        weight = wave_sum_f64(weight);
        if ((tid & 63) == 0) room[tid >> 6] = __builtin_bit_cast(u64, weight);
        lds_barrier();
        weight = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) weight += __builtin_bit_cast(double, room[i]);
    } else {
        lds_barrier();
        // the histogram goes out, and the bins down to which there is room in the list
        unsigned n[2] = {counts[2 * tid], counts[2 * tid + 1]};
        const size_t to = ((size_t)row * a.chunks + c) * kSampleBins + 2 * tid;
        if (r.weighed()) {
            const u64 two[2] = {hist[2 * tid], hist[2 * tid + 1]};
            n[0] = (unsigned)(two[0] >> kCountShift), n[1] = (unsigned)(two[1] >> kCountShift);
            a.masses[to] = two[0] & kMassBits, a.masses[to + 1] = two[1] & kMassBits;
        }
        a.counts[to] = n[0], a.counts[to + 1] = n[1];
        unsigned sum = wave_inclusive_sum(n[0] + n[1]);
        if ((tid & 63) == 63) upto[tid >> 6] = sum;
        lds_barrier();
        for (int w = 0; w < tid >> 6; ++w) sum += upto[w];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const unsigned room_for = part && r.more() ? kSampleMore : kSampleList;
            // (lanes before one that has room have it too)
            const u64 one = __builtin_amdgcn_ballot_w64(sum - n[1] <= room_for), both = __builtin_amdgcn_ballot_w64(sum <= room_for);
            const int wave_last = 63 - __builtin_clzll(one | 1);
            if ((tid & 63) == 0 && one) atomicMax(&last_bin[part], 2 * (tid + wave_last) + (int)(both >> wave_last & 1));
        }
        lds_barrier();
        int cover[2];
        float least[2];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            cover[part] = last_bin[part] < 0 ? grid.top + 1 : grid.least(last_bin[part]);
            least[part] = fmaxf(least_of(r, cover[part]), -FLT_MAX);
        }
        u64* const list = a.list + ((size_t)row * a.chunks + c) * kSampleListed;
        unsigned here[2] = {0, 0}, at[2];
#pragma unroll
        for (int i = 0; i < kSampleItems; ++i) here[0] += v[i] >= least[0], here[1] += v[i] >= least[1];
        here[1] -= here[0];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const unsigned before = wave_inclusive_sum(here[part]);
            unsigned base = 0;
            if ((tid & 63) == 63) base = atomicAdd(&n_listed[part], before);
            at[part] = (part ? kSampleList : 0) + (unsigned)__builtin_amdgcn_readlane((int)base, 63) + before - here[part];
        }
#pragma unroll
        for (int i = 0; i < kSampleItems; ++i)
        {   // (without a branch: a lane that has none writes to a spare place of its own)
            const bool top = v[i] >= least[0], any = v[i] >= least[1];
            const unsigned to = min(top ? at[0] : at[1], kSampleListed - 1u);
            hist[any ? to : kSampleListed + (tid & 63)] = (u64)__float_as_uint(v[i]) << 32 | index(i);
            at[0] += top, at[1] += any & !top;
        }
        lds_barrier();
        const unsigned n_first = min(n_listed[0], (unsigned)kSampleList), n_more = min(n_listed[1], (unsigned)kSampleMore);
        for (unsigned i = tid; i < kSampleList + n_more; i += kSampleThreads)
            if (i < n_first || i >= kSampleList) list[i] = place_of(__uint_as_float((uint32_t)(hist[i] >> 32)), (unsigned)hist[i]);
        if (tid == 0) out->cover[0] = cover[0], out->cover[1] = cover[1], out->listed[0] = n_first, out->listed[1] = n_more;
    }
    if (tid == 0) out->weight = weight, out->top = grid.top, out->most = most, out->first = 0, out->count = all_count;
}

// ---- the second: a row -------------------------------------------------------------------------------------------
// The chunks' histograms added up say down to which bin there are tokens that may be kept. Mostly they are few: those of the chunks' lists, which are put in order by counting.
// Else the bins of the cuts are sorted out by themselves, by 512 ranges of places at a time, from lists of their tokens or, where even a bin has more than the list has room for, from the row.
// A chain of short steps by one workgroup a row, mostly waits: 13 us for 64 rows of 16 chunks that keep a few (30 000 cycles: what the chunks left 4 500, their histograms added up 6 500,
// the lists' tokens 5 000, the two orders 7 000), 25 for a thousand by their order in the list, 37 to 50 for thousands by top-p (a bin's tokens from the row 25 000 cycles, the cut 13 000, the
// draw 13 000). Rows past the bins are read from the first token on for their largest, for each cut and for what is kept: one of 131 072 111 to 640 us. Rows whose bins have more than the list holds (131 072 logits within a hundredth of the temperature) 230 and more: they are read again for each of some four cuts.
struct PickShared {
    SampleTable table;
    double eighth[8];                      // what a bin weighs more than the first of its eight
    u64 room[kPickWaves];
    u64 chunk_mass[kSampleMaxChunks];
    unsigned light[kSampleMaxChunks / 32];  // a bit of each chunk: it has kept tokens that count nothing
    int top[kSampleMaxChunks], cover[2][kSampleMaxChunks];
    unsigned listed[2][kSampleMaxChunks];  // the first + 1; 0: a chunk without tokens
    unsigned count[kSampleBins + kWave];   // of the bins, then of all up to them
    u64 mass[kSampleBins + kWave];
    unsigned sub_count[kPickSubs];
    u64 sub_mass[kPickSubs];
    u64 few[kPickFew], few_mass[kPickFew], few_upto[kPickFew], by_index[kPickFew], index_upto[kPickFew];
    unsigned rank_of[kPickFew];
    u64 list[kPickList];                   // places
    unsigned n, found;
    u64 lo, hi, cut, before;
    unsigned rank, n_ahead;
    int k_bin, p_bin, m_bin;
};

template <bool BF16>
struct Pick {
    const SampleArgs& a;
    const SampleRow r;
    PickShared& sh;
    const int row;
    const SampleGrid grid;
    double least;                          // weight that min-p keeps
    float base;                            // SampleEnd's
    static constexpr int N = Logits<BF16>::N;
    // The weight of a logit, that of the top bin's beginning being one.
    __device__ __forceinline__ double weight_of(float x) const {
        const float t = place_in(r, x, base), floor_t = floorf(t);
        return rounded_in(r, t - floor_t) * (sh.table.of(grid.top - (int)floor_t) * (1 / kBinOne));
    }
    // The logarithm of a share; past the table, where a weight is none, by the logits themselves.
    __device__ __forceinline__ float log_share(float x, double weight, double whole, float most) const {
        if (weight > 0.0) return (float)log(weight / whole);
        return (float)(((double)x - (double)most) * r.inv_h * r.a - log(whole / weight_of(most)));
    }
    // f(x, index) of all of a row's; then done(first token) after every piece that the workgroup's threads have together: of one chunk.
    template <class F, class D>
    __device__ __forceinline__ void row_each(F f, D done) const {
        constexpr int kLoads = 4;
        for (int from = 0; from < a.vocab; from += kLoads * N * kPickThreads) {
            Logits<BF16> v[kLoads];
            load_logits(v, a.logits, (long long)row * a.stride, from, N * (int)threadIdx.x, N * kPickThreads, a.vocab);
#pragma unroll 1
            for (int j = 0; j < kLoads; ++j) {
                Logits<BF16> one = v[0];
#pragma unroll
                for (int k = 1; k < kLoads; ++k)
                    if (j == k) one = v[k];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float x = logit(r, one[i]);
                    if (x != -INFINITY) f(x, (unsigned)(from + N * ((int)threadIdx.x + j * kPickThreads) + i));
                }
                done(from + N * j * kPickThreads);
            }
        }
    }
    // A wave's chunks' lists: of the first two of its chunks, asked for when the kernel begins.
    static constexpr int kEarly = 2, kListed = kSampleList / kWave;
    struct Lists {
        u64 p[kEarly][kListed];
    };
    __device__ __forceinline__ void list_of(int c, u64 (&p)[kListed]) const {
        const u64* const from = a.list + ((size_t)row * a.chunks + min(c, a.chunks - 1)) * kSampleListed;
#pragma unroll
        for (int i = 0; i < kListed; ++i) p[i] = from[(threadIdx.x & 63) + kWave * i];
    }
    // The places of the tokens of bins lo .. hi into the list, in no order: from the chunks' lists, or from the chunks that have more of them.
    __device__ __forceinline__ void gather(int lo, int hi, const Lists& early) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        lds_barrier();
        if (threadIdx.x == 0) sh.n = 0;
        lds_barrier();
        const auto put = [&](u64 place) {
            const unsigned at = atomicAdd(&sh.n, 1u);
            if (at < kPickList) sh.list[at] = place;
        };
        const auto use = [&](u64 p, bool is) {
            const int b = bin_of(r, logit_of(p));
            if (is && b >= lo && b <= hi) put(p);
        };
        // which chunks have such tokens, and where: a lane has one
        u64 raw[kSampleMaxChunks / kWave] = {};
#pragma unroll
        for (int base = 0; base < kSampleMaxChunks; base += kWave) {
            if (base >= a.chunks) continue;
            const int c = base + lane;
            const unsigned listed = sh.listed[0][c], more = sh.listed[1][c];
            const bool has = c < a.chunks && listed != 0 && sh.top[c] >= lo, both = sh.cover[1][c] <= lo, first = sh.cover[0][c] <= lo;
            raw[base / kWave] = __builtin_amdgcn_ballot_w64(has && !both);
            // the wave's own of those that are listed: every eighth
            const u64 mine = 0x0101010101010101ull << wave;
            const u64 lists = __builtin_amdgcn_ballot_w64(has && both) & mine, seconds = __builtin_amdgcn_ballot_w64(has && both && !first) & mine;
            static_assert(kPickWaves == 8, "every eighth chunk is a wave's");
            if (base == 0) {
#pragma unroll
                for (int k = 0; k < kEarly; ++k) {
                    const int at = wave + k * kPickWaves;
                    if (lists >> at & 1) {
                        const unsigned n = (unsigned)__builtin_amdgcn_readlane((int)listed, at) - 1;
#pragma unroll
                        for (int i = 0; i < kListed; ++i) use(early.p[k][i], (unsigned)(lane + kWave * i) < n);
                    }
                }
            }
            for (u64 left = base == 0 ? lists >> (kEarly * kPickWaves) << (kEarly * kPickWaves) : lists; left; left &= left - 1) {
                const int at = __builtin_ctzll(left);
                const unsigned n = (unsigned)__builtin_amdgcn_readlane((int)listed, at) - 1;
                u64 p[kListed];
                list_of(base + at, p);
#pragma unroll
                for (int i = 0; i < kListed; ++i) use(p[i], (unsigned)(lane + kWave * i) < n);
            }
            for (u64 left = seconds; left; left &= left - 1) {
                const int at = __builtin_ctzll(left);
                const unsigned n = (unsigned)__builtin_amdgcn_readlane((int)more, at);
                const u64* const from = a.list + ((size_t)row * a.chunks + base + at) * kSampleListed + kSampleList;
                constexpr int kEach = kSampleMore / kWave;
                u64 p[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) p[i] = from[kWave * i + lane];
#pragma unroll
                for (int i = 0; i < kEach; ++i) use(p[i], (unsigned)(kWave * i + lane) < n);
            }
        }
        // the chunks that have more than is listed, by all threads, four of them on their way at once
        // (as they are: a NaN is in no range, what counts as the most is in the top bin, past which nothing is: a NaN)
        const float least_x = fmaxf(least_of(r, lo), __uint_as_float(__float_as_uint(-r.most) - 1)), past_x = hi >= grid.top ? __uint_as_float(0x7fc00000u) : least_of(r, hi + 1);
        constexpr int kChunks = 4, kLoads = kSampleChunk / (N * kPickThreads);
#pragma unroll 1
        for (int c0 = 0; c0 < a.chunks; c0 += kChunks) {
            u64 of = raw[0];
#pragma unroll
            for (int w = 1; w < kSampleMaxChunks / kWave; ++w) of = c0 / kWave == w ? raw[w] : of;
            if ((of >> (c0 % kWave) & ((1 << kChunks) - 1)) == 0) continue;
            Logits<BF16> v[kChunks * kLoads];
            load_logits(v, a.logits, (long long)row * a.stride, c0 * kSampleChunk, N * (int)threadIdx.x, N * kPickThreads, a.vocab);
            // which of a lane's are: a word's first in its top bit; few, mostly, so that those are read again by themselves rather than looked for among registers
            static_assert(kChunks == 4 && kLoads * N == 16, "two words of two chunks");
            uint32_t got[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < kChunks * kLoads * N; ++i) {
                const float x = v[i / N][i % N];
                got[i >> 5] = 2 * got[i >> 5] + (x >= least_x && !(x >= past_x) ? 1u : 0u);
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const unsigned asked = (unsigned)(of >> ((c0 + 2 * w) % kWave));
                got[w] &= (asked & 1 ? 0xffff0000u : 0u) | (asked & 2 ? 0xffffu : 0u);
            }
            while (__builtin_amdgcn_ballot_w64((got[0] | got[1]) != 0) != 0) {
                constexpr int kAgain = 4;
                int index[kAgain];
                float x[kAgain];
                unsigned here = 0;
#pragma unroll
                for (int q = 0; q < kAgain; ++q) {
                    const int w = got[0] ? 0 : 1;
                    const uint32_t left = w ? got[1] : got[0];
                    const int i = 32 * w + (left ? __builtin_clz(left) : 0);
                    index[q] = left ? (c0 + (i >> 4)) * kSampleChunk + N * ((int)threadIdx.x + ((i & 15) / N) * kPickThreads) + i % N : 0;
                    here += left ? 1u : 0u;
                    const uint32_t rest = left & ~(0x80000000u >> (i & 31));
                    got[0] = w ? 0u : rest, got[1] = w ? rest : got[1];
                    x[q] = Logits<BF16>::one(a.logits, (long long)row * a.stride + index[q]);
                }
                const unsigned before = wave_inclusive_sum(here);
                unsigned base = 0;
                if (lane == 63) base = atomicAdd(&sh.n, before);
                const unsigned at = (unsigned)__builtin_amdgcn_readlane((int)base, 63) + before - here;
#pragma unroll
                for (int q = 0; q < kAgain; ++q)
                    if ((unsigned)q < here && at + q < kPickList) sh.list[at + q] = place_of(logit(r, x[q]), (unsigned)index[q]);
            }
        }
        lds_barrier();
        if (threadIdx.x == 0) sh.n = min(sh.n, (unsigned)kPickList);
        lds_barrier();
    }
    // f(place) of the tokens of bins lo .. hi: those in the list, or all of the row's.
    template <class F>
    __device__ __forceinline__ void each(bool listed, int lo, int hi, F f) const {
        if (listed) {
            for (unsigned i = threadIdx.x; i < sh.n; i += kPickThreads) {
                const int b = bin_of(r, logit_of(sh.list[i]));
                if (b >= lo && b <= hi) f(sh.list[i]);
            }
        } else {
            row_each([&](float x, unsigned i) { f(place_of(x, i)); }, [](int) {});
        }
    }
    // Up to kPickFew unlike keys, the largest first, with the masses of theirs (a thread has its own key's) and the sums of those up to each. A key's number is
    // that of the keys above it: a thread compares two of them, or four where there are more, with a quarter of all.
    template <int K>
    __device__ __forceinline__ void count_above(int n, int rounds, const u64* keys) const {
        const int part = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 7), first = threadIdx.x & 127;
        u64 its[K];
        unsigned above[K] = {};
#pragma unroll
        for (int i = 0; i < K; ++i) its[i] = keys[min(first + 128 * i, 32 * rounds - 1)];
#pragma unroll 1
        for (int j = 0; j < rounds; ++j) {
            u64 k[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) k[i] = keys[32 * j + 8 * part + i];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int t = 0; t < K; ++t) above[t] += k[i] > its[t];
        }
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (first + 128 * i < n) atomicAdd(&sh.rank_of[first + 128 * i], above[i]);
    }
    __device__ __forceinline__ void order(int n, u64* keys, u64 mass, u64* sorted, u64* sorted_mass, u64* upto) const {
        const int tid = threadIdx.x;
        static_assert(kPickThreads == 512 && kPickFew == 512, "four keys a thread at most, four parts");
        const int rounds = (n + 31) / 32;
        if (tid >= n && tid < 32 * rounds) keys[tid] = 0;  // above none
        sh.rank_of[tid] = 0;
        lds_barrier();
        const u64 own = tid < n ? keys[tid] : 0;
        if (n <= 256) count_above<2>(n, rounds, keys);
        else count_above<4>(n, rounds, keys);
        lds_barrier();
        if (tid < n) {
            const unsigned at = sh.rank_of[tid];
            sorted[at] = own, sorted_mass[at] = mass;
        }
        lds_barrier();
        if (tid < kWave) {
            constexpr int kEach = kPickFew / kWave;
            u64 m[kEach], sum = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) m[i] = kEach * tid + i < n ? sorted_mass[kEach * tid + i] : 0, sum += m[i];
            u64 run = wave_upto(sum) - sum;
#pragma unroll
            for (int i = 0; i < kEach; ++i) upto[kEach * tid + i] = run += m[i];
        }
        lds_barrier();
    }
    // The cut among those: the place of the rank-th, or (by mass) of the last whose tokens before it weigh less than `left`; and what they weigh up to
    // it. Places are sorted out by 512 ranges at a time until few are left, which are compared with each other.
    __device__ __forceinline__ void resolve(bool listed, int b_lo, int b_hi, bool by_mass, unsigned rank, u64 left, u64& cut, u64& upto) const {
        const int tid = threadIdx.x;
        u64 most = 0, least_place = 0;  // (the second inverted)
        unsigned n = 0;
        each(listed, b_lo, b_hi, [&](u64 p) { most = max(most, p), least_place = max(least_place, ~p), ++n; });
        u64 hi = all_most<kPickWaves>(most, sh.room), lo = ~all_most<kPickWaves>(least_place, sh.room);
        n = (unsigned)all_sum<kPickWaves>(n, sh.room);
        u64 before = 0;
        unsigned ahead = 0;
        while (n > kPickFew) {
            const u64 span = hi - lo;
            const int bits = 64 - __builtin_clzll(span | 1), shift = bits > 9 ? bits - 9 : 0;
            static_assert(kPickSubs == 1 << 9 && kPickSubs == kPickThreads, "a thread's each");
            lds_barrier();
            sh.sub_count[tid] = 0, sh.sub_mass[tid] = 0;
            if (tid == 0) sh.rank = ~0u;
            lds_barrier();
            each(listed, b_lo, b_hi, [&](u64 p) {
                if (p < lo || p > hi) return;
                const int s = (int)((hi - p) >> shift);
                atomicAdd(&sh.sub_count[s], 1u);
                atomicAdd(&sh.sub_mass[s], mass_of(weight_of(logit_of(p))));
            });
            lds_barrier();
            const unsigned dk = sh.sub_count[tid];
            const u64 dm = sh.sub_mass[tid];
            unsigned k_at = wave_inclusive_sum(dk);
            u64 m_at = wave_upto(dm);
            if ((tid & 63) == 63) sh.few[tid >> 6] = k_at, sh.few_mass[tid >> 6] = m_at;
            lds_barrier();
            unsigned k_all = 0;
            u64 m_all = 0;
#pragma unroll
            for (int w = 0; w < kPickWaves; ++w) {
                if (w < tid >> 6) k_at += (unsigned)sh.few[w], m_at += sh.few_mass[w];
                k_all += (unsigned)sh.few[w], m_all += sh.few_mass[w];
            }
            // the sub-bin of the cut: the first up to which there is enough; the last that has a token where there never is
            const bool never = by_mass && before + m_all < left;
            const bool hit = never ? dk && k_at == k_all
                                   : by_mass ? dk && before + m_at >= left && (before + m_at - dm < left || k_at == dk) : k_at - dk + ahead < rank && k_at + ahead >= rank;
            if (hit) atomicMin(&sh.rank, (unsigned)tid);
            lds_barrier();
            if ((unsigned)tid == sh.rank) {
                const u64 size = (1ull << shift) - 1;
                sh.hi = hi - ((u64)tid << shift);
                sh.lo = sh.hi - lo > size ? sh.hi - size : lo;
                sh.before = m_at - dm, sh.found = dk, sh.n_ahead = k_at - dk;
            }
            lds_barrier();
            hi = sh.hi, lo = sh.lo, before += sh.before, ahead += sh.n_ahead, n = sh.found;
        }
        lds_barrier();
        if (tid == 0) sh.found = 0;
        lds_barrier();
        each(listed, b_lo, b_hi, [&](u64 p) {
            if (p < lo || p > hi) return;
            const unsigned k = atomicAdd(&sh.found, 1u);
            if (k < kPickFew) sh.few[k] = p, sh.few_mass[k] = mass_of(weight_of(logit_of(p)));
        });
        lds_barrier();
        order((int)n, sh.few, tid < (int)n ? sh.few_mass[tid] : 0, sh.by_index, sh.sub_mass, sh.few_upto);
        // the last that stays (the first does whatever it takes: it is where the cut is)
        const auto stays = [&](unsigned t) { return t < n && (t == 0 || (by_mass ? before + sh.few_upto[t - 1] < left : ahead + t < rank)); };
        if (stays(tid) && !stays(tid + 1)) sh.cut = sh.by_index[tid], sh.before = sh.few_upto[tid];
        lds_barrier();
        cut = sh.cut, upto = before + sh.before;
        lds_barrier();
    }
};

template <bool BF16>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(const SampleArgs a) {
    __shared__ PickShared sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    const SampleChunk* const chunks = a.chunk + (size_t)row * a.chunks;
    SampleChunk mine{0, 0, {0, 0}, -INFINITY, 0, 0, {0, 0}};
    if (tid < a.chunks) mine = chunks[tid];
    SampleRow r = sample_row(a, row);
    const float u = a.uniforms[row];
    // What the chunks have left, all on its way before anything is waited for: their histograms' words of the thread's bin, sixteen chunks at once, and their lists.
    constexpr int kAtOnce = 16;
    const bool weighed = r.weighed(), asks = r.filtered() && !r.greedy;
    u64 masses[kAtOnce];
    unsigned counts[kAtOnce];
    const auto words_of = [&](int c0) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) counts[j] = a.counts[((size_t)row * a.chunks + min(c0 + j, a.chunks - 1)) * kSampleBins + tid];
        if (weighed) {
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) masses[j] = a.masses[((size_t)row * a.chunks + min(c0 + j, a.chunks - 1)) * kSampleBins + tid];
        }
    };
    typename Pick<BF16>::Lists lists;
    if (asks) {
        words_of(0);
        const Pick<BF16> early{a, r, sh, row, SampleGrid(0), 0.0, 0.0f};
#pragma unroll
        for (int k = 0; k < Pick<BF16>::kEarly; ++k) early.list_of((tid >> 6) + k * kPickWaves, lists.p[k]);
    }
    make_table(sh.table, r);
    if (tid >= 128 && tid < 136) sh.eighth[tid - 128] = exp(r.a * (double)(tid - 128));
    sh.count[tid] = 0, sh.mass[tid] = 0;
    if (tid < kSampleMaxChunks) {
        sh.chunk_mass[tid] = 0;
        sh.top[tid] = mine.top, sh.cover[0][tid] = mine.cover[0], sh.cover[1][tid] = mine.cover[1];
        sh.listed[0][tid] = mine.count ? mine.listed[0] + 1 : 0, sh.listed[1][tid] = mine.listed[1];
    }
    if (tid < kSampleMaxChunks / 32) sh.light[tid] = 0;
    if (tid == 0) sh.n = 0, sh.k_bin = sh.p_bin = sh.m_bin = kSampleBins;
    u64 best = wave_most64(mine.count ? place_of(mine.most, (unsigned)mine.first) : 0);
    unsigned candidates = (unsigned)wave_sum64(mine.count);
    if ((tid & 63) == 0) sh.few[tid >> 6] = best, sh.room[tid >> 6] = candidates;
    lds_barrier();
    best = 0, candidates = 0;
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w) best = max(best, sh.few[w]), candidates += (unsigned)sh.room[w];
    lds_barrier();
    const auto finish = [&](int token, unsigned kept, float logprob, const SampleEnd& end) {
        a.tokens[row] = token;
        if (a.n_kept) a.n_kept[row] = (int)kept;
        if (a.logprobs) a.logprobs[row] = logprob;
        a.end[row] = end;
    };
    if (candidates == 0) {
        if (tid == 0) finish(-1, 0, -INFINITY, SampleEnd{0, 0, 0, -1, 0, 0});
        return;
    }
    if (r.greedy) {
        if (tid == 0) finish((int)index_of(best), 1, 0.0f, SampleEnd{0, 0, 0, (int)index_of(best), 1, 0});
        return;
    }
    float most = logit_of(best);
    // Past the bins: the largest logit out of the row, and nothing of what the chunks left but their numbers of tokens.
    const bool far = most >= r.most;
    if (far) {
        r.cap = FLT_MAX;
        const Pick<BF16> look{a, r, sh, row, SampleGrid(0), 0.0, 0.0f};
        u64 top = 0;
        look.row_each([&](float x, unsigned i) { top = max(top, place_of(x, i)); }, [](int) {});
        most = logit_of(all_most<kPickWaves>(top, sh.room));
    }
    Pick<BF16> pick{a, r, sh, row, SampleGrid(far ? 0 : bin_of(r, most)), 0.0, far ? most : 0.0f};
    const SampleGrid& grid = pick.grid;
    if (r.m_on) pick.least = r.m * pick.weight_of(most);
    u64 cut = 0;
    unsigned kept = candidates;
    double whole_weight = 0.0;             // of what is kept, where it is had but as a whole number
    if (!r.filtered() && !far) {
        const double weight = mine.count ? mine.weight * sh.table.of(grid.top - mine.top) : 0.0;
        if (mine.count) sh.chunk_mass[tid] = max((u64)(weight * kMassOne + 0.5), 1ull);  // (every chunk that has tokens is found by some u)
        const double of_wave = wave_sum_f64(weight);
        if ((tid & 63) == 0) sh.few[tid >> 6] = __builtin_bit_cast(u64, of_wave);
        lds_barrier();
#pragma unroll
        for (int w = 0; w < kPickWaves; ++w) whole_weight += __builtin_bit_cast(double, sh.few[w]);
    } else {
        // ---- the row's histogram
        // (no branches: what has no bin goes to spare ones, a lane's own)
        for (int c0 = 0; !far;) {
            // (a chunk's top is a scalar)
            const int top_of = sh.top[min(c0 + (tid & (kAtOnce - 1)), kSampleMaxChunks - 1)];
            const unsigned there_of = sh.listed[0][min(c0 + (tid & (kAtOnce - 1)), kSampleMaxChunks - 1)];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const SampleGrid of(__builtin_amdgcn_readlane(top_of, j));
                const bool there = c0 + j < a.chunks && __builtin_amdgcn_readlane((int)there_of, j) != 0;
                const int b = of.least(tid), number = grid.of(b);
                const bool in = there && counts[j] != 0 && number < kSampleBins;
                const int to = in ? number : kSampleBins + (tid & 63);
                atomicAdd(&sh.count[to], counts[j]);
                if (weighed) {
                    u64 m = masses[j];
                    if (in && tid < kFine && number >= kFine) m = scaled(m, sh.eighth[b & 7]);
                    atomicAdd(&sh.mass[to], m);
                }
            }
            c0 += kAtOnce;
            if (c0 >= a.chunks) break;
            words_of(c0);
        }
        lds_barrier();
        // sums up to each bin
        unsigned count = sh.count[tid];
        const unsigned count_of = count;
        u64 mass = weighed ? scaled(sh.mass[tid], sh.table.of(grid.top - grid.least(tid)) * (kMassOne / kBinOne)) : 0;
        const u64 mass_of_bin = mass;
        count = wave_inclusive_sum(count);
        if (weighed) mass = wave_upto(mass);
        if ((tid & 63) == 63) sh.few[tid >> 6] = count, sh.few_mass[tid >> 6] = mass;
        lds_barrier();
        u64 total = 0;
#pragma unroll
        for (int w = 0; w < kPickWaves; ++w) {
            if (w < tid >> 6) count += (unsigned)sh.few[w], mass += sh.few_mass[w];
            total += sh.few_mass[w];
        }
        sh.count[tid] = count, sh.mass[tid] = mass;
        // the first bins up to which there is enough, none being the tail; the first whose beginning is too light for min-p
        // (a k of more tokens than there are cuts nothing, but stands for the weights that the histogram has not)
        const unsigned k = min((unsigned)r.k, candidates);
        const bool by_k = r.k_on && (k < candidates || !weighed);
        const auto share = [&](u64 of) -> u64 { return max((u64)ceil(r.p * (double)of), 1ull); };
        if (by_k && count - count_of < k && count >= k) sh.k_bin = tid;
        if (!by_k && r.p_on && mass - mass_of_bin < share(total) && mass >= share(total)) sh.p_bin = tid;
        const auto light = [&](int i) { return sh.table.of(grid.top - grid.least(i)) < pick.least; };
        if (r.m_on && !far && light(tid) && (tid == 0 || !light(tid - 1))) sh.m_bin = tid;
        lds_barrier();
        const int k_bin = sh.k_bin, m_bin = sh.m_bin;
        int p_bin = sh.p_bin;
        // the lowest that may have a kept token, or one whose weight is asked for: what the first k weigh is, by top-p, wherever min-p ends
        const int depth = by_k ? (r.p_on ? k_bin : min(k_bin, m_bin)) : min(p_bin, m_bin);
        const unsigned deep = depth < kSampleBins ? sh.count[depth] : ~0u;
        const auto count_in = [&](int b) { return b >= kSampleBins ? ~0u : sh.count[b] - (b ? sh.count[b - 1] : 0u); };
        if (deep <= kPickList) pick.gather(grid.least(depth), INT_MAX, lists);
        if (deep <= (r.k_on || r.p_on ? kPickInOrder : kPickInOrderByM)) {
            // ---- few: in order, with what they weigh up to each
            const int n = (int)sh.n;
            pick.order(n, sh.list, tid < n ? mass_of(pick.weight_of(logit_of(sh.list[tid]))) : 0, sh.few, sh.few_mass, sh.few_upto);
            // thread t has the t-th
            if (by_k && r.p_on) total = sh.few_upto[min(n, (int)k) - 1];
            const auto stays = [&](int t) {
                if (t >= n || (by_k && t >= (int)k)) return false;
                if (t == 0) return true;
                return (!r.p_on || sh.few_upto[t - 1] < share(total)) && (!r.m_on || pick.weight_of(logit_of(sh.few[t])) >= pick.least);
            };
            const bool mine_stays = stays(tid);
            if (mine_stays && !stays(tid + 1)) sh.rank = tid + 1, sh.cut = sh.few[tid], sh.before = sh.few_upto[tid];
            // those by their indexes, with their numbers
            if (mine_stays) sh.list[tid] = (u64)(kSampleMaxVocab - 1 - index_of(sh.few[tid])) << 9 | (u64)tid;
            lds_barrier();
            kept = sh.rank;
            const u64 all = sh.before;
            const double of_wave = wave_sum_f64(mine_stays ? pick.weight_of(logit_of(sh.few[tid])) : 0.0);
            if ((tid & 63) == 0) sh.room[tid >> 6] = __builtin_bit_cast(u64, of_wave);
            pick.order((int)kept, sh.list, mine_stays ? sh.few_mass[tid] : 0, sh.by_index, sh.sub_mass, sh.index_upto);
            if (tid < (int)kept) {
                const double target = (double)u * (double)all;
                const u64 upto = sh.index_upto[tid], before = tid ? sh.index_upto[tid - 1] : 0;
                // the first whose sum is past the target, by a u of none the first whatever it weighs; where none's is, the last
                if (u <= 0.0f ? tid == 0 : (double)all > target ? (double)upto > target && !((double)before > target) : tid == (int)kept - 1) {
                    const u64 p = sh.few[sh.by_index[tid] & (kPickFew - 1)];
#pragma unroll
                    for (int w = 0; w < kPickFew / kWave; ++w) whole_weight += __builtin_bit_cast(double, sh.room[w]);
                    finish((int)index_of(p), kept, pick.log_share(logit_of(p), pick.weight_of(logit_of(p)), whole_weight, most), SampleEnd{1.0 / whole_weight, sh.cut, grid.top, (int)index_of(p), 2, 0});
                }
            }
            return;
        }
        // ---- many: the cuts by themselves. From lists of all down to there, or of the cuts' bins alone, or from the row
        const bool whole_list = deep <= kPickList;
        if (far && r.p_on && !by_k) {
            u64 of = 0;
            pick.row_each([&](float x, unsigned) { of += mass_of(pick.weight_of(x)); }, [](int) {});
            total = all_sum<kPickWaves>(of, sh.room);
        }
        const auto mass_before = [&](int b) { return b ? sh.mass[b - 1] : 0ull; };
        int held = -1;                     // the bin that the list is of
        bool by_bins = !whole_list && weighed && depth < kSampleBins && (!by_k || count_in(k_bin) <= kPickList);
        int end_bin = min(by_k ? k_bin : p_bin, m_bin);  // of the cut
#pragma unroll 1
        for (int step = 0; step < 2; ++step) {
            const bool by_mass = step == 1;
            // (a cut below what min-p keeps is none)
            if (by_mass ? !r.p_on || (!by_k && m_bin < p_bin) : !by_k || (!r.p_on && m_bin < k_bin)) continue;
            const u64 want = by_mass ? share(total) : 0;
            if (by_mass && by_k && weighed) {  // (the first bin up to which there is enough)
                lds_barrier();
                if (tid == 0) sh.p_bin = k_bin;
                lds_barrier();
                if (tid < k_bin && sh.mass[tid] >= want && (tid == 0 || sh.mass[tid - 1] < want)) sh.p_bin = tid;
                lds_barrier();
                p_bin = sh.p_bin;
            }
            const int bin = by_mass ? p_bin : k_bin;
            // (a list of all without weights in its histogram: the row's order from its first token on)
            const bool from_bin = weighed && (whole_list || by_bins);
            if (from_bin && by_bins && count_in(bin) > kPickList) by_bins = false;
            const bool binned = from_bin && (whole_list || by_bins);
            if (binned && by_bins && held != bin) pick.gather(grid.least(bin), bin < kFine ? grid.least(bin) : grid.least(bin) + 7, lists), held = bin;
            const int lo = binned ? grid.least(bin) : INT_MIN, hi = binned ? (bin < kFine ? lo : lo + 7) : INT_MAX;
            const u64 ahead = binned ? mass_before(bin) : 0;
            const unsigned k_ahead = binned && bin ? sh.count[bin - 1] : 0;
            u64 upto, its_cut;
            pick.resolve(whole_list || binned, lo, hi, by_mass, k - k_ahead, by_mass ? (want > ahead ? want - ahead : 1) : 0, its_cut, upto);
            cut = max(cut, its_cut);
            if (!by_mass) total = ahead + upto;
            end_bin = min(end_bin, by_mass ? p_bin : k_bin);
        }
        lds_barrier();
        if (by_bins && (end_bin >= kSampleBins || count_in(end_bin) > kPickList)) by_bins = false;
        // ---- what is kept, by chunk
        unsigned n = 0;
        u64 end = 0;                       // (inverted: the last kept token's place)
        const auto keep = [&](u64 p, u64& mass) -> bool {
            if (p < cut) return false;
            const double w = pick.weight_of(logit_of(p));
            if (w < pick.least) return false;
            ++n, end = max(end, ~p), mass = mass_of(w);
            return true;
        };
        const auto found_light = [&](int c) { atomicOr(&sh.light[c >> 5], 1u << (c & 31)); };
        if (by_bins) {
            // bins in front of the cut's out of the histograms; its own tokens one by one
            if (held != end_bin) pick.gather(grid.least(end_bin), end_bin < kFine ? grid.least(end_bin) : grid.least(end_bin) + 7, lists);
            for (int c = tid >> 6; c < a.chunks; c += kPickWaves) {
                if (sh.listed[0][c] == 0) continue;
                const SampleGrid of(sh.top[c]);
                u64 sum = 0;
                bool some = false;
                for (int i = tid & 63; i < kSampleBins; i += kWave) {
                    const u64 v = a.masses[((size_t)row * a.chunks + c) * kSampleBins + i];
                    const bool in = v && grid.of(of.least(i)) < end_bin;
                    if (in) sum += scaled(v, sh.table.of(grid.top - of.least(i)) * (kMassOne / kBinOne));
                    some |= in;
                }
                sum = wave_sum64(sum), some = __builtin_amdgcn_ballot_w64(some) != 0;
                if ((tid & 63) == 0 && sum) atomicAdd(&sh.chunk_mass[c], sum);
                if ((tid & 63) == 0 && some && !sum) found_light(c);
            }
        }
        if (whole_list || by_bins) {
            for (unsigned i = tid; i < sh.n; i += kPickThreads) {
                u64 m;
                if (!keep(sh.list[i], m)) continue;
                const int c = (int)(index_of(sh.list[i]) / kSampleChunk);
                if (m) atomicAdd(&sh.chunk_mass[c], m);
                else found_light(c);
            }
        } else {
            u64 piece = 0;
            bool some = false;
            pick.row_each([&](float x, unsigned i) {
                u64 m;
                if (keep(place_of(x, i), m)) piece += m, some = true;
            }, [&](int from) {
                piece = wave_sum64(piece), some = __builtin_amdgcn_ballot_w64(some) != 0;
                if (piece && (tid & 63) == 0) atomicAdd(&sh.chunk_mass[from / kSampleChunk], piece);
                if (some && !piece && (tid & 63) == 0) found_light(from / kSampleChunk);
                piece = 0, some = false;
            });
        }
        kept = (unsigned)all_sum<kPickWaves>(n, sh.room) + (by_bins && end_bin ? sh.count[end_bin - 1] : 0u);
        const u64 last = all_most<kPickWaves>(end, sh.room);
        // (none of the cut's bin kept, by min-p: whatever is in the bins in front of it is)
        cut = last ? ~last : place_of(least_of(r, grid.least(end_bin - 1)), kSampleMaxVocab - 1);
    }
    // ---- the chunk that the draw falls into, in every wave: a lane has four. Chunks' masses are other roundings than their tokens': of the bins' sums, or of the
    // chunk's; and a chunk that has kept tokens counts as one at least, so that the first and the last of them are in the first and the last chunk that counts.
    u64 mass[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = 4 * (tid & 63) + i;
        mass[i] = sh.chunk_mass[c];
        if (mass[i] == 0) mass[i] = sh.light[c >> 5] >> (c & 31) & 1;
        sum += mass[i];
    }
    u64 run = wave_upto(sum);
    const u64 all = ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(run >> 32), 63) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)run, 63);
    run -= sum;
    const double target = (double)u * (double)all;
    int c = -1, last_c = -1;
    u64 run_c = 0, run_last = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (mass[i]) {
            if (c < 0 && (double)(run + mass[i]) > target) c = 4 * (tid & 63) + i, run_c = run;
            last_c = 4 * (tid & 63) + i, run_last = run;
        }
        run += mass[i];
    }
    const u64 hits = __builtin_amdgcn_ballot_w64(c >= 0), lasts = __builtin_amdgcn_ballot_w64(last_c >= 0);
    const int lane = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(lasts);
    c = __builtin_amdgcn_readlane(hits ? c : last_c, lane);
    run_c = __shfl(hits ? run_c : run_last, lane, kWave);
    // ---- the token: by running sums of the chunk's weights as they are. (As whole numbers, weights below 2^-43 are none: in a chunk of nothing else none was ever past the target.)
    constexpr int kEach = kSampleChunk / kPickThreads, N = Logits<BF16>::N;
    float x[kEach];
    double w[kEach], own = 0.0;
    unsigned in = 0;                       // which of a thread's are kept
    const int from = c * kSampleChunk + kEach * tid;
    Logits<BF16> v[kEach / N];
#pragma unroll
    for (int i = 0; i < kEach; i += N) {
        if ((c + 1) * kSampleChunk <= a.vocab) v[i / N].load(static_cast<const char*>(a.logits) + ((long long)row * a.stride + c * kSampleChunk + i) * (BF16 ? 2 : 4), (unsigned)(kEach * tid));
        else v[i / N].some(a.logits, (long long)row * a.stride, from + i, a.vocab);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = logit(r, v[i / N][i % N]);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const bool kept_one = x[i] != -INFINITY && place_of(x[i], (unsigned)(from + i)) >= cut;
        in |= kept_one ? 1u << i : 0u;
        w[i] = kept_one ? pick.weight_of(x[i]) : 0.0;
        own += w[i];
    }
    // the threads' sums in order
    const double upto = wave_upto_f64(own);
    lds_barrier();
    if ((tid & 63) == 63) sh.room[tid >> 6] = __builtin_bit_cast(u64, upto);
    lds_barrier();
    const double lane_before = __shfl(upto, (tid & 63) - 1, kWave);  // (of the first lane: not used)
    double before = 0.0, whole_chunk = 0.0;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) {
        if (i == tid >> 6) before = whole_chunk;
        whole_chunk += __builtin_bit_cast(double, sh.room[i]);
    }
    if ((tid & 63) != 0) before += lane_before;
    // What a sum has to be past: less than the chunk's own, whichever rounding found the chunk; nothing where u is none, so that the first is drawn whatever it weighs; more than
    // any where no chunk was past the target.
    const double past = u <= 0.0f ? -1.0 : hits ? fmin((target - (double)run_c) / kMassOne, whole_chunk * (1.0 - 0x1p-40)) : (double)INFINITY;
    int hit = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        before += w[i];
        if (hit < 0 && (in >> i & 1) && before > past) hit = from + i;
    }
    const int last = in ? from + 31 - __builtin_clz(in) : -1;
    // the first hit; where there is none, the last token
    const u64 hit_lanes = __builtin_amdgcn_ballot_w64(hit >= 0), last_lanes = __builtin_amdgcn_ballot_w64(last >= 0);
    const int wave_hit = hit_lanes ? __builtin_amdgcn_readlane(hit, __builtin_ctzll(hit_lanes)) : -1;
    const int wave_last = last_lanes ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(last_lanes)) : -1;
    if ((tid & 63) == 0) sh.few[tid >> 6] = (u64)(uint32_t)wave_hit << 32 | (uint32_t)wave_last;
    lds_barrier();
    int token = -1, last_token = -1;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) {
        const int h = (int)(sh.few[i] >> 32), l = (int)(uint32_t)sh.few[i];
        if (token < 0) token = h;
        if (l >= 0) last_token = l;
    }
    if (token < 0) token = last_token;
    if (token >= from && token < from + kEach) {
        float of = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) of = token - from == i ? x[i] : of;
        // (a whole number's last bits are those of its tokens': where one is nearly all of it, as a whole number too)
        double weight = pick.weight_of(of);
        if (r.filtered() || far) {
            whole_weight = (double)all / kMassOne;
            if (weight > 0.25 * whole_weight) weight = (double)mass_of(weight) / kMassOne;
        }
        finish(token, kept, pick.log_share(of, weight, whole_weight, most), SampleEnd{1.0 / whole_weight, cut, grid.top, token, 2, pick.base});
    }
}

// ---- the third, where probabilities are asked for -------------------------------------------------------------------
// A chunk whose list has all of its tokens that are kept is not read again: zeros, and those of the list over them.
// 256 rows of 131 072 fp32 logits, most of them cut to a few tokens: 31 us, 4.3 TB/s written (all chunks read again: 42).
template <bool BF16>
__global__ __launch_bounds__(kSampleThreads) void sample_probs_kernel(const SampleArgs a) {
    __shared__ SampleTable table;
    constexpr int N = Logits<BF16>::N, kLoads = kSampleItems / N;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks, tid = threadIdx.x;
    const SampleEnd end = a.end[row];
    const SampleChunk of = a.chunk[blockIdx.x];
    SampleRow r = sample_row(a, row);
    const bool far = end.base != 0.0f;     // (the lists and bins are not its logits')
    if (far) r.cap = FLT_MAX;
    float* const out = a.probs + (long long)row * a.probs_stride;
    const float least = end.cut ? logit_of(end.cut) : -FLT_MAX;
    const int cut_bin = bin_of(r, least);
    const bool none = end.kind != 2 || of.count == 0 || (end.cut && !far && of.top < cut_bin);
    const bool listed = none || (end.cut && !far && of.cover[1] <= cut_bin);
    typedef float f32x4v __attribute__((ext_vector_type(4)));
    typedef f32x4v words __attribute__((aligned(4)));
    const auto probability = [&](float x) {
        const float t = place_in(r, x, end.base), floor_t = floorf(t);
        return (float)(rounded_in(r, t - floor_t) * (table.of(end.top - (int)floor_t) * (1 / kBinOne)) * end.inv);
    };
    const auto store = [&](int at, const float* p) {
        if (at + N <= a.vocab) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<words*>(out + at + i) = f32x4v{p[i], p[i + 1], p[i + 2], p[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < a.vocab) out[at + i] = p[i];
        }
    };
    if (listed) {
        constexpr int kEach = (kSampleListed + kSampleThreads - 1) / kSampleThreads;
        u64 p[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int i = tid + k * kSampleThreads;
            const bool is = !none && (i < kSampleList ? i < (int)of.listed[0] : i - kSampleList < (int)of.listed[1]);
            p[k] = is ? a.list[(size_t)blockIdx.x * kSampleListed + i] : 0;
        }
        if (!none) make_table(table, r);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const float zeros[N] = {};
            store(c * kSampleChunk + N * (tid + j * kSampleThreads), zeros);
        }
        __syncthreads();                   // the zeros are there before what comes over them
        if (end.kind == 1 && tid == 0 && (unsigned)end.token < (unsigned)a.vocab && end.token / kSampleChunk == c) out[end.token] = 1.0f;
        if (none) return;
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (p[k] && p[k] >= end.cut) out[index_of(p[k])] = probability(logit_of(p[k]));
        return;
    }
    Logits<BF16> v[kLoads];
    load_logits(v, a.logits, (long long)row * a.stride, c * kSampleChunk, N * tid, N * kSampleThreads, a.vocab);
    make_table(table, r);
    lds_barrier();
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int at = c * kSampleChunk + N * (tid + j * kSampleThreads);
        float p[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = logit(r, v[j][i]);
            p[i] = x >= least && place_of(x, (unsigned)(at + i)) >= end.cut ? probability(x) : 0.0f;
        }
        store(at, p);
    }
}

static size_t sample_chunks(int vocab) { return ((size_t)vocab + kSampleChunk - 1) / kSampleChunk; }
static size_t sample_bytes(int n_rows, int vocab) {
    if (n_rows <= 0 || vocab <= 0 || vocab > kSampleMaxVocab) return 0;
    const size_t chunks = (size_t)n_rows * sample_chunks(vocab);
    return chunks * ((kSampleBins + kSampleListed) * sizeof(u64) + kSampleBins * sizeof(unsigned) + sizeof(SampleChunk)) + (size_t)n_rows * sizeof(SampleEnd);
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
    rk::u64* const masses = static_cast<rk::u64*>(workspace);
    rk::u64* const list = masses + all * rk::kSampleBins;
    unsigned* const counts = reinterpret_cast<unsigned*>(list + all * rk::kSampleListed);
    rk::SampleChunk* const chunk = reinterpret_cast<rk::SampleChunk*>(counts + all * rk::kSampleBins);
    rk::SampleEnd* const end = reinterpret_cast<rk::SampleEnd*>(chunk + all);
    const rk::SampleArgs a{logits, temperatures, top_ps, min_ps, uniforms, top_ks, n_rows, vocab, (int)chunks, stride, probs_stride, tokens, n_kept,
                           logprobs, probs, chunk, masses, list, counts, end};
    return bf16 ? rk::sample_rows<true>(a, (hipStream_t)stream) : rk::sample_rows<false>(a, (hipStream_t)stream);
}
