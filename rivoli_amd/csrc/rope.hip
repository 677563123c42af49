// Rotary positions: the table of (cos, sin) pairs and the rotation of rows by it. The table's layout,
// [position][rd / 2] pairs of f32, is what the compressor's finish reads (rivoli_comp_finish.freqs).
// Launch-only.
#include <cfloat>
#include <cmath>

#include "codec.hpp"

namespace rk {

// ---- the table --------------------------------------------------------------------------------------------
// Pair j turns by p * f_j at position p, f_j = base^(-2j / rd), stretched for a longer context either as a whole
// (f_j / factor) or by parts: pairs that turn often within the original context keep f_j, pairs that turn
// hardly ever have f_j / factor, a ramp over the pairs between (the published NTK-by-parts rule).
// Angles are taken in turns and in 64 bits: at position 10^6 a product's 24 bits would leave 0.06 of a radian. A thread has a pair at
// kTableRun positions at even distances and takes two sines and cosines, of the first angle and of the distance; the others come by
// turning, (c + is)(dc + ids), four 64-bit operations a step whose error, some 10^-16 a step, is nothing to f32.
// 163 840 positions of 32 pairs, 42 MB, 8.7 us (6.1 at a fill's rate; 9.2 by 32 positions a thread; 10.8 with a 32-bit sine and cosine of every reduced angle).
struct RopeTableArgs {
    float* table;
    int first, n, pairs;
    double log2_base, factor, low, high;  // ramp over pairs low .. high; high < 0: every pair is stretched
    double mscale;
};
constexpr int kTableRun = 16;

__global__ __launch_bounds__(256) void rope_table_kernel(const RopeTableArgs a) {
    const unsigned at = blockIdx.x * 256u + threadIdx.x;
    const int j = (int)(at % (unsigned)a.pairs);
    // a run's positions are apart by the number of runs, so that neighbours in the launch are neighbours in memory
    const unsigned run = at / (unsigned)a.pairs, runs = ((unsigned)a.n + kTableRun - 1) / kTableRun;
    if (run >= runs) return;
    double f = exp2(-(double)j / (double)a.pairs * a.log2_base);
    double stretched = 1.0;
    if (a.high >= 0.0) stretched = fmin(1.0, fmax(0.0, ((double)j - a.low) / (a.high - a.low)));
    f = f / a.factor * stretched + f * (1.0 - stretched);
    const double turns = f * 0.15915494309189533577;  // 1 / (2 pi)
    const auto angle = [&](double p, double& s, double& c) {
        double t = p * turns;
        t -= rint(t);  // its whole turns
        sincospi(2.0 * t, &s, &c);
    };
    double s, c, ds, dc;
    angle((double)a.first + (double)run, s, c);
    angle((double)runs, ds, dc);
#pragma unroll 4
    for (int i = 0; i < kTableRun; ++i) {
        const unsigned p = run + (unsigned)i * runs;
        if (p >= (unsigned)a.n) return;
        reinterpret_cast<f32x2*>(a.table)[(size_t)p * a.pairs + j] = f32x2{(float)(c * a.mscale), (float)(s * a.mscale)};
        const double was = c;
        c = c * dc - s * ds, s = was * ds + s * dc;
    }
}

// ---- the rows ---------------------------------------------------------------------------------------------
// (x, y) -> (x c - y s, x s + y c) for the pairs of a head's rd values: neighbours, or half of them apart. Memory
// bound: every value is read and written once, a token's table row serves all of its heads. A thread has one
// piece of up to kRopeHeads heads: 16 bytes of neighbouring pairs, or the 16 bytes of either half that belong together, so
// that rows may be rotated in place. 8 192 tokens of 128 heads, the last 64 of 192 values, 53 us: 270 MB at a large copy's rate.
struct RopeArgs {
    const void* x;
    void* out;
    const float* table;
    const int* positions;
    int n_tokens, n_heads, groups;  // of heads: head g, g + groups, ...
    int rd, pieces, n_positions;
    long long x_token, x_head, out_token, out_head;  // in elements
    unsigned int* bad;
};
constexpr int kRopeHeads = 4;

template <class T>
__device__ __forceinline__ T as_row(float v);
template <>
__device__ __forceinline__ float as_row<float>(float v) { return v; }
template <>
__device__ __forceinline__ __bf16 as_row<__bf16>(float v) { return (__bf16)v; }

// N pairs a piece. Rows whose starts, strides or widths are off the 16 bytes go a pair a piece.
template <class T, bool HALF, int N, int HEADS>
__global__ __launch_bounds__(256) void rope_rows_kernel(const RopeArgs a) {
    constexpr int kVec = HALF ? N : 2 * N;
    typedef T row_vec __attribute__((ext_vector_type(kVec)));
    const unsigned at = blockIdx.x * 256u + threadIdx.x, item = at / (unsigned)a.pieces;
    const int piece = (int)(at - item * (unsigned)a.pieces);
    const unsigned token = item / (unsigned)a.groups;
    const int h0 = (int)(item - token * (unsigned)a.groups);
    if (token >= (unsigned)a.n_tokens) return;
    const int pos = a.positions[token];
    if ((unsigned)pos >= (unsigned)a.n_positions) {
        if (a.bad && piece == 0 && h0 == 0) atomicAdd(a.bad, 1u);
        return;
    }
    const T* const x = static_cast<const T*>(a.x) + (long long)token * a.x_token + (HALF ? piece * N : 2 * piece * N);
    T* const out = static_cast<T*>(a.out) + (long long)token * a.out_token + (HALF ? piece * N : 2 * piece * N);
    const int apart = a.rd / 2;
    row_vec v[HEADS], w[HALF ? HEADS : 1];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {  // (a head past the last re-reads the last)
        const T* const src = x + (long long)min(h0 + k * a.groups, a.n_heads - 1) * a.x_head;
        if constexpr (N == 1) {
            v[k][0] = src[0];
            if constexpr (HALF) w[k][0] = src[apart];
            else v[k][1] = src[1];
        } else {
            v[k] = *reinterpret_cast<const row_vec*>(src);
            if constexpr (HALF) w[k] = *reinterpret_cast<const row_vec*>(src + apart);
        }
    }
    f32x2 turn[N];
    const f32x2* const row = reinterpret_cast<const f32x2*>(a.table) + (size_t)pos * apart + piece * N;
#pragma unroll
    for (int i = 0; i < N; ++i) turn[i] = row[i];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        const int h = h0 + k * a.groups;
        if (h >= a.n_heads) return;
        row_vec p, q;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float c = turn[i].x, s = turn[i].y;
            const float e = (float)(HALF ? v[k][i] : v[k][2 * i]), o = (float)(HALF ? w[k][i] : v[k][2 * i + 1]);
            const T re = as_row<T>(e * c - o * s), im = as_row<T>(e * s + o * c);
            if constexpr (HALF) p[i] = re, q[i] = im;
            else p[2 * i] = re, p[2 * i + 1] = im;
        }
        T* const dst = out + (long long)h * a.out_head;
        if constexpr (N == 1) {
            dst[0] = p[0];
            if constexpr (HALF) dst[apart] = q[0];
            else dst[1] = p[1];
        } else {
            *reinterpret_cast<row_vec*>(dst) = p;
            if constexpr (HALF) *reinterpret_cast<row_vec*>(dst + apart) = q;
        }
    }
}

template <class T, bool HALF>
static int rope_rows(RopeArgs& a, bool wide, hipStream_t st) {
    constexpr int kWide = (HALF ? 16 : 8) / (int)sizeof(T);  // pairs of 16 bytes, or of 16 bytes of either half
    a.pieces = wide ? a.rd / 2 / kWide : a.rd / 2;
    const bool many = a.n_heads >= kRopeHeads;
    a.groups = many ? (a.n_heads + kRopeHeads - 1) / kRopeHeads : a.n_heads;
    // (pieces and groups are 512 and 2^29 at most)
    const unsigned long long per_token = (unsigned long long)a.groups * a.pieces;
    if (per_token > kLaunchThreads || (unsigned long long)a.n_tokens > kLaunchThreads / per_token) return 1002;
    const unsigned long long blocks = (a.n_tokens * per_token + 255) / 256;
    (void)hipGetLastError();
    const dim3 grid((unsigned)blocks), block(256);
    if (wide && many) launch_kernel(rope_rows_kernel<T, HALF, kWide, kRopeHeads>, grid, block, 0, st, a);
    else if (wide) launch_kernel(rope_rows_kernel<T, HALF, kWide, 1>, grid, block, 0, st, a);
    else if (many) launch_kernel(rope_rows_kernel<T, HALF, 1, kRopeHeads>, grid, block, 0, st, a);
    else launch_kernel(rope_rows_kernel<T, HALF, 1, 1>, grid, block, 0, st, a);
    return launch_status();
}

}  // namespace rk

extern "C" int rivoli_rope_table(float* table, int first, int n_positions, int rd, float base, float factor,
                                 int orig_ctx, float beta_fast, float beta_slow, float mscale, void* stream) {
    if (!table || first < 0 || n_positions <= 0 || rd <= 0 || orig_ctx < 0) return 1001;
    if (!(base > 1.0f && base <= FLT_MAX) || !(factor > 0.0f && factor <= FLT_MAX) || !std::isfinite(mscale)) return 1001;
    if (orig_ctx > 0 && !(beta_slow > 0.0f && beta_fast > beta_slow && beta_fast <= FLT_MAX)) return 1001;
    if (rd > 1024 || (long long)first + n_positions > 0x7fffffffll) return 1002;
    if (rd % 2 != 0 || (uintptr_t)table % 8 != 0) return 1004;
    rk::RopeTableArgs a{table, first, n_positions, rd / 2, std::log2((double)base), factor, 0.0, -1.0, mscale};
    if (orig_ctx > 0) {
        // the pair that turns so many times in the original context
        const auto pair_of = [&](double turns) {
            return rd * std::log(orig_ctx / (turns * 2 * 3.14159265358979323846)) / (2 * std::log((double)base));
        };
        a.low = std::fmax(std::floor(pair_of(beta_fast)), 0.0);
        a.high = std::fmin(std::ceil(pair_of(beta_slow)), rd - 1.0);
        if (a.high < 0.0) a.high = 0.0;
        if (a.high <= a.low) a.high = a.low + 0.001;
    }
    const long long runs = ((long long)n_positions + rk::kTableRun - 1) / rk::kTableRun;
    if ((unsigned long long)(runs * a.pairs) > rk::kLaunchThreads) return 1002;
    const long long blocks = (runs * a.pairs + 255) / 256;
    (void)hipGetLastError();
    rk::launch_kernel(rk::rope_table_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
    return rk::launch_status();
}

extern "C" int rivoli_rope_rows(const void* x, void* out, const float* table, const int* positions, int n_tokens,
                                int n_heads, int rd, int n_positions, long long x_token_stride,
                                long long x_head_stride, long long out_token_stride, long long out_head_stride,
                                int half, int bf16, unsigned int* bad_positions, void* stream) {
    if (!x || !out || !table || !positions || n_tokens <= 0 || n_heads <= 0 || rd <= 0 || n_positions <= 0) return 1001;
    if (rd > 1024) return 1002;
    const uintptr_t size = bf16 ? 2 : 4;
    if (rd % 2 != 0 || (uintptr_t)table % 8 != 0 || (uintptr_t)x % size != 0 || (uintptr_t)out % size != 0) return 1004;
    // whole 16-byte pieces from 16-byte boundaries, in every row
    const long long unit = 16 / (long long)size;
    const bool wide = rk::aligned16(x) && rk::aligned16(out) && (half ? rd / 2 : rd) % unit == 0 &&
                      x_token_stride % unit == 0 && x_head_stride % unit == 0 && out_token_stride % unit == 0 &&
                      out_head_stride % unit == 0;
    rk::RopeArgs a{x, out, table, positions, n_tokens, n_heads, 0, rd, 0, n_positions, x_token_stride, x_head_stride,
                   out_token_stride, out_head_stride, bad_positions};
    const hipStream_t st = (hipStream_t)stream;
    if (bf16) return half ? rk::rope_rows<__bf16, true>(a, wide, st) : rk::rope_rows<__bf16, false>(a, wide, st);
    return half ? rk::rope_rows<float, true>(a, wide, st) : rk::rope_rows<float, false>(a, wide, st);
}
