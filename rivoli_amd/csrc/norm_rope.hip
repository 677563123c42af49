// Norm and rotation of a token's rows in one pass: of query and key heads into rows or into the paged index keys, and
// of the latent row into its page as codes. Launch-only.
//
// A row's first norm_n values become (x - c) * r * w + b, r = 1 / sqrt(mean of (x - c)^2 + eps), c their mean (or zero); then
// the pairs of its rd values from rope_at on turn by the table's row of the token's position, (x, y) -> (x c - y s, x s + y c);
// the others are copied. Sums, statistics and values are f32 from the load to the one rounding at the store: in two
// calls the normed values were rounded, written and read again in between.
#include <cfloat>
#include <cmath>

#include "codec.hpp"

namespace rk {

struct NormRopeArgs {
    const void* x;
    void* out;
    const float *weight, *bias, *table;
    const int *positions, *slots;
    int n_tokens, n_heads, groups;  // of heads: head g, g + groups, ...
    int width, norm_n, rope_at, rd, n_positions;
    long long n_slots;
    long long x_token, x_head, out_token, out_head, weight_head;  // in elements
    float eps;
    int center, half;
    int lanes_log2;                 // of a row
    unsigned int* bad;
};

typedef float f32x4n __attribute__((ext_vector_type(4)));

struct NormRopeRow {
    int norm_n, rope_at, rd, center, half, lanes_log2;
    float eps;
};

// A lane's eight values of a row: of unit u = lane + 64 s (a row of up to 512 values has 2^lanes_log2 lanes and one step) they are 8 u ..; where pairs are
// halves apart, units of the part that is turned have four values of either half instead, so that pairs meet in a lane.
struct Piece {
    int lo, hi;                  // where its first and its last four begin
    int pairs;                   // of them the first in the table's row, as numbers; negative: nothing is turned
    bool apart;
};
__device__ __forceinline__ Piece piece_of(const NormRopeRow& p, int unit) {
    const int o = 8 * unit - p.rope_at;
    const bool turned = o >= 0 && o < p.rd, apart = turned && p.half;
    Piece r;
    r.lo = apart ? p.rope_at + o / 2 : 8 * unit;
    r.hi = apart ? r.lo + p.rd / 2 : r.lo + 4;
    r.pairs = turned ? o : -1, r.apart = apart;
    return r;
}
__device__ __forceinline__ void load8(const __bf16* row, const Piece& at, float (&v)[8]) {
    u32x4 w;
    if (at.apart) {
        const u32x2 a = *reinterpret_cast<const u32x2*>(row + at.lo), b = *reinterpret_cast<const u32x2*>(row + at.hi);
        w = u32x4{a.x, a.y, b.x, b.y};
    } else {
        w = *reinterpret_cast<const u32x4*>(row + at.lo);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo_to_f32(w[i]), v[2 * i + 1] = bf16_hi_to_f32(w[i]);
}
__device__ __forceinline__ void load8(const float* row, const Piece& at, float (&v)[8]) {
    typedef f32x4n any __attribute__((aligned(4)));
    const f32x4n a = *reinterpret_cast<const any*>(row + at.lo), b = *reinterpret_cast<const any*>(row + at.hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}
__device__ __forceinline__ void store8(__bf16* row, const Piece& at, const float (&v)[8]) {
    const u32x4 w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    if (at.apart) {
        *reinterpret_cast<u32x2*>(row + at.lo) = u32x2{w.x, w.y};
        *reinterpret_cast<u32x2*>(row + at.hi) = u32x2{w.z, w.w};
    } else {
        *reinterpret_cast<u32x4*>(row + at.lo) = w;
    }
}
__device__ __forceinline__ void store8(float* row, const Piece& at, const float (&v)[8]) {
    *reinterpret_cast<f32x4n*>(row + at.lo) = f32x4n{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4n*>(row + at.hi) = f32x4n{v[4], v[5], v[6], v[7]};
}

// A sum over a row's lanes, in each of them: neighbours, pairs, quads and eights by instruction operands, sixteens and halves of the wave by swaps.
template <int CTRL>
__device__ __forceinline__ float lane_of(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum(float x, int lanes_log2) {
    if (lanes_log2 > 0) x += lane_of<0xb1>(x);   // quad_perm [1, 0, 3, 2]
    if (lanes_log2 > 1) x += lane_of<0x4e>(x);   // quad_perm [2, 3, 0, 1]
    if (lanes_log2 > 2) x += lane_of<0x141>(x);  // row_half_mirror
    if (lanes_log2 > 3) x += lane_of<0x140>(x);  // row_mirror
    if (lanes_log2 > 4) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if (lanes_log2 > 5) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return x;
}

template <int S>
__device__ __forceinline__ void norm_row(const NormRopeRow& p, const Piece (&at)[S], float (&v)[S][8], const float (&w)[S][8], const float (&b)[S][8]) {
    const float n = (float)p.norm_n;
    const auto in = [&](int s, int i) { return (i < 4 ? at[s].lo : at[s].hi) < p.norm_n; };  // (borders are eights': four values are in or out)
    float c = 0.0f;
    if (p.center) {
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += in(s, i) ? v[s][i] : 0.0f;
        c = row_sum(sum, p.lanes_log2) / n;
    }
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = in(s, i) ? v[s][i] - c : 0.0f;
            sum = __builtin_fmaf(d, d, sum);
        }
    const float r = 1.0f / sqrtf(row_sum(sum, p.lanes_log2) / n + p.eps);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[s][i] = in(s, i) ? __builtin_fmaf((v[s][i] - c) * r, w[s][i], b[s][i]) : v[s][i];
}

// (Written out: every kernel rounds the same products.)
__device__ __forceinline__ void turn_pair(float x, float y, float c, float n, float& re, float& im) {
    re = __builtin_fmaf(x, c, -(y * n)), im = __builtin_fmaf(x, n, y * c);
}
template <int S>
__device__ __forceinline__ void rotate_row(const NormRopeRow& p, const Piece (&at)[S], float (&v)[S][8], const float (&turn)[S][8]) {
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (at[s].pairs >= 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float c = turn[s][2 * i], n = turn[s][2 * i + 1];
                if (p.half) {
                    const float x = v[s][i], y = v[s][i + 4];
                    turn_pair(x, y, c, n, v[s][i], v[s][i + 4]);
                } else {
                    const float x = v[s][2 * i], y = v[s][2 * i + 1];
                    turn_pair(x, y, c, n, v[s][2 * i], v[s][2 * i + 1]);
                }
            }
        }
}

// The lane's four pairs of the table's row.
template <int S>
__device__ __forceinline__ void turns_of(const Piece (&at)[S], const float* row, float (&turn)[S][8]) {
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (at[s].pairs >= 0) load8(row, Piece{at[s].pairs, at[s].pairs + 4, 0, false}, turn[s]);
}

// The lane's weights or biases: eight numbers, or four and four, of those that there are.
template <int S>
__device__ __forceinline__ void weights_of(const NormRopeRow& p, const Piece (&at)[S], const float* from, float otherwise, float (&w)[S][8]) {
    typedef f32x4n any __attribute__((aligned(4)));
#pragma unroll
    for (int s = 0; s < S; ++s) {
        f32x4n a = {otherwise, otherwise, otherwise, otherwise}, b = a;
        if (from && at[s].lo < p.norm_n) a = *reinterpret_cast<const any*>(from + at[s].lo);
        if (from && at[s].hi < p.norm_n) b = *reinterpret_cast<const any*>(from + at[s].hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[s][i] = a[i], w[s][4 + i] = b[i];
    }
}

// Rows of whole 16-byte pieces. A row's lanes have it in S steps; HEADS of them go through at once, so that their loads are on their way
// together and the weights and the table's row serve them all. Bound by memory: every value is read and written once. 8 192 tokens of 64 bf16 heads of 128 values 60 us, 4.5 TB/s
// (a large copy 4.96 to 5.2); by four heads a thread 62, by one 64; with halves exchanged through LDS instead of loaded together 71. Stores past the caches take 57, and cost
// the kernel that reads the rows next more than that (with a sum over them 85.7 us and 82.7).
template <class TX, class TO, int S, int HEADS>
__global__ __launch_bounds__(256) void norm_rope_rows_kernel(const NormRopeArgs a) {
    const unsigned long long at = blockIdx.x * 256ull + threadIdx.x;
    const unsigned item = (unsigned)(at >> a.lanes_log2);
    const int lane = (int)(at & ((1u << a.lanes_log2) - 1));
    const unsigned token_of = item / (unsigned)a.groups;
    const int h0 = (int)(item - token_of * (unsigned)a.groups);
    const bool past = token_of >= (unsigned)a.n_tokens;  // (a wave's rows stay together)
    const int token = past ? 0 : (int)token_of;
    const NormRopeRow p{a.norm_n, a.rope_at, a.rd, a.center, a.half, a.lanes_log2, a.eps};
    const TX* const x = static_cast<const TX*>(a.x) + (long long)token * a.x_token;
    Piece part[S];
    bool there[S];
#pragma unroll
    for (int s = 0; s < S; ++s) part[s] = piece_of(p, lane + kWave * s), there[s] = 8 * (lane + kWave * s) < a.width;
    float v[HEADS][S][8];
#pragma unroll
    for (int k = 0; k < HEADS; ++k)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            // (a head past the last re-reads the last)
            if (there[s]) load8(x + (long long)min(h0 + k * a.groups, a.n_heads - 1) * a.x_head, part[s], v[k][s]);
            else
                for (int i = 0; i < 8; ++i) v[k][s][i] = 0.0f;
        }
    const int pos = a.rd ? a.positions[token] : 0;
    const int slot = a.slots ? a.slots[token] : token;
    const bool bad = (a.rd && (unsigned)pos >= (unsigned)a.n_positions) || (a.slots && slot >= a.n_slots);
    const bool skip = past || bad || slot < 0;
    if (!past && bad && slot >= 0 && a.bad && lane == 0 && h0 == 0) atomicAdd(a.bad, 1u);
    float turn[S][8], w[S][8], b[S][8];
    if (a.rd) turns_of<S>(part, a.table + (size_t)(skip ? 0 : pos) * a.rd, turn);
    if (a.weight_head == 0) weights_of<S>(p, part, a.weight, 1.0f, w), weights_of<S>(p, part, a.bias, 0.0f, b);
    TO* const out = static_cast<TO*>(a.out) + (long long)slot * a.out_token;
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        const int h = h0 + k * a.groups;
        if (a.weight_head != 0) {
            const long long of = (long long)min(h, a.n_heads - 1) * a.weight_head;
            weights_of<S>(p, part, a.weight ? a.weight + of : nullptr, 1.0f, w);
            weights_of<S>(p, part, a.bias ? a.bias + of : nullptr, 0.0f, b);
        }
        norm_row<S>(p, part, v[k], w, b);
        if (a.rd) rotate_row<S>(p, part, v[k], turn);
        if (skip || h >= a.n_heads) continue;
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (there[s]) store8(out + (long long)h * a.out_head, part[s], v[k][s]);
    }
}

// Rows that start or end off the 16 bytes: a wave a row, its values by ones through LDS. Bound by its instructions and loads of two bytes: 8 192 tokens of 16 bf16 heads of 127 values
// 57 us, 1.2 TB/s (of 128 by pieces 16.6 us), of two of 999 32 (of 1 000 15.9). Paths call it with odd widths alone.
constexpr int kNormWidth = 1024;
template <class TX, class TO>
__global__ __launch_bounds__(kWave) void norm_rope_any_kernel(const NormRopeArgs a) {
    __shared__ float row[kNormWidth];
    const int lane = threadIdx.x;
    const unsigned token = blockIdx.x / (unsigned)a.n_heads;
    const int h = (int)(blockIdx.x - token * (unsigned)a.n_heads);
    const int pos = a.rd ? a.positions[token] : 0;
    const long long slot = a.slots ? a.slots[token] : (int)token;
    const bool bad = (a.rd && (unsigned)pos >= (unsigned)a.n_positions) || (a.slots && slot >= a.n_slots);
    if (bad || slot < 0) {
        if (bad && slot >= 0 && a.bad && lane == 0 && h == 0) atomicAdd(a.bad, 1u);
        return;
    }
    const TX* const x = static_cast<const TX*>(a.x) + (long long)token * a.x_token + (long long)h * a.x_head;
    TO* const out = static_cast<TO*>(a.out) + slot * a.out_token + (long long)h * a.out_head;
    const float n = (float)a.norm_n;
    float sum = 0.0f, squares = 0.0f;
    for (int i = lane; i < a.width; i += kWave) {
        const float v = (float)x[i];
        row[i] = v;
        sum += i < a.norm_n ? v : 0.0f;
    }
    const float c = a.center ? row_sum(sum, 6) / n : 0.0f;
    for (int i = lane; i < a.norm_n; i += kWave) {
        const float v = row[i] - c;
        squares = __builtin_fmaf(v, v, squares);
    }
    const float r = 1.0f / sqrtf(row_sum(squares, 6) / n + a.eps);
    const long long of = (long long)h * a.weight_head;
    for (int i = lane; i < a.norm_n; i += kWave)
        row[i] = __builtin_fmaf((row[i] - c) * r, a.weight ? a.weight[of + i] : 1.0f, a.bias ? a.bias[of + i] : 0.0f);
    __syncthreads();
    for (int i = lane; i < a.width; i += kWave) {
        const int o = i - a.rope_at, apart = a.rd / 2;
        float v = row[i];
        if (o >= 0 && o < a.rd) {
            const bool first = a.half ? o < apart : o % 2 == 0;
            const float y = row[first ? i + (a.half ? apart : 1) : i - (a.half ? apart : 1)];
            const f32x2 turn = reinterpret_cast<const f32x2*>(a.table)[(size_t)pos * apart + (a.half ? (first ? o : o - apart) : o / 2)];
            float other;
            if (first) turn_pair(v, y, turn.x, turn.y, v, other);
            else turn_pair(y, v, turn.x, turn.y, other, v);
        }
        out[i] = (TO)v;
    }
}

template <class TX, class TO>
static int norm_rope_rows(NormRopeArgs& a, bool wide, hipStream_t st) {
    (void)hipGetLastError();
    if (!wide) {
        const unsigned long long rows = (unsigned long long)a.n_tokens * a.n_heads;
        if (rows > kLaunchThreads / kWave) return 1002;
        launch_kernel(norm_rope_any_kernel<TX, TO>, dim3((unsigned)rows), dim3(kWave), 0, st, a);
        return launch_status();
    }
    const int units = a.width / 8, steps = units > kWave ? 2 : 1;
    a.lanes_log2 = 0;
    while (a.lanes_log2 < 6 && 1 << a.lanes_log2 < units) ++a.lanes_log2;
    const bool many = steps == 1 && a.n_heads >= 2;
    a.groups = many ? (a.n_heads + 1) / 2 : a.n_heads;
    const unsigned long long per_token = (unsigned long long)a.groups << a.lanes_log2;
    if (per_token > kLaunchThreads || (unsigned long long)a.n_tokens > kLaunchThreads / per_token) return 1002;
    const dim3 grid((unsigned)((a.n_tokens * per_token + 255) / 256)), block(256);
    if (steps == 2) launch_kernel(norm_rope_rows_kernel<TX, TO, 2, 1>, grid, block, 0, st, a);
    else if (many) launch_kernel(norm_rope_rows_kernel<TX, TO, 1, 2>, grid, block, 0, st, a);
    else launch_kernel(norm_rope_rows_kernel<TX, TO, 1, 1>, grid, block, 0, st, a);
    return launch_status();
}

// ---- the latent row into its page -----------------------------------------------------------------------------
// A wave a token: the row is normed over its latent values and rotated over the others as above, and its largest value makes the scale, 448 of which it is; codes are those of the
// quotients. All of it is in 64 bits up to the scale's rounding and the codes': a row is quantized once, and which of two codes a quotient next to their middle gets is decided by the last
// bits of f32 and by the order of sums there, some one in a million values. 8 192 rows 9.2 us, in f32 8.3; 32 rows 4.6.
struct NormAppendArgs {
    const void* x;
    const int* slots;
    const float *weight, *table;
    const int* positions;
    uint8_t* pool;
    int n_tokens, width, page_tokens, n_positions;
    long long x_stride, n_slots;
    size_t page_bytes;
    NormRopeRow row;
    unsigned int* bad;
};

// Over a row's lanes, in each of them (row_sum's order).
template <int CTRL>
__device__ __forceinline__ double lane_of64(double x) {
    const unsigned long long v = __builtin_bit_cast(unsigned long long, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)v, CTRL, 0xf, 0xf, true), hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(v >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
template <int LANES, class F>
__device__ __forceinline__ double row_all64(double x, F f) {
    static_assert(LANES == 16 || LANES == 64, "a row of lanes or the wave");
    x = f(x, lane_of64<0xb1>(x)), x = f(x, lane_of64<0x4e>(x)), x = f(x, lane_of64<0x141>(x)), x = f(x, lane_of64<0x140>(x));
    if constexpr (LANES == 64) {
        const auto halves = [&](auto swap) {
            const unsigned long long v = __builtin_bit_cast(unsigned long long, x);
            const auto l = swap((uint32_t)v), h = swap((uint32_t)(v >> 32));
            x = f(__builtin_bit_cast(double, ((unsigned long long)h[0] << 32) | l[0]), __builtin_bit_cast(double, ((unsigned long long)h[1] << 32) | l[1]));
        };
        halves([](uint32_t u) { return __builtin_amdgcn_permlane16_swap(u, u, false, false); });
        halves([](uint32_t u) { return __builtin_amdgcn_permlane32_swap(u, u, false, false); });
    }
    return x;
}
template <int LANES>
__device__ __forceinline__ double row_sum64(double x) {
    return row_all64<LANES>(x, [](double a, double b) { return a + b; });
}
template <int LANES>
__device__ __forceinline__ double row_top64(double x) {
    return row_all64<LANES>(x, [](double a, double b) { return fmax(a, b); });
}

// A latent piece by its weights, before the norm: y = x w; the squares of x.
__device__ __forceinline__ void weigh_piece(const float (&x)[8], const float (&w)[8], double (&y)[8], double& squares, double& top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double d = x[i];
        squares = __builtin_fma(d, d, squares);
        y[i] = __builtin_fma(d, (double)w[i], 0.0);
        top = fmax(top, fabs(y[i]));
    }
}
__device__ __forceinline__ void turn_piece(const float (&x)[8], const float (&turn)[8], int half, double (&y)[8], double& top) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double one = half ? x[i] : x[2 * i], two = half ? x[i + 4] : x[2 * i + 1], c = turn[2 * i], n = turn[2 * i + 1];
        const double re = __builtin_fma(one, c, -(two * n)), im = __builtin_fma(one, n, two * c);
        (half ? y[i] : y[2 * i]) = re, (half ? y[i + 4] : y[2 * i + 1]) = im;
        top = fmax(top, fmax(fabs(re), fabs(im)));
    }
}
// What a row's values are times for their quotients: normed ones and turned ones; and its scale.
struct RowScale {
    double normed, turned;
    float scale;
    __device__ __forceinline__ RowScale(double squares, double top_normed, double top_turned, int n, float eps) {
        const double r = 1.0 / sqrt(squares / n + (double)eps), top = fmax(top_normed * r, top_turned);
        turned = top > 0.0 ? 448.0 / top : 1.0, normed = r * turned;
        scale = top > 0.0 ? (float)(top / 448.0) : 1.0f;
    }
};

// Eight codes of y * by. The hardware's conversion from f32 has the rule's result but below 2^-6, where the rule rounds halves away, and for what is no number; and f32 has the middle
// of two codes for quotients next to it. These show in the f32 quotients' bits (sizes: without their sign and less one, so that a zero is the largest; it goes the long way, to the same code).
__device__ __forceinline__ u32x2 codes8(const double (&y)[8], double by) {
    float q[8];
    uint32_t low = 0xffffffffu, high = 0, middle = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = (float)(y[i] * by);
        const uint32_t bits = __float_as_uint(q[i]), size = (bits << 1) - 1u;
        low = min(low, size), high = max(high, size), middle = min(middle, (bits << 12) ^ 0x80000000u);
    }
    constexpr uint32_t kLeast = (0x3c800000u << 1) - 1u, kInfinite = 0xff000000u;  // of 2^-6
    if (low >= kLeast && high < kInfinite && middle != 0) return u32x2{e4m3x4_hw(q[0], q[1], q[2], q[3]), e4m3x4_hw(q[4], q[5], q[6], q[7])};
    u32x2 codes = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // in f32 towards zero, the last bit set where that is not all of it: a middle only where it is one
        const double d = y[i] * by;
        uint32_t bits = __float_as_uint(q[i]);
        if (fabs((double)q[i]) > fabs(d)) --bits;
        if ((double)__uint_as_float(bits) != d) bits |= 1u;
        codes[i / 4] |= f32_to_e4m3_sw(__uint_as_float(bits)) << (8 * (i & 3));
    }
    return codes;
}

template <class TX, int S>
__global__ __launch_bounds__(256) void kv_norm_append_kernel(const NormAppendArgs a) {
    const int lane = threadIdx.x & 63;
    const unsigned token = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (token >= (unsigned)a.n_tokens) return;
    const TX* const x = static_cast<const TX*>(a.x) + (long long)token * a.x_stride;
    Piece part[S];
    float v[S][8], w[S][8], turn[S][8];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        part[s] = piece_of(a.row, lane + kWave * s);
        if (8 * (lane + kWave * s) < a.width) load8(x, part[s], v[s]);
        else
            for (int i = 0; i < 8; ++i) v[s][i] = 0.0f;
    }
    weights_of<S>(a.row, part, a.weight, 1.0f, w);
    const int slot = a.slots[token], pos = a.positions[token];
    if (slot < 0) return;
    if (slot >= a.n_slots || (unsigned)pos >= (unsigned)a.n_positions) {
        if (a.bad && lane == 0) atomicAdd(a.bad, 1u);
        return;
    }
    turns_of<S>(part, a.table + (size_t)pos * a.row.rd, turn);
    double y[S][8], squares = 0.0, top_normed = 0.0, top_turned = 0.0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (part[s].pairs >= 0) turn_piece(v[s], turn[s], a.row.half, y[s], top_turned);
        else weigh_piece(v[s], w[s], y[s], squares, top_normed);
    }
    const RowScale by(row_sum64<kWave>(squares), row_top64<kWave>(top_normed), row_top64<kWave>(top_turned), a.row.norm_n, a.row.eps);
    const int page = slot / a.page_tokens, off = slot - page * a.page_tokens;
    uint8_t* const pg = a.pool + (size_t)page * a.page_bytes;
    uint8_t* const to = pg + (size_t)off * a.width;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (8 * (lane + kWave * s) >= a.width) continue;
        const u32x2 codes = codes8(y[s], part[s].pairs >= 0 ? by.turned : by.normed);
        if (part[s].apart) *reinterpret_cast<uint32_t*>(to + part[s].lo) = codes.x, *reinterpret_cast<uint32_t*>(to + part[s].hi) = codes.y;
        else *reinterpret_cast<u32x2*>(to + part[s].lo) = codes;
    }
    if (lane == 0) *reinterpret_cast<float*>(pg + (size_t)a.page_tokens * a.width + 4 * (size_t)off) = by.scale;
}

// The same for many rows of 512 + 64: sixteen lanes a token, which have four latent pieces each and half of them one of the others (a wave a token has its 72 pieces in two
// steps of 64). A lane's latent pieces lie in pairs, whose codes are 16 bytes.
// 8 192 rows of bf16 9.2 us, 1.5 TB/s, a wave a token 14.4; 16 000 14.6 and 22.6; 4 096 6.1 and 8.0; but 2 048 5.5 either way, 1 024 5.4 and 4.7, f32 rows alike: the empty launch and a
// chain of loads, sums, quotients and stores are some 4 us of each. Half of the rest is the quotients' and codes' instructions.
constexpr int kManyTokens = 16;            // a workgroup's
constexpr int kWaveTokens = 2048;          // up to so many a call, a wave has each
template <class TX>
__global__ __launch_bounds__(256) void kv_norm_append_many_kernel(const NormAppendArgs a) {
    const int lane = threadIdx.x & 15;
    const unsigned token = blockIdx.x * (unsigned)kManyTokens + (threadIdx.x >> 4);
    const bool past = token >= (unsigned)a.n_tokens, has_roped = lane < 8;
    const TX* const x = static_cast<const TX*>(a.x) + (past ? 0ll : (long long)token * a.x_stride);
    const auto begin_of = [&](int s) { return 256 * (s >> 1) + 16 * lane + 8 * (s & 1); };
    Piece roped;
    roped.lo = 512 + (a.row.half ? 4 : 8) * (lane & 7), roped.hi = roped.lo + (a.row.half ? 32 : 4), roped.pairs = 8 * (lane & 7), roped.apart = a.row.half != 0;
    float v[5][8], w[4][8], turn[8];
#pragma unroll
    for (int s = 0; s < 4; ++s) load8(x, Piece{begin_of(s), begin_of(s) + 4, -1, false}, v[s]);
    if (has_roped) load8(x, roped, v[4]);
    const int slot = past ? -1 : a.slots[token], pos = past ? 0 : a.positions[token];
    const bool bad = slot >= a.n_slots || (unsigned)pos >= (unsigned)a.n_positions, skip = slot < 0 || bad;
    if (slot >= 0 && bad && a.bad && lane == 0) atomicAdd(a.bad, 1u);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        if (a.weight) load8(a.weight, Piece{begin_of(s), begin_of(s) + 4, 0, false}, w[s]);
        else
            for (int i = 0; i < 8; ++i) w[s][i] = 1.0f;
    }
    if (has_roped) load8(a.table + (size_t)(skip ? 0 : pos) * 64, Piece{roped.pairs, roped.pairs + 4, 0, false}, turn);
    // (pieces' sums in the order in which a wave adds them up: a token's row is the same by either kernel)
    double y[5][8], of[2], top_normed = 0.0, top_turned = 0.0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        double squares[2] = {0.0, 0.0};
        weigh_piece(v[2 * g], w[2 * g], y[2 * g], squares[0], top_normed);
        weigh_piece(v[2 * g + 1], w[2 * g + 1], y[2 * g + 1], squares[1], top_normed);
        of[g] = row_sum64<16>(squares[0] + squares[1]);
    }
    if (has_roped) turn_piece(v[4], turn, a.row.half, y[4], top_turned);
    const RowScale by(of[0] + of[1], row_top64<16>(top_normed), row_top64<16>(top_turned), 512, a.row.eps);
    if (skip) return;
    const int page = slot / a.page_tokens, off = slot - page * a.page_tokens;
    uint8_t* const pg = a.pool + (size_t)page * a.page_bytes;
    uint8_t* const to = pg + (size_t)off * 576;
#pragma unroll
    for (int s = 0; s < 4; s += 2) {
        const u32x2 one = codes8(y[s], by.normed), two = codes8(y[s + 1], by.normed);
        *reinterpret_cast<u32x4*>(to + begin_of(s)) = u32x4{one.x, one.y, two.x, two.y};
    }
    if (has_roped) {
        const u32x2 codes = codes8(y[4], by.turned);
        if (roped.apart) *reinterpret_cast<uint32_t*>(to + roped.lo) = codes.x, *reinterpret_cast<uint32_t*>(to + roped.hi) = codes.y;
        else *reinterpret_cast<u32x2*>(to + roped.lo) = codes;
    }
    if (lane == 8) *reinterpret_cast<float*>(pg + (size_t)a.page_tokens * 576 + 4 * (size_t)off) = by.scale;
}

}  // namespace rk

extern "C" int rivoli_norm_rope_rows(const void* x, void* out, const float* weight, const float* bias, const float* table,
                                     const int* positions, const int* slots, int n_tokens, int n_heads, int width, int norm_n,
                                     int rope_at, int rd, int n_positions, int n_slots, long long x_token_stride,
                                     long long x_head_stride, long long out_token_stride, long long out_head_stride,
                                     long long weight_head_stride, float eps, int center, int half, int x_bf16, int out_bf16,
                                     unsigned int* bad_tokens, void* stream) {
    if (!x || !out || n_tokens <= 0 || n_heads <= 0 || width <= 0 || norm_n <= 0 || rope_at < 0 || rd < 0 || weight_head_stride < 0) return 1001;
    if (rd > 0 && (!table || !positions || n_positions <= 0)) return 1001;
    if (slots && n_slots <= 0) return 1001;
    if (!(eps >= 0.0f && eps <= FLT_MAX)) return 1001;
    if (width > rk::kNormWidth || norm_n > width || (long long)rope_at + rd > width) return 1002;
    const uintptr_t x_size = x_bf16 ? 2 : 4, out_size = out_bf16 ? 2 : 4;
    if (rd % 2 != 0 || (rd > 0 && (uintptr_t)table % 8 != 0) || (uintptr_t)x % x_size != 0 || (uintptr_t)out % out_size != 0 ||
        (uintptr_t)weight % 4 != 0 || (uintptr_t)bias % 4 != 0)
        return 1004;
    // whole 16-byte pieces from 16-byte boundaries, in every row, and no pair, and no border, inside of a lane's eight values
    const long long xu = 16 / (long long)x_size, ou = 16 / (long long)out_size;
    const bool wide = rk::aligned16(x) && rk::aligned16(out) && x_token_stride % xu == 0 && x_head_stride % xu == 0 && out_token_stride % ou == 0 &&
                      out_head_stride % ou == 0 && width % 8 == 0 && norm_n % 8 == 0 && rope_at % 8 == 0 && rd % (half ? 16 : 8) == 0;
    rk::NormRopeArgs a{x, out, weight, bias, table, positions, slots, n_tokens, n_heads, 0, width, norm_n, rope_at, rd, n_positions, n_slots,
                       x_token_stride, x_head_stride, out_token_stride, out_head_stride, weight || bias ? weight_head_stride : 0, eps, center, half, 0,
                       bad_tokens};
    const hipStream_t st = (hipStream_t)stream;
    if (x_bf16) return out_bf16 ? rk::norm_rope_rows<__bf16, __bf16>(a, wide, st) : rk::norm_rope_rows<__bf16, float>(a, wide, st);
    return out_bf16 ? rk::norm_rope_rows<float, __bf16>(a, wide, st) : rk::norm_rope_rows<float, float>(a, wide, st);
}

extern "C" int rivoli_kv_norm_append_paged(const void* x, const int* slot_mapping, const float* weight, const float* table,
                                           const int* positions, unsigned char* pool, int n_tokens, long long x_stride, int kvl,
                                           int rope, int n_positions, int page_tokens, int n_pages, float eps, int half, int bf16,
                                           unsigned int* bad_tokens, void* stream) {
    if (!x || !slot_mapping || !table || !positions || !pool || n_tokens <= 0 || kvl <= 0 || rope <= 0 || n_positions <= 0 || page_tokens <= 0 ||
        n_pages <= 0 || !(eps >= 0.0f && eps <= FLT_MAX))
        return 1001;
    if ((long long)kvl + rope > rk::kNormWidth || (unsigned)n_tokens > rk::kLaunchThreads / rk::kWave) return 1002;
    const int width = kvl + rope;
    const long long unit = bf16 ? 8 : 4;
    if (width % 16 != 0 || kvl % 8 != 0 || rope % (half ? 16 : 8) != 0 || page_tokens % 4 != 0 || x_stride % unit != 0 || !rk::aligned16(x) ||
        !rk::aligned16(pool) || (uintptr_t)table % 8 != 0 || (uintptr_t)weight % 4 != 0)
        return 1004;
    const rk::NormAppendArgs a{x, slot_mapping, weight, table, positions, pool, n_tokens, width, page_tokens, n_positions, x_stride,
                               (long long)n_pages * page_tokens, (size_t)page_tokens * (size_t)(width + 4),
                               rk::NormRopeRow{kvl, kvl, rope, 0, half, 6, eps}, bad_tokens};
    const dim3 grid((unsigned)((n_tokens + 3) / 4)), block(256);
    const hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();
    if (kvl == 512 && rope == 64 && n_tokens > rk::kWaveTokens) {
        const dim3 many((unsigned)((n_tokens + rk::kManyTokens - 1) / rk::kManyTokens));
        if (bf16) rk::launch_kernel(rk::kv_norm_append_many_kernel<__bf16>, many, block, 0, st, a);
        else rk::launch_kernel(rk::kv_norm_append_many_kernel<float>, many, block, 0, st, a);
    } else if (width > 512) {
        if (bf16) rk::launch_kernel(rk::kv_norm_append_kernel<__bf16, 2>, grid, block, 0, st, a);
        else rk::launch_kernel(rk::kv_norm_append_kernel<float, 2>, grid, block, 0, st, a);
    } else {
        if (bf16) rk::launch_kernel(rk::kv_norm_append_kernel<__bf16, 1>, grid, block, 0, st, a);
        else rk::launch_kernel(rk::kv_norm_append_kernel<float, 1>, grid, block, 0, st, a);
    }
    return rk::launch_status();
}
