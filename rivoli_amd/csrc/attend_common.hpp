// Pieces the attention kernels share: operand vector types, typed LDS pointers, the
// reductions over the four 16-lane rows of a wave, the order in which a 32-token tile's
// tokens sit in the value contraction, codes to bf16, transfers from memory into LDS.
#pragma once
#include "codec.hpp"

namespace rk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
template <class T>
using lds_ptr = __attribute__((address_space(3))) T*;

constexpr float kLazyRescale = 8.0f;       // log2 units
constexpr float kLog2e = 1.4426950408889634f;

// max / sum of a value over the four 16-lane rows of the wave, in every lane. gfx950's row
// swaps stay in the vector ALU; the generic cross-lane shuffle goes through the LDS crossbar.
__device__ __forceinline__ float rows_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));  // rows {0,1} and {2,3} paired
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// In the score tile (rows = tokens, 16 per MFMA) a lane of row group g holds rows 4g..4g+3
// of both 16-token halves, and those 8 values are element j = 4*half + i of the value MFMA's
// A operand for contraction index 8g + j. Staging wave w (of 8) owns contraction indices
// 4w..4w+3 — tile positions 16*(w&1) + 4*(w>>1) + i, four consecutive tokens.
__device__ __forceinline__ int tile_pos_of(int wave, int i) { return 16 * (wave & 1) + 4 * (wave >> 1) + i; }

// e4m3 codes -> bf16, exact: four codes (one dword) -> two dwords
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t c, uint32_t& lo, uint32_t& hi) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true));
}

// Sixteen bytes per lane from memory straight into LDS: lane L's land at dst + 16 L (dst is
// wave-uniform). Issued as text: through the builtin the compiler makes every later LDS read wait
// for the transfer, whichever buffer it reads. The caller waits (vmcnt) before the data is used.
__device__ __forceinline__ void dma16(const uint8_t* src, lds_ptr<uint8_t> dst) {
    const uint32_t base = (uint32_t)(uintptr_t)dst;
    uint32_t keep;  // m0 is the instruction's LDS base; the compiler's own value of it is put back
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(src), "s"(base)
                 : "memory");
}

// The same from a wave-uniform address plus a 32-bit offset per lane (the instruction's scalar
// base form: no 64-bit add, and offsets kept across a loop cost one register each). The base is
// made scalar here: an operand that reaches the statement through a loop-carried value may
// otherwise sit in vector registers, which the assembler accepts and the instruction misreads.
__device__ __forceinline__ void dma16_from(const uint8_t* base_uniform, uint32_t off, lds_ptr<uint8_t> dst) {
    const uint32_t lds_base = (uint32_t)(uintptr_t)dst;
    const uint64_t b = (uint64_t)(uintptr_t)base_uniform;
    const uint64_t sb = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) |
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(sb), "s"(lds_base)
                 : "memory");
}

// Four bytes per lane from memory into LDS, as dma16.
__device__ __forceinline__ void few_dma4(const void* src, lds_ptr<uint8_t> dst) {
    const uint32_t base = (uint32_t)(uintptr_t)dst;
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(src), "s"(base)
                 : "memory");
}

// A lane's four pieces of a row's codes, 128 bytes apart in memory and 1024 in LDS, and its fifth, of the roped codes, for the lanes of
// `roped`. The instruction's offset counts in memory and in LDS, so m0 makes up the difference and the address is one. All lanes are here.
__device__ __forceinline__ void few_dma_row(const uint8_t* src, lds_ptr<uint8_t> to, lds_ptr<uint8_t> to_rope, unsigned long long roped) {
    const uint32_t base = (uint32_t)(uintptr_t)to, rope = (uint32_t)(uintptr_t)to_rope - 512u;
    uint32_t keep;
    unsigned long long all;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\t"
                 "s_add_u32 m0, m0, 896\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off offset:128\n\t"
                 "s_add_u32 m0, m0, 896\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off offset:256\n\t"
                 "s_add_u32 m0, m0, 896\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off offset:384\n\t"
                 "s_mov_b32 m0, %4\n\ts_and_saveexec_b64 %1, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off offset:512\n\t"
                 "s_mov_b64 exec, %1\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep), "=&s"(all)
                 : "v"(src), "s"(base), "s"(rope), "s"(roped)
                 : "memory", "scc");
}

}  // namespace rk
