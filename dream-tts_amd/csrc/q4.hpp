// 4-bit pages: rows of D values in groups of 32, value = f16(c d + b) with c = 64 + n, n the value's 4 bits, d and b the
// group's f16 pair. As an f16, 64 + n is the bits 0x5400 | n << 4, so two codes of a word become two numbers with one
// and-or (after a shift, for three of four), and one packed fma makes them the two values with their one rounding. With codes
// from 0 on, a subtraction would come between. (11 instructions for 8 values against 13; an attention tile of 32 keys of 128
// dimensions spends 192 of its 350 on them, and over 5 x 65000 keys vector issue, 0.63 of the cycles, is what it waits for most.)
//
// A page of a kv head (5 D / 8 bytes a row, against 2 D) is first the rows' codes, D / 8 words of 32 a row: element 8 w + 2 i
// of a row in bits 4 i of its word w, element 8 w + 2 i + 1 in bits 16 + 4 i, so that a pair of neighbours is one number apart
// from its shift. Then the pairs (d, b), [D / 32][row].
//   keys:   words [row][w]: a lane of the score product takes one key's neighbouring dimensions, 16 bytes
//   values: words [row / 4][w][row % 4]: a lane of the output product takes eight dimensions of four neighbouring keys, 16 bytes,
//           and so do their four pairs of one group
#pragma once

#include "common.hpp"

namespace dtts {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kQ4Code = 0x00f000f0u, kQ4Base = 0x54005400u;
// The two in registers: as literals the and-or became two instructions (a three-operand one takes no literal).
struct Q4Bits {
    uint32_t code = kQ4Code, base = kQ4Base;
    __device__ __forceinline__ Q4Bits() {
        asm("" : "+s"(code));
        asm("" : "+v"(base));
    }
};
constexpr float kQ4First = 64.0f, kQ4Last = 79.0f;  // the codes' least and greatest

// Bytes of a row, and byte offsets in a page of a kv head.
template <int D>
struct Q4Row {
    static constexpr int kWords = D / 8, kBytes = D / 2 + D / 8;
    __device__ __forceinline__ static int key_word(int row, int w) { return (row * kWords + w) * 4; }
    __device__ __forceinline__ static int value_word(int row, int w) { return (((row >> 2) * kWords + w) * 4 + (row & 3)) * 4; }
    __device__ __forceinline__ static int pair(int page, int row, int group) { return page * (D / 2) + (group * page + row) * 4; }
};

// The i-th pair of codes of a word (i a constant), as f16 numbers.
__device__ __forceinline__ half2_t q4_codes(uint32_t word, int i, const Q4Bits &bits) {
    const uint32_t at = i == 0 ? word << 4 : i == 1 ? word : i == 2 ? word >> 4 : word >> 8;
    return __builtin_bit_cast(half2_t, (at & bits.code) | bits.base);
}

// Halves of two words: the low ones, the high ones.
__device__ __forceinline__ uint32_t low_halves(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); }

// The eight values of a word, in order.
__device__ __forceinline__ half8_t q4_values(uint32_t word, uint32_t pair, const Q4Bits &bits) {
    const half2_t d = __builtin_bit_cast(half2_t, low_halves(pair, pair)), b = __builtin_bit_cast(half2_t, high_halves(pair, pair));
    half8_t y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t v = __builtin_elementwise_fma(q4_codes(word, i, bits), d, b);
        y[2 * i] = v[0];
        y[2 * i + 1] = v[1];
    }
    return y;
}

}  // namespace
}  // namespace dtts
