// Block scales: e4m3 operands with one power of two for each 128 values of the contraction.
//
// A block stands for q * 2^S with q in e4m3 and S the smallest exponent >= -126 for which max|block| <= 448 * 2^S, so q = v / 2^S
// is exact before it is rounded and never saturates.  S is kept as the biased byte S + 127 that
// v_mfma_scale_f32_16x16x128_f8f6f4 takes (E8M0): the matrix instruction applies the scales of both operands itself, a block scale
// costs no vector arithmetic.  A block that holds an infinity or a NaN stands for NaN throughout.
//
// Bytes of the scales of an operand of `rows` rows contracting over k (padded to a multiple of 128): [k/128][rows padded to 128],
// row r of a group of 128 at (r % 16) * 8 + r / 16.  A lane of the MFMA needs the scales of the rows l % 16 of each of its
// 16-row tiles: with this order they are neighbours, eight tiles one 8-byte read, and the instruction picks the byte.
#pragma once
#include "f8mi_common.h"

namespace f8mi {

constexpr int BLOCK = 128;

__host__ __device__ inline int64_t block_rows_padded(int64_t rows) { return (rows + BLOCK - 1) / BLOCK * BLOCK; }
__host__ __device__ constexpr int block_scale_at(int row) { return (row % 16) * 8 + row / 16; }  // of a row inside its group of 128

// S + 127 of a block whose largest magnitude has these fp32 bits: 448 = 1.75 * 2^8.  (0 and the smallest subnormals: S = -126.)
__device__ __forceinline__ uint32_t block_exponent(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23);
    if (e == 255) return 127u;
    const int s = e - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(s < 1 ? 1 : s);
}
// 2^-S; NaN for a block that holds something that is not finite (then every value of it becomes the NaN code)
__device__ __forceinline__ float block_factor(uint32_t amax_bits) {
    return amax_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - block_exponent(amax_bits)) << 23);
}

}  // namespace f8mi
