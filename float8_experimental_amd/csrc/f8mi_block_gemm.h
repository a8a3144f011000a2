// What the translation units of the products with block scales share: operands, and the launches of each kernel.
#pragma once
#include "f8mi_block.h"
#include "f8mi_gemm_util.h"

namespace f8mi {

// C [M][N] = A Bt^T (+ bias).  A [K/64][M][64]; Bt [K/64][N][64], or with b_tr the copy of another product, [N/64][K][64], read
// transposed.  Scales: f8mi_block.h.
struct BlockGemm {
    const uint8_t *A, *sa, *Bt, *sb;
    int M, N, K;
    void* C;
    int64_t ldc;
    const void* bias;
    int c_dtype, b_tr, c_vec_ok;
    hipStream_t stream;
    int a_rows;  // of A's copy, of which the M from A on are multiplied

    int64_t a_unit() const { return (int64_t)a_rows * 64; }
    int64_t b_unit() const { return (int64_t)(b_tr ? K : N) * 64; }
    int64_t sa_ld() const { return block_rows_padded(a_rows); }
    int64_t sb_ld() const { return block_rows_padded(N); }
    BlockGemm rows_from(int first) const {  // a multiple of 128
        BlockGemm g = *this;
        g.A += (int64_t)first * 64;
        g.sa += first;
        g.C = (uint8_t*)C + (int64_t)first * ldc * (c_dtype == F8MI_FP32 ? 4 : 2);
        g.M -= first;
        return g;
    }
};

int launch_block_mid(const BlockGemm& g, bool wide, int k_splits, float* partial);
// M <= SKINNY_MAX_M, operands as they are
int launch_block_few(const BlockGemm& g);
// tiles_m tile rows of 256 from the first; K >= 384.  The second is taken by the first for such rows of C, the third for b_tr.
int launch_block_large(const BlockGemm& g, int tiles_m, int tiles_n);
int launch_block_large_odd(const BlockGemm& g, int tiles_m, int tiles_n);
int launch_block_large_tr(const BlockGemm& g, int tiles_m, int tiles_n);

}  // namespace f8mi
