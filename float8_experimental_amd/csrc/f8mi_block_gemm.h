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

    int64_t a_unit() const { return (int64_t)M * 64; }
    int64_t b_unit() const { return (int64_t)(b_tr ? K : N) * 64; }
    int64_t sa_ld() const { return block_rows_padded(M); }
    int64_t sb_ld() const { return block_rows_padded(N); }
};

int launch_block_mid(const BlockGemm& g, bool wide, int k_splits, float* partial);

}  // namespace f8mi
