// Products of operands with block scales on 256 x 256 tiles: the main loop of f8mi_gemm_dma16_impl.h with its places for the scales.
// Bound by the matrix cores at the clock that the power cap leaves.  Measured, bf16: 8192 x 28672 over 8192 1.31 ms (2.94 PFLOP/s), the weight read
// transposed 1.26 ms (3.05); within 2 - 4 % of the same tiles with one scale for an operand on the same bytes.
#pragma once
#include "f8mi_block_gemm.h"
#include "f8mi_gemm_dma16_impl.h"

namespace f8mi {

template <int C_DT, bool ODD, bool B_TR, bool ODD_ROWS>
__global__ __launch_bounds__(GEMM_THREADS) void block_gemm_large_kernel(
    const uint8_t* __restrict__ A, int64_t a_unit, const uint8_t* __restrict__ sa, int64_t sa_ld, const uint8_t* __restrict__ Bt, int64_t b_unit,
    const uint8_t* __restrict__ sb, int64_t sb_ld, int M, int N, int K, void* __restrict__ C, int64_t ldc, const void* __restrict__ bias, int tiles_m,
    int tiles_n, int c_vec_ok) {
    gemm_dma16_tile<0, 0, C_DT, ODD, false, B_TR, ODD_ROWS, 8, false, true>(blockIdx.x, gridDim.x, A, 64, a_unit, Bt, 64, b_unit, M, N, K, nullptr, nullptr, C, ldc, bias, tiles_m,
                                                                           tiles_n, c_vec_ok, 0, sa, sa_ld, sb, sb_ld);
}

template <int C_DT, bool ODD, bool B_TR, bool ODD_ROWS>
static int launch_large3(const BlockGemm& g, int tiles_m, int tiles_n) {
    static std::atomic<uint64_t> lds_allowed{0};
    auto kern = block_gemm_large_kernel<C_DT, ODD, B_TR, ODD_ROWS>;
    if (int rc = allow_big_lds(kern, LargeCfg<8>::LDS, lds_allowed)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(tiles_m * tiles_n)), dim3(GEMM_THREADS), LargeCfg<8>::LDS, g.stream, g.A, g.a_unit(), g.sa, g.sa_ld(), g.Bt, g.b_unit(), g.sb,
                       g.sb_ld(), g.M, g.N, g.K, g.C, g.ldc, g.bias, tiles_m, tiles_n, g.c_vec_ok);
    return check_hip(hipGetLastError(), "block-scaled gemm kernel launch");
}
template <int C_DT, bool B_TR, bool ODD_ROWS>
static int launch_large2(const BlockGemm& g, int tiles_m, int tiles_n) {
    if ((g.K / 128) & 1) return launch_large3<C_DT, true, B_TR, ODD_ROWS>(g, tiles_m, tiles_n);
    return launch_large3<C_DT, false, B_TR, ODD_ROWS>(g, tiles_m, tiles_n);
}

}  // namespace f8mi
