// Products of operands with block scales (f8mi_block.h) on 128-row tiles, and the choice of kernel.  Main loop, LDS layout and epilogue are
// those of f8mi_gemm_mid_impl.h; the choice is by the estimates of f8mi_gemm_util.h, fitted to products with one scale: for these only the split of k
// (block_k_splits) was measured.  A stage brings 256 bytes of scales more for each wave, and the matrix instruction applies them.
// Bound by the loads into LDS and their latency.  Measured, bf16: 2048 x 4096 over 4096 30 us (2.3 PFLOP/s), the weight read transposed 32 us, 512 x 1024
// over 1024 7.7 us.
#include <algorithm>

#include "f8mi_block_gemm.h"
#include "f8mi_gemm_mid_impl.h"

namespace f8mi {

template <int C_DT, int TJ, bool B_TR, bool ODD_ROWS>
__global__ __launch_bounds__(GEMM_THREADS) void block_gemm_mid_kernel(
    const uint8_t* __restrict__ A, int64_t a_unit, const uint8_t* __restrict__ sa, int64_t sa_ld, const uint8_t* __restrict__ Bt, int64_t b_unit,
    const uint8_t* __restrict__ sb, int64_t sb_ld, int M, int N, int K, void* __restrict__ C, int64_t ldc, const void* __restrict__ bias, int tiles_m,
    int tiles_n, int c_vec_ok, int k_splits) {
    gemm_mid_tile<0, 0, C_DT, TJ, false, B_TR, ODD_ROWS, false, true>(blockIdx.x, gridDim.x, blockIdx.y, A, 64, a_unit, Bt, 64, b_unit, M, N, K, nullptr, nullptr, C, ldc,
                                                                      bias, tiles_m, tiles_n, c_vec_ok, k_splits, 0, sa, sa_ld, sb, sb_ld);
}

template <int C_DT, int TJ, bool B_TR, bool ODD_ROWS>
static int launch_mid4(const BlockGemm& g, int k_splits, void* C, int64_t ldc, const void* bias) {
    static std::atomic<uint64_t> lds_allowed{0};
    using Cfg = MidCfg<TJ, true>;
    auto kern = block_gemm_mid_kernel<C_DT, TJ, B_TR, ODD_ROWS>;
    if (int rc = allow_big_lds(kern, Cfg::LDS, lds_allowed)) return rc;
    const int tiles_m = (g.M + MID_TILE_M - 1) / MID_TILE_M, tiles_n = (g.N + Cfg::TILE_N - 1) / Cfg::TILE_N;
    hipLaunchKernelGGL(kern, dim3((unsigned)(tiles_m * tiles_n), (unsigned)k_splits), dim3(GEMM_THREADS), Cfg::LDS, g.stream, g.A, g.a_unit(), g.sa, g.sa_ld(), g.Bt,
                       g.b_unit(), g.sb, g.sb_ld(), g.M, g.N, g.K, C, ldc, bias, tiles_m, tiles_n, g.c_vec_ok, k_splits);
    return check_hip(hipGetLastError(), "block-scaled gemm (128-row tiles) kernel launch");
}
template <int C_DT, bool B_TR, bool ODD_ROWS>
static int launch_mid3(const BlockGemm& g, bool wide, int k_splits, void* C, int64_t ldc, const void* bias) {
    if (wide) return launch_mid4<C_DT, 8, B_TR, ODD_ROWS>(g, k_splits, C, ldc, bias);
    return launch_mid4<C_DT, 4, B_TR, ODD_ROWS>(g, k_splits, C, ldc, bias);
}
template <int C_DT>
static int launch_mid2(const BlockGemm& g, bool wide) {
    if (!c_is_fp32(C_DT) && g.c_vec_ok && rows_at_odd_addresses(g.C, g.ldc, C_DT)) {
        if constexpr (!c_is_fp32(C_DT))
            if (!g.b_tr) return launch_mid3<C_DT, false, true>(g, wide, 1, g.C, g.ldc, g.bias);
    }
    if (g.b_tr) return launch_mid3<C_DT, true, false>(g, wide, 1, g.C, g.ldc, g.bias);
    return launch_mid3<C_DT, false, false>(g, wide, 1, g.C, g.ldc, g.bias);
}

// k_splits > 1: the parts go to `partial` (k_splits x M x N floats, N rounded up to a multiple of four) and are added by a second launch
int launch_block_mid(const BlockGemm& g, bool wide, int k_splits, float* partial) {
    if (k_splits > 1) {
        const int pitch = (g.N + 3) / 4 * 4;
        BlockGemm part = g;
        part.c_vec_ok = 1;
        if (int rc = g.b_tr ? launch_mid4<F8MI_FP32, 4, true, false>(part, k_splits, partial, pitch, nullptr) : launch_mid4<F8MI_FP32, 4, false, false>(part, k_splits, partial, pitch, nullptr)) return rc;
        return launch_splitk_reduce(g.c_dtype, k_splits, partial, pitch, g.stream, g.M, g.N, nullptr, nullptr, g.C, g.ldc, g.bias, g.c_vec_ok);
    }
    if (g.c_dtype == F8MI_BF16) return launch_mid2<F8MI_BF16>(g, wide);
    if (g.c_dtype == F8MI_FP16) return launch_mid2<F8MI_FP16>(g, wide);
    return launch_mid2<F8MI_FP32>(g, wide);
}

// Into how many parts a long contraction of at most 128 tiles of 128 x 128 is split so that the CUs get one each; 0: it is not.  Estimates: a
// round of tiles takes 5 us and 2.4 ns for each unit of k with few tiles, 4.2 with one on every CU; the split costs another launch and the parts
// written and read.  Any number of parts, of whole steps, and any width, unlike with one scale for an operand (whole / split, us:
// 640 x 427 over 27648: 72 / 23; 128 x 5632 over 16640: 45 / 25; 267 x 4522 over 9728: 29 / 25; 2002 x 256 over 13312: 36 / 20; 512 x 256 over 4096: 14.2 / 11.9;
// the number taken is within 5 % of the best of 2 - 8 at each).
static int block_k_splits(int64_t m, int64_t n, int64_t k, bool b_tr, int64_t ws_bytes) {
    if (use_mid_tiles(m, n, k) != 1 || m <= 16) return 0;
    const int64_t tiles = ((m + 127) / 128) * ((n + 127) / 128), part = m * ((n + 3) / 4 * 4) * 4;
    if (tiles > 128) return 0;
    const auto round = [&](int s) { return 5.0 + (2.4 + 1.8 * (double)(tiles * s) / 256.0) * 1e-3 * (double)((k / 128 + s - 1) / s * 128); };
    const double whole = round(1), few = !b_tr && use_skinny(m, n, k) ? skinny_time_us(m, n, k) : whole;
    double best_time = 0.9 * std::min(whole, few);  // the estimates are not better than that
    int best = 0;
    for (int s = 2; s <= 8 && tiles * s <= 256 && k / s >= 1024 && s * part <= ws_bytes; s++) {
        const double t = round(s) + 4.0 + (double)s * (double)part * 2.0 / 5e6;
        if (t < best_time) { best_time = t; best = s; }
    }
    return best;
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int64_t f8mi_block_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const int as_is = block_k_splits(m, n, k, false, F8MI_GEMM_WORKSPACE_BYTES), transposed = n % 128 == 0 ? block_k_splits(m, n, k, true, F8MI_GEMM_WORKSPACE_BYTES) : 0;
    return std::max(as_is, transposed) * m * ((n + 3) / 4 * 4) * 4;
}

extern "C" int f8mi_block_gemm(const void* a, const void* a_scales, const void* bt, const void* b_scales, int b_transposed, int64_t m, int64_t n, int64_t k,
                               void* c, int c_dtype, int64_t ldc, const void* bias_dev, void* workspace, int64_t workspace_bytes, void* stream_) {
    if (m < 0 || n < 0 || k < 0 || ldc < n) { set_error("f8mi_block_gemm: bad shape m=%lld n=%lld k=%lld ldc=%lld", (long long)m, (long long)n, (long long)k, (long long)ldc); return F8MI_ERR_INVALID_ARG; }
    if (c_dtype < 0 || c_dtype > 2) { set_error("f8mi_block_gemm: unknown dtype code %d", c_dtype); return F8MI_ERR_INVALID_ARG; }
    if (m == 0 || n == 0) return F8MI_OK;
    if (k % 128 != 0 || k < 128) { set_error("f8mi_block_gemm: k is the padded contraction, a positive multiple of 128 (k=%lld)", (long long)k); return F8MI_ERR_INVALID_ARG; }
    if (b_transposed && n % 128 != 0) { set_error("f8mi_block_gemm: an operand that is read transposed needs its rows to be a multiple of 128 (n=%lld)", (long long)n); return F8MI_ERR_UNSUPPORTED; }
    if (!a || !a_scales || !bt || !b_scales || !c) { set_error("f8mi_block_gemm: null pointer"); return F8MI_ERR_INVALID_ARG; }
    for (const void* p : {a, a_scales, bt, b_scales, (const void*)workspace})
        if ((uintptr_t)p % 16 != 0) { set_error("f8mi_block_gemm: operands, scales and workspace are 16-byte aligned"); return F8MI_ERR_INVALID_ARG; }
    if (m > 0x7fffff00 || n > 0x7fffff00 || k > 0x7fffff || ((m + 127) / 128) * ((n + 127) / 128) > 0x7fffffff) { set_error("f8mi_block_gemm: dimension too large"); return F8MI_ERR_UNSUPPORTED; }
    const BlockGemm g{(const uint8_t*)a, (const uint8_t*)a_scales, (const uint8_t*)bt, (const uint8_t*)b_scales, (int)m, (int)n, (int)k, c, ldc, bias_dev, c_dtype,
                      b_transposed != 0, (uintptr_t)c % (c_dtype == F8MI_FP32 ? 4 : 2) == 0, (hipStream_t)stream_, (int)m};
    ProfScope prof(F8MI_K_GEMM, 2.0 * (double)m * (double)n * (double)k, g.stream);
    const int splits = workspace ? block_k_splits(m, n, k, b_transposed != 0, workspace_bytes) : 0;
    if (splits > 1) return launch_block_mid(g, false, splits, (float*)workspace);
    if (!b_transposed && use_skinny(m, n, k)) return launch_block_few(g);
    if (const int mid = use_mid_tiles(m, n, k)) return launch_block_mid(g, mid == 2, 1, nullptr);
    if (k < 384) return launch_block_mid(g, true, 1, nullptr);
    // the tile rows that fill whole rounds of 256 x 256 tiles, and the rest on 128-row tiles where that is faster
    const int64_t tiles_m = (m + BM - 1) / BM, tiles_n = (n + BN - 1) / BN;
    const RowSplit split = split_last_round(tiles_m, tiles_n, k);
    if (!split.rows_large) return launch_block_large(g, (int)tiles_m, (int)tiles_n);
    if (int rc = launch_block_large(g, (int)split.rows_large, (int)tiles_n)) return rc;
    return launch_block_mid(g.rows_from((int)split.rows_large * BM), split.mid == 2, 1, nullptr);
}
