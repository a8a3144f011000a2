// 256 x 256 tiles on operands as they are.
#include "f8mi_block_gemm_large_impl.h"

namespace f8mi {

int launch_block_large(const BlockGemm& g, int tiles_m, int tiles_n) {
    if (g.b_tr) return launch_block_large_tr(g, tiles_m, tiles_n);
    if (g.c_vec_ok && rows_at_odd_addresses(g.C, g.ldc, g.c_dtype)) return launch_block_large_odd(g, tiles_m, tiles_n);
    if (g.c_dtype == F8MI_BF16) return launch_large2<F8MI_BF16, false, false>(g, tiles_m, tiles_n);
    if (g.c_dtype == F8MI_FP16) return launch_large2<F8MI_FP16, false, false>(g, tiles_m, tiles_n);
    return launch_large2<F8MI_FP32, false, false>(g, tiles_m, tiles_n);
}

}  // namespace f8mi
