// 256 x 256 tiles, Bt read transposed from the copy of another product.
#include "f8mi_block_gemm_large_impl.h"

namespace f8mi {

int launch_block_large_tr(const BlockGemm& g, int tiles_m, int tiles_n) {
    if (g.c_dtype == F8MI_BF16) return launch_large2<F8MI_BF16, true, false>(g, tiles_m, tiles_n);
    if (g.c_dtype == F8MI_FP16) return launch_large2<F8MI_FP16, true, false>(g, tiles_m, tiles_n);
    return launch_large2<F8MI_FP32, true, false>(g, tiles_m, tiles_n);
}

}  // namespace f8mi
