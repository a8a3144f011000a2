// 256 x 256 tiles, rows of a 16-bit C at odd multiples of two bytes.
#include "f8mi_block_gemm_large_impl.h"

namespace f8mi {

int launch_block_large_odd(const BlockGemm& g, int tiles_m, int tiles_n) {
    if (g.c_dtype == F8MI_BF16) return launch_large2<F8MI_BF16, false, true>(g, tiles_m, tiles_n);
    return launch_large2<F8MI_FP16, false, true>(g, tiles_m, tiles_n);
}

}  // namespace f8mi
