// Dropout whose mask is not stored: out = residual + (kept ? x / (1 - p) : 0), and with dout in the place of x its own gradient.
//
// Element i is kept if its random word is at least p * 2^32: word i % 4 of the counter-based generator Philox 4x32 (J. Salmon et al., "Parallel random numbers:
// as easy as 1, 2, 3", 2011) with 7 rounds, the fewest that the authors found no test to fail, the seed's 64 bits as the key and the counter i / 4.  A round is two 32 x 32 -> 64 products and
// four exclusive ors of four words: 25 products and about 100 other vector instructions for a lane's 8 16-bit values, which run beside the loads and stores.
//
// HBM-bound.  Measured: 8192 x 8192 bf16 with a residual 62 us (6.5 TB/s), its gradient 46 (5.9); 512 x 1024 2.7 us, latency.  Keeping the mask would add a byte or a bit a value to both
// passes and hold it from one to the other.
#include <algorithm>

#include "f8mi_row.h"

namespace f8mi {

constexpr int DROPOUT_THREADS = 256, DROPOUT_ROUNDS = 7;

// The four words of a counter
__device__ __forceinline__ void philox(uint64_t counter, uint32_t key0, uint32_t key1, uint32_t (&out)[4]) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0u, c3 = 0u;
#pragma unroll
    for (int i = 0; i < DROPOUT_ROUNDS; i++) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ key0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ key1;
        c3 = (uint32_t)p0;
        key0 += 0x9E3779B9u;  // the same in every lane
        key1 += 0xBB67AE85u;
    }
    out[0] = c0;
    out[1] = c1;
    out[2] = c2;
    out[3] = c3;
}

// A lane has pieces of 16 bytes, the next of them DROPOUT_THREADS * gridDim.x pieces on
template <int DT, bool RES>
__global__ __launch_bounds__(DROPOUT_THREADS) void dropout_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ residual, int64_t n, const uint64_t* __restrict__ seed,
                                                                  uint32_t threshold, float factor, uint8_t* __restrict__ out) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    const uint64_t key = *seed;
    const uint32_t key0 = (uint32_t)key, key1 = (uint32_t)(key >> 32);
    const int64_t step = (int64_t)gridDim.x * DROPOUT_THREADS * V;
    for (int64_t at = ((int64_t)blockIdx.x * DROPOUT_THREADS + threadIdx.x) * V; at < n; at += step) {
        float v[V], r[V];
        ln_unpack<DT>(ln_load<DT, int64_t>(x, at, n), v);
        if constexpr (RES) ln_unpack<DT>(ln_load<DT, int64_t>(residual, at, n), r);
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            uint32_t word[4];
            philox((uint64_t)(at + i) >> 2, key0, key1, word);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float kept = word[j] >= threshold ? v[i + j] * factor : 0.f;
                v[i + j] = RES ? r[i + j] + kept : kept;
            }
        }
        ln_store<DT, int64_t>(out, at, n, v);
    }
}

template <int DT>
static int launch_dropout(const void* x, const void* residual, int64_t n, const void* seed, uint32_t threshold, float factor, void* out, hipStream_t stream) {
    constexpr int64_t per = DROPOUT_THREADS * Ln<DT>::V;
    const dim3 grid((unsigned)std::min<int64_t>((n + per - 1) / per, (int64_t)cu_count() * 8 * 8));
    if (residual) hipLaunchKernelGGL((dropout_kernel<DT, true>), grid, dim3(DROPOUT_THREADS), 0, stream, (const uint8_t*)x, (const uint8_t*)residual, n, (const uint64_t*)seed, threshold, factor, (uint8_t*)out);
    else hipLaunchKernelGGL((dropout_kernel<DT, false>), grid, dim3(DROPOUT_THREADS), 0, stream, (const uint8_t*)x, nullptr, n, (const uint64_t*)seed, threshold, factor, (uint8_t*)out);
    return check_hip(hipGetLastError(), "dropout kernel launch");
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int f8mi_dropout(const void* x, const void* residual, int64_t n, int dtype, double p, const int64_t* seed_dev, void* out, void* stream) {
    if (dtype < 0 || dtype > 2) { set_error("f8mi_dropout: unknown dtype code %d", dtype); return F8MI_ERR_INVALID_ARG; }
    if (!(p >= 0.0 && p < 1.0)) { set_error("f8mi_dropout: p=%g is not in [0, 1)", p); return F8MI_ERR_INVALID_ARG; }
    if (n < 0 || (n > 0 && (!x || !seed_dev || !out || (uintptr_t)seed_dev % 8 != 0))) { set_error("f8mi_dropout: null pointer or n=%lld", (long long)n); return F8MI_ERR_INVALID_ARG; }
    if (n == 0) return F8MI_OK;
    // (of a p just below 1 the threshold would round to 2^32)
    const uint32_t threshold = (uint32_t)std::min(4294967295.0, __builtin_rint(p * 4294967296.0));
    const float factor = (float)(1.0 / (1.0 - p));
    if (dtype == F8MI_BF16) return launch_dropout<F8MI_BF16>(x, residual, n, seed_dev, threshold, factor, out, (hipStream_t)stream);
    if (dtype == F8MI_FP16) return launch_dropout<F8MI_FP16>(x, residual, n, seed_dev, threshold, factor, out, (hipStream_t)stream);
    return launch_dropout<F8MI_FP32>(x, residual, n, seed_dev, threshold, factor, out, (hipStream_t)stream);
}
