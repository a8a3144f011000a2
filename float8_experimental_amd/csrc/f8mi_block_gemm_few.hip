// Linears of few rows with block scales: reading the weight once is all the work there is.
//
// As in f8mi_gemm_skinny.hip a workgroup of eight waves owns 16 or 32 columns of C and all rows (up to 128) of A; the waves split k eight ways, stream
// their part of the weight straight into operands of the matrix instruction, several steps of 128 k in flight, and their partial sums meet in LDS and
// are added in a fixed order.  The scales of a step come with it: a byte for each 16-row tile of the weight, a word for four tiles of A.
//
// Up to 16 rows and F8MI_FEW_ROWS_ELEMS activations need no cast in front: every workgroup converts all activations into its LDS while the first
// weights are on their way.  A block of 128 is 16 (fp32: 32) neighbouring lanes, so its maximum is four (five) steps between lanes and,
// unlike one scale for all of x, nothing waits for the rest of the workgroup.
//
// Bound by the read of the weight.  Measured: one bf16 token through 8192 x 8192 in one kernel 13.7 us (4.9 TB/s of the weight; cast and product
// in two launches on 128-row tiles: 27.3).
#include "f8mi_block_gemm.h"

namespace f8mi {

typedef float v4f_w __attribute__((ext_vector_type(4)));

constexpr int FEW_WAVES = 8, FEW_THREADS = FEW_WAVES * 64;
constexpr int FEW_LDS_PAD = 16;  // bytes between rows of x in LDS
// steps in flight per wave: what the fragments of A, or x itself, leave registers for
constexpr int few_depth(int mt) { return mt <= 2 ? 4 : mt <= 4 ? 2 : 1; }
constexpr int few_cast_depth(int nt, int dt) { return nt == 2 && dt == F8MI_FP32 ? 2 : 4; }

__device__ __forceinline__ v8i few_load(const uint8_t* p) {
    const uint4 lo = *(const uint4*)p, hi = *(const uint4*)(p + 16);
    return (v8i){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}
// byte `at` of the word that scales A's tiles; the weight's byte is the lowest
template <int AT>
__device__ __forceinline__ v4f_w few_mfma_at(const v8i& w, const v8i& a, const v4f_w& acc, uint32_t sw, uint32_t sa) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, (int)sw, AT, (int)sa);
}
__device__ __forceinline__ v4f_w few_mfma(int at, const v8i& w, const v8i& a, const v4f_w& acc, uint32_t sw, uint32_t sa) {
    switch (at) {  // a constant once the caller's loop is unrolled
        case 0: return few_mfma_at<0>(w, a, acc, sw, sa);
        case 1: return few_mfma_at<1>(w, a, acc, sw, sa);
        case 2: return few_mfma_at<2>(w, a, acc, sw, sa);
        default: return few_mfma_at<3>(w, a, acc, sw, sa);
    }
}

// The eight partial sums of every output, in a fixed order, biased, converted and stored.  acc[mt][nt]: lane l holds row 16 mt + l % 16 and
// columns n0 + 16 nt + 4 * (l / 16) + e.
template <int C_DT, int MT, int NT>
__device__ __forceinline__ void few_finish(const v4f_w (&acc)[MT][NT], float4 (&part)[FEW_WAVES / 2][MT * NT][64], int M, int N, int n0, void* C, int64_t ldc,
                                           const void* bias) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave >= FEW_WAVES / 2) {
#pragma unroll
        for (int i = 0; i < MT * NT; i++) part[wave - FEW_WAVES / 2][i][lane] = make_float4(acc[i / NT][i % NT][0], acc[i / NT][i % NT][1], acc[i / NT][i % NT][2], acc[i / NT][i % NT][3]);
    }
    __syncthreads();
    if (wave < FEW_WAVES / 2) {
#pragma unroll
        for (int i = 0; i < MT * NT; i++) {
            const float4 p = part[wave][i][lane];
            const v4f_w& a = acc[i / NT][i % NT];
            part[wave][i][lane] = make_float4(a[0] + p.x, a[1] + p.y, a[2] + p.z, a[3] + p.w);
        }
    }
    __syncthreads();
    for (int item = threadIdx.x; item < MT * NT * 64; item += FEW_THREADS) {
        const int tile = item >> 6, l = item & 63;
        float4 sum = part[0][tile][l];
#pragma unroll
        for (int w = 1; w < FEW_WAVES / 2; w++) {
            const float4 p = part[w][tile][l];
            sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
        }
        const int row = (tile / NT) * 16 + (l & 15), col = n0 + (tile % NT) * 16 + 4 * (l >> 4);
        if (row >= M || col >= N) continue;
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (col + e >= N) break;
            const float r = v[e] + (bias ? load_bias<C_DT>(bias, col + e) : 0.f);
            const int64_t at = (int64_t)row * ldc + col + e;
            if constexpr (C_DT == F8MI_FP32) ((float*)C)[at] = r;
            else ((uint16_t*)C)[at] = (uint16_t)(pack2<C_DT>(r, 0.f) & 0xffffu);
        }
    }
}

// The weight of a workgroup's columns: a lane's 32 bytes of step s of tile nt, and its scale; rows past the end re-read the last one.
template <int NT>
struct FewWeight {
    const uint8_t *p[NT], *scale;
    int64_t step, scale_step;
    __device__ __forceinline__ FewWeight(const uint8_t* W, const uint8_t* scales, int N, int n0) {
        const int lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4;
        const int64_t unit = (int64_t)N * 64;
        step = 2 * unit;
        scale_step = block_rows_padded(N);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) p[nt] = W + (int64_t)min(n0 + nt * 16 + lm, N - 1) * 64 + (lq >> 1) * unit + (lq & 1) * 32;
        scale = scales + (n0 & ~127) + lm * 8 + ((n0 & 127) >> 4);  // n0: a multiple of 16 NT, so the tiles' bytes are neighbours
    }
    __device__ __forceinline__ void load(int s, v8i (&w)[NT], uint32_t& sw) const {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) w[nt] = few_load(p[nt] + s * step);
        const uint8_t* at = scale + s * scale_step;
        sw = NT == 1 ? *at : *(const uint16_t*)at;
    }
};

template <int C_DT, int MT, int NT, int DEPTH>
__global__ __launch_bounds__(FEW_THREADS) void block_gemm_few_kernel(const uint8_t* __restrict__ A, int64_t a_unit, const uint8_t* __restrict__ sa, int64_t sa_ld,
                                                                     const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw_all, int M_all, int N, int K,
                                                                     void* __restrict__ C_all, int64_t ldc, const void* __restrict__ bias) {
    __shared__ float4 part[FEW_WAVES / 2][MT * NT][64];
    // blockIdx.y: which block of 16 * MT rows (more than one: 128) this workgroup multiplies
    const int m_base = blockIdx.y * (16 * MT), M = min(M_all - m_base, 16 * MT);
    void* C = (uint8_t*)C_all + (int64_t)m_base * ldc * (C_DT == F8MI_FP32 ? 4 : 2);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lm = lane & 15, lq = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const int steps = K / 128, s0 = steps * wave / FEW_WAVES, s1 = steps * (wave + 1) / FEW_WAVES;
    const FewWeight<NT> weight(W, sw_all, N, n0);
    const uint8_t* pa[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) pa[mt] = A + (int64_t)(m_base + min(mt * 16 + lm, M - 1)) * 64 + (lq >> 1) * a_unit + (lq & 1) * 32;
    const uint8_t* psa = sa + (m_base & ~127) + lm * 8;

    v4f_w acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT * NT; i++) acc[i / NT][i % NT] = (v4f_w){0.f, 0.f, 0.f, 0.f};
    v8i fa[DEPTH][MT], fw[DEPTH][NT];
    uint32_t fsw[DEPTH], fsa[DEPTH][(MT + 3) / 4];
    auto load = [&](int d, int s) __attribute__((always_inline)) {  // past the wave's range: a valid address, the product is skipped
        const int sd = min(s, s1 - 1);
        weight.load(sd, fw[d], fsw[d]);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) fa[d][mt] = few_load(pa[mt] + 2 * (int64_t)sd * a_unit);
#pragma unroll
        for (int i = 0; i < (MT + 3) / 4; i++) fsa[d][i] = *(const uint32_t*)(psa + sd * sa_ld + 4 * i);
    };
    auto multiply = [&](int d) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[mt][nt] = few_mfma(mt & 3, fw[d][nt], fa[d][mt], acc[mt][nt], fsw[d] >> (8 * nt), fsa[d][mt >> 2]);
    };
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) load(d, s0 + d);
    }
    int s = s0;
    for (; s + DEPTH < s1; s += DEPTH) {  // a slot is filled again as soon as it has been multiplied
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            multiply(d);
            load(d, s + DEPTH + d);
        }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (s + d < s1) multiply(d);
    few_finish<C_DT, MT, NT>(acc, part, M, N, n0, C, ldc, bias);
}

// x [M][K] in its own type (K: not padded; Kp: padded)
template <int DT, int NT, int DEPTH>
__global__ __launch_bounds__(FEW_THREADS, 4) void block_linear_few_kernel(const uint8_t* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ W,
                                                                          const uint8_t* __restrict__ sw_all, int M, int N, int K, int Kp, void* __restrict__ C, int64_t ldc,
                                                                          const void* __restrict__ bias) {
    constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2, V = 16 / SIZE;
    constexpr int PIECES = F8MI_FEW_ROWS_ELEMS / V / FEW_THREADS;
    extern __shared__ __align__(16) uint8_t x8[];  // [M][Kp + FEW_LDS_PAD], then the scales [M][Kp / 128]
    __shared__ float4 part[FEW_WAVES / 2][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lm = lane & 15, lq = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const int steps = Kp / 128, pitch = Kp + FEW_LDS_PAD;
    const int s0 = steps * wave / FEW_WAVES, s1 = steps * (wave + 1) / FEW_WAVES;
    uint8_t* const xs = x8 + M * pitch;

    // x, ahead of the weights: needed first.  Piece i of V values: a block of 128 is 128 / V neighbouring lanes
    const uint32_t per_row = (uint32_t)Kp / V, items = (uint32_t)M * per_row;
    uint4 v[PIECES];
#pragma unroll
    for (int u = 0; u < PIECES; u++) {
        const uint32_t i = u * FEW_THREADS + threadIdx.x;
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (i < items) {
            const uint32_t row = i / per_row;
            const int col = (int)(i - row * per_row) * V;
            const uint8_t* p = x + (row * ldx + col) * SIZE;
            if (col + V <= K) {
                const u32x4 t = *(const u32x4_any*)p;
                v[u] = make_uint4(t.x, t.y, t.z, t.w);
            } else {
                uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (col + e < K) {
                        if constexpr (DT == F8MI_FP32) w[e] = ((const uint32_t*)p)[e];
                        else w[e >> 1] |= (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1));
                    }
                v[u] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    const FewWeight<NT> weight(W, sw_all, N, n0);
    v8i fw[DEPTH][NT];
    uint32_t fsw[DEPTH];
    auto load = [&](int d, int s) __attribute__((always_inline)) { weight.load(min(s, s1 - 1), fw[d], fsw[d]); };
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) load(d, s0 + d);
    }
#pragma unroll
    for (int u = 0; u < PIECES; u++) {
        const uint32_t i = u * FEW_THREADS + threadIdx.x;
        if (u * FEW_THREADS >= items) break;  // the same for every lane
        const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        uint32_t m = 0u;
#pragma unroll
        for (int e = 0; e < 4; e++) m = DT == F8MI_FP32 ? max(m, w[e] & 0x7fffffffu) : absmax16x2(w[e], m);
        if constexpr (DT != F8MI_FP32) m = fold16(m);
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, true));  // row_ror 1, 2, 4, 8
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, true));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, true));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, true));
        if constexpr (DT == F8MI_FP32) m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        const uint32_t bits = __float_as_uint(abs_bits_to_float(m, DT));
        const float f = block_factor(bits);
        if (i < items) {
            const uint32_t row = i / per_row, at = i - row * per_row;
            uint32_t c[2] = {0u, 0u};
#pragma unroll
            for (int h = 0; h < V / 4; h++) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (DT == F8MI_FP32) e[j] = __uint_as_float(w[j]);
                    else {
                        const uint32_t b = (j & 1) ? w[2 * h + j / 2] >> 16 : w[2 * h + j / 2] & 0xffffu;
                        e[j] = DT == F8MI_BF16 ? bf16_bits_to_float(b) : fp16_bits_to_float(b);
                    }
                }
                c[h] = cvt4_fp8<F8MI_E4M3FN>(e[0] * f, e[1] * f, e[2] * f, e[3] * f);
            }
            uint8_t* dst = x8 + row * pitch + at * V;
            if constexpr (DT == F8MI_FP32) *(uint32_t*)dst = c[0];
            else *(uint2*)dst = make_uint2(c[0], c[1]);
            if (at % (128 / V) == 0) xs[row * steps + at / (128 / V)] = (uint8_t)block_exponent(bits);
        }
    }
    lds_barrier();  // (does not wait for the weights)
    const uint8_t* px = x8 + min(lm, M - 1) * pitch + lq * 32;
    const uint8_t* ps = xs + min(lm, M - 1) * steps;

    v4f_w acc[1][NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) acc[0][nt] = (v4f_w){0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int d, int s) __attribute__((always_inline)) {
        const v8i fa = read_frag(px + s * 128, px + s * 128 + 16);
        const uint32_t sa = ps[s];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) acc[0][nt] = few_mfma_at<0>(fw[d][nt], fa, acc[0][nt], fsw[d] >> (8 * nt), sa);
    };
    int s = s0;
    for (; s + DEPTH < s1; s += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            multiply(d, s + d);
            load(d, s + DEPTH + d);
        }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (s + d < s1) multiply(d, s + d);
    few_finish<DT, 1, NT>(acc, part, M, N, n0, C, ldc, bias);
}

template <int C_DT, int MT, int NT, int DEPTH>
static int launch_few4(const BlockGemm& g) {
    const dim3 grid((unsigned)((g.N + 16 * NT - 1) / (16 * NT)), (unsigned)((g.M + 16 * MT - 1) / (16 * MT)));
    hipLaunchKernelGGL((block_gemm_few_kernel<C_DT, MT, NT, DEPTH>), grid, dim3(FEW_THREADS), 0, g.stream, g.A, g.a_unit(), g.sa, g.sa_ld(), g.Bt, g.sb, g.M, g.N, g.K, g.C, g.ldc, g.bias);
    return check_hip(hipGetLastError(), "block-scaled gemm (few rows) kernel launch");
}
// no more slots than a wave has steps: they would hold registers for nothing
template <int C_DT, int MT, int NT>
static int launch_few3(const BlockGemm& g) {
    constexpr int DEPTH = few_depth(MT);
    const int steps = (g.K / 128 + FEW_WAVES - 1) / FEW_WAVES;  // of the wave that has most
    if constexpr (DEPTH > 1)
        if (steps <= 1) return launch_few4<C_DT, MT, NT, 1>(g);
    if constexpr (DEPTH > 2)
        if (steps <= 2 || (MT == 2 && steps <= 4 && g.N > 32 * cu_count())) return launch_few4<C_DT, MT, NT, 2>(g);
    return launch_few4<C_DT, MT, NT, DEPTH>(g);
}
template <int C_DT>
static int launch_few2(const BlockGemm& g) {
    if (g.M > 64) return launch_few3<C_DT, 8, 2>(g);  // the weight is read once per 128 rows
    if (g.M > 32) return launch_few3<C_DT, 4, 2>(g);
    if (g.M > 16) return launch_few3<C_DT, 2, 2>(g);
    if (g.N <= 16 * cu_count()) return launch_few3<C_DT, 1, 1>(g);  // 32 columns a workgroup would leave half of the CUs without one
    return launch_few3<C_DT, 1, 2>(g);
}
int launch_block_few(const BlockGemm& g) {
    if (g.c_dtype == F8MI_BF16) return launch_few2<F8MI_BF16>(g);
    if (g.c_dtype == F8MI_FP16) return launch_few2<F8MI_FP16>(g);
    return launch_few2<F8MI_FP32>(g);
}

struct FewLinear {
    const uint8_t* x;
    int64_t ldx;
    const uint8_t *w, *scales;
    int M, N, K, Kp;
    void* C;
    int64_t ldc;
    const void* bias;
    hipStream_t stream;
};
template <int DT, int NT, int DEPTH>
static int launch_few_linear3(const FewLinear& a) {
    hipLaunchKernelGGL((block_linear_few_kernel<DT, NT, DEPTH>), dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT))), dim3(FEW_THREADS),
                       (size_t)a.M * (a.Kp + FEW_LDS_PAD + a.Kp / 128), a.stream, a.x, a.ldx, a.w, a.scales, a.M, a.N, a.K, a.Kp, a.C, a.ldc, a.bias);
    return check_hip(hipGetLastError(), "block-scaled few-row linear kernel launch");
}
template <int DT, int NT>
static int launch_few_linear2(const FewLinear& a) {
    constexpr int DEPTH = few_cast_depth(NT, DT);
    const int steps = (a.Kp / 128 + FEW_WAVES - 1) / FEW_WAVES;
    if (steps <= 1) return launch_few_linear3<DT, NT, 1>(a);
    if constexpr (DEPTH > 2)
        if (steps <= 2) return launch_few_linear3<DT, NT, 2>(a);
    return launch_few_linear3<DT, NT, DEPTH>(a);
}
template <int DT>
static int launch_few_linear(const FewLinear& a) {
    // 32 columns a workgroup where that leaves every CU with one (each converts all of x), else 16
    if (a.N > 32 * cu_count()) return launch_few_linear2<DT, 2>(a);
    return launch_few_linear2<DT, 1>(a);
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int f8mi_block_linear_few_rows(const void* x, int64_t ldx, int dtype, const void* w, const void* w_scales, int64_t m, int64_t n, int64_t k, void* c, int64_t ldc,
                                          const void* bias_dev, void* stream) {
    if (dtype < 0 || dtype > 2) { set_error("f8mi_block_linear_few_rows: unknown dtype code %d", dtype); return F8MI_ERR_INVALID_ARG; }
    if (m < 0 || n < 0 || k < 0 || (ldx < k && ldx != 0) || ldc < n) { set_error("f8mi_block_linear_few_rows: bad shape m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k); return F8MI_ERR_INVALID_ARG; }
    if (m == 0 || n == 0) return F8MI_OK;
    const int64_t kp = f8mi_padded_k(k);
    if (m > 16 || k < 1 || m * kp > F8MI_FEW_ROWS_ELEMS || n > 0x7fffff00LL) { set_error("f8mi_block_linear_few_rows: at most 16 rows and %d activations, padded (m=%lld k=%lld)", F8MI_FEW_ROWS_ELEMS, (long long)m, (long long)k); return F8MI_ERR_UNSUPPORTED; }
    if (!x || !w || !w_scales || !c) { set_error("f8mi_block_linear_few_rows: null pointer"); return F8MI_ERR_INVALID_ARG; }
    if ((uintptr_t)w % 16 != 0 || (uintptr_t)w_scales % 16 != 0) { set_error("f8mi_block_linear_few_rows: weight and scales are 16-byte aligned"); return F8MI_ERR_INVALID_ARG; }
    const FewLinear a{(const uint8_t*)x, ldx, (const uint8_t*)w, (const uint8_t*)w_scales, (int)m, (int)n, (int)k, (int)kp, c, ldc, bias_dev, (hipStream_t)stream};
    ProfScope prof(F8MI_K_GEMM, 2.0 * (double)m * (double)n * (double)k, a.stream);
    if (dtype == F8MI_BF16) return launch_few_linear<F8MI_BF16>(a);
    if (dtype == F8MI_FP16) return launch_few_linear<F8MI_FP16>(a);
    return launch_few_linear<F8MI_FP32>(a);
}
