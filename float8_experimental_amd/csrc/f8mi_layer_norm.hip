// Layer norm over the last dimension: y = (x - mean) * rstd * w + b with rstd = 1 / sqrt(var + eps), and its backward pass
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  g = dy * w,  xhat = (x - mean) * rstd,
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy.
// HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx.  A row stays in the registers of T lanes between its
// first read and its last use (mean first, then the squares of what is left of it: no cancellation); a workgroup takes every
// (number of workgroups)-th row, so that w and b are read once and, backward, a lane sums the columns it owns over its rows in
// registers.  Backward's workgroups write those sums, fp32, and a second launch adds them in a fixed order.  Statistics and sums are fp32.
//
// Measured, both passes, of the bytes of x, y, x, dy and dx: 8192 rows of 4096 bf16 73 us (4.6 TB/s; a copy: 4.9), 4099 of 4097 fp32 77 us (4.4), 4096 of 8192
// bf16 87 us (3.9), 12252 of 15170 fp32 784 us (4.7); the launches, the first rows' latency and the sums' rows are what is left at these sizes.
//
// Rows that do not fit (backward more than 16384 values, forward those whose parameters do not fit in LDS or more than 32768 of 16 bits, 16384 of fp32)
// are read once for each statistic and once for the result, out of the L2 after the first time, and the column sums have a kernel of their own:
// 1683 us where the rows of 15170 fp32 values above now take 784.
#include <algorithm>

#include "f8mi_row.h"

namespace f8mi {

// Mean and sum of squares about it, of the T lanes of a row that hold VPT pieces each.  A wave finds its own (in two passes over its
// registers, so nothing cancels), and those of the waves are put together: the squares about the common mean are a wave's own plus count * (mean of
// the wave - mean)^2.  One barrier a row.
template <int T, int VPT, int V>
__device__ __forceinline__ int wave_count(int wave, int cols) {  // values of the row in this wave of it
    int n = 0;
#pragma unroll
    for (int p = 0; p < VPT; p++) n += min(max(cols - (p * T + wave * 64) * V, 0), 64 * V);
    return n;
}
// a / n by inv, 1 / n rounded: the rounded quotient, where the product alone is an ulp off for one n in seven.  The mean of a constant row is then its
// value: an ulp of a large one, squared, would be its variance.
__device__ __forceinline__ float quotient(float a, float n, float inv) {
    const float q = a * inv;
    return __builtin_fmaf(__builtin_fmaf(-q, n, a), inv, q);
}
template <int T, int VPT, int V>
__device__ __forceinline__ void row_moments(float& mean, float& m2, int cols, float inv_cols, float2* slots) {
    if constexpr (T > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slots[wave] = make_float2(mean, m2);
        __syncthreads();
        const int first = wave / (T / 64) * (T / 64);
        float total = 0.f;
#pragma unroll 4
        for (int i = 0; i < T / 64; i++) total = __builtin_fmaf(slots[first + i].x, (float)wave_count<T, VPT, V>(i, cols), total);
        mean = quotient(total, (float)cols, inv_cols);
        m2 = 0.f;
#pragma unroll 4
        for (int i = 0; i < T / 64; i++) {
            const float2 w = slots[first + i];
            const float d = w.x - mean, n = (float)wave_count<T, VPT, V>(i, cols);
            m2 += n > 0.f ? __builtin_fmaf(d * d, n, w.y) : 0.f;  // (the square of a large mean is infinite, and zero times that a NaN)
        }
    }
}

// Rows of one 16-byte piece a lane have the parameters in registers (64 a lane up to 512 lanes, so that a CU holds 2048).  Longer ones have up to four
// pieces and the parameters in LDS, in their own type, which leaves registers to have the next row on its way while this one's sums are
// waited for (2048 rows of 8192 fp32 values, both passes: 117 -> 77 us, of 16384 bf16 values 118 -> 99).
constexpr int LN_ROW_LANES = 1024;
constexpr int ln_threads(int t) { return t < 256 ? 256 : t; }
constexpr int ln_waves_a_simd(int t, int vpt) { return t < LN_ROW_LANES && vpt == 1 ? 8 : 4; }
constexpr int ln_backward_threads(int t, int vpt) { return vpt > 1 ? t : LN_ROW_LANES; }
// Rows asked for ahead, forward: two where a lone workgroup's rows are short for the time a load takes (4096 rows of 8192 bf16: 39.5 us with one, 37.5 with two).
constexpr int ln_ahead(int t, int vpt) { return t == LN_ROW_LANES && vpt < 3 ? 2 : 1; }

// T lanes a row, VPT pieces of 16 bytes a lane (only the last of them can lie past the end of the row: ln_shape)
template <int DT, int PT, int T, int VPT>
__global__ __launch_bounds__(ln_threads(T), ln_waves_a_simd(T, VPT)) void layer_norm_kernel(const uint8_t* __restrict__ x, int64_t ld, int64_t rows, int cols, const void* __restrict__ weight,
                                                                   const void* __restrict__ bias, float eps, uint8_t* __restrict__ y, float2* __restrict__ stats) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, GROUPS = ln_threads(T) / T, AHEAD = ln_ahead(T, VPT);
    constexpr bool SHARED = VPT > 1;
    __shared__ float2 slots[2][ln_threads(T) / 64];
    extern __shared__ uint4 ln_shared[];
    const int t = threadIdx.x % T, group = __builtin_amdgcn_readfirstlane(threadIdx.x / T);
    const LnLane<T, VPT, V> lane(t, cols);
    const float inv_cols = 1.0f / (float)cols;
    const int64_t stride = (int64_t)gridDim.x * GROUPS, first = (int64_t)blockIdx.x * GROUPS;
    uint4 next[AHEAD][VPT];  // rows after this one: asked for before this one's sums have to wait for each other
    auto fetch = [&](uint4 (&q)[VPT], int64_t row) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < VPT; p++) q[p] = row < rows ? lane.template load<DT>(x + row * ld * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) fetch(next[i], first + i * stride + group);
    LnShared<PT, V> ws{ln_shared, (cols + V - 1) / V}, bs{ln_shared + ws.pieces * ws.PARTS, ws.pieces};
    float w[V], b[V];
    if constexpr (SHARED) {
        ws.fill(weight, cols, 1.f);
        bs.fill(bias, cols, 0.f);
        __syncthreads();
    } else {
        ln_param<PT, V, int>(weight, lane.last, cols, 1.f, w);
        ln_param<PT, V, int>(bias, lane.last, cols, 0.f, b);
    }
    const float count = (float)max(wave_count<T, VPT, V>(t >> 6, cols), 1), inv_count = 1.0f / count;
    auto one = [&](uint4 (&ahead)[VPT], int64_t row, float2* slot) __attribute__((always_inline)) {
        uint4 q[VPT];  // the row as it came: unpacking it again costs less than registers that keep waves from running
#pragma unroll
        for (int p = 0; p < VPT; p++) q[p] = ahead[p];
        if (row - group + AHEAD * stride < rows) fetch(ahead, row + AHEAD * stride);
        float s = 0.f, v[V];
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            ln_unpack<DT>(q[p], v);
#pragma unroll
            for (int i = 0; i < V; i++) s += T == 64 || lane.has(p, i) ? v[i] : 0.f;
        }
        float mean = quotient(wave_sum(s), count, inv_count);
        s = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            set_apart<DT>(q[p]);
            ln_unpack<DT>(q[p], v);
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[i] -= mean;
                if (lane.has(p, i)) s = __builtin_fmaf(v[i], v[i], s);
            }
        }
        s = wave_sum(s);
        row_moments<T, VPT, V>(mean, s, cols, inv_cols, slot);
        const float rstd = 1.0f / __builtin_sqrtf(s * inv_cols + eps);
        if (row >= rows) return;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            set_apart<DT>(q[p]);
            ln_unpack<DT>(q[p], v);
            if constexpr (SHARED) {
                ws.read(p * T + t, w);
                bs.read(p * T + t, b);
            }
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = __builtin_fmaf((v[i] - mean) * rstd, w[i], b[i]);
            lane.template store<DT>(y + row * cols * SIZE, p, cols, v);
        }
        if (stats && t == 0) stats[row] = make_float2(mean, rstd);
    };
    int parity = 0;
    for (int64_t r0 = first; r0 < rows; r0 += AHEAD * stride, parity ^= 1) {
        one(next[0], r0 + group, slots[AHEAD == 1 ? parity : 0]);
        if constexpr (AHEAD == 2)
            if (r0 + stride < rows) one(next[1], r0 + stride + group, slots[1]);
    }
}

template <int DT, int PT, int T, int VPT>
__global__ __launch_bounds__(ln_backward_threads(T, VPT), 4) void layer_norm_backward_kernel(const uint8_t* __restrict__ dy, int64_t ld_dy, const uint8_t* __restrict__ x, int64_t ld, int64_t rows, int cols,
                                                                            const void* __restrict__ weight, const float2* __restrict__ stats, uint8_t* __restrict__ dx,
                                                                            float* __restrict__ partial) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, GROUPS = ln_backward_threads(T, VPT) / T;
    constexpr bool SHARED = VPT > 1;
    __shared__ float2 slots[2][ln_backward_threads(T, VPT) / 64];
    __shared__ float sums[GROUPS > 1 ? (GROUPS - 1) * T * 2 * V : 1];
    extern __shared__ uint4 ln_shared[];
    const int t = threadIdx.x % T, group = __builtin_amdgcn_readfirstlane(threadIdx.x / T);
    const LnLane<T, VPT, V> lane(t, cols);
    const float inv_cols = 1.0f / (float)cols;
    const int64_t stride = (int64_t)gridDim.x * GROUPS, first = (int64_t)blockIdx.x * GROUPS;
    struct Next {  // of rows after this one: asked for before this one's sums have to wait for each other
        uint4 x[VPT], g[VPT];
        float2 stats;
    } next;
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
        const bool in = row < rows;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            next.x[p] = in ? lane.template load<DT>(x + row * ld * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
            next.g[p] = in ? lane.template load<DT>(dy + row * ld_dy * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);
        }
        next.stats = in ? stats[row] : make_float2(0.f, 0.f);
    };
    fetch(first + group);
    LnShared<PT, V> ws{ln_shared, (cols + V - 1) / V};
    float w[V], dw[VPT][V], db[VPT][V];
    if constexpr (SHARED) {
        ws.fill(weight, cols, 1.f);
        __syncthreads();
    } else {
        ln_param<PT, V, int>(weight, lane.last, cols, 1.f, w);
    }
#pragma unroll
    for (int p = 0; p < VPT; p++)
#pragma unroll
        for (int i = 0; i < V; i++) dw[p][i] = db[p][i] = 0.f;
    int parity = 0;
    for (int64_t r0 = first; r0 < rows; r0 += stride, parity ^= 1) {
        const int64_t row = r0 + group;
        uint4 qx[VPT], qg[VPT];
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            qx[p] = next.x[p];
            qg[p] = next.g[p];
        }
        const float2 st = next.stats;
        if (r0 + stride < rows) fetch(row + stride);
        float xh[V], g[V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);  // one piece at a time: unpacked together they do not fit in registers
            ln_unpack<DT>(qx[p], xh);
            ln_unpack<DT>(qg[p], g);
            if constexpr (SHARED) ws.read(p * T + t, w);
#pragma unroll
            for (int i = 0; i < V; i++) {
                xh[i] = (xh[i] - st.x) * st.y;
                if (!lane.has(p, i)) (T > 64 ? g[i] : xh[i]) = 0.f;  // (past the end of a row g is zero, but xh may be infinite)
                dw[p][i] = __builtin_fmaf(g[i], xh[i], dw[p][i]);
                db[p][i] += g[i];
                g[i] *= w[i];
                s1 += g[i];
                s2 = __builtin_fmaf(g[i], xh[i], s2);
                asm volatile("" : "+v"(dw[p][i]), "+v"(db[p][i]));  // added here: behind the barrier, where the compiler moves it, everything waits for it (8192 values: 98 -> 87 us)
            }
        }
        if (!dx) continue;
        row_sums<T>(s1, s2, slots[parity]);
        s1 *= inv_cols;
        s2 *= inv_cols;
        if (row >= rows) continue;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);
            set_apart<DT>(qx[p]);
            set_apart<DT>(qg[p]);
            ln_unpack<DT>(qx[p], xh);
            ln_unpack<DT>(qg[p], g);
            if constexpr (SHARED) ws.read(p * T + t, w);
#pragma unroll
            for (int i = 0; i < V; i++) {
#pragma clang fp contract(off)  // what two lanes store has the same bits
                g[i] = st.y * __builtin_fmaf((xh[i] - st.x) * st.y, -s2, g[i] * w[i] - s1);
            }
            lane.template store<DT>(dx + row * cols * SIZE, p, cols, g);
        }
    }
    if (!partial) return;
    // one row of sums a workgroup: dw, then db
    float* out = partial + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int p = 0; p < VPT; p++) {
        if constexpr (GROUPS > 1) {
            __syncthreads();
            if (group > 0)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    sums[(((group - 1) * 2 + 0) * V + i) * T + t] = dw[p][i];
                    sums[(((group - 1) * 2 + 1) * V + i) * T + t] = db[p][i];
                }
            __syncthreads();
            if (group > 0) continue;
#pragma unroll 1
            for (int k = 0; k < GROUPS - 1; k++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    dw[p][i] += sums[((k * 2 + 0) * V + i) * T + t];
                    db[p][i] += sums[((k * 2 + 1) * V + i) * T + t];
                }
        }
        const int col = lane.col(p);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane.has(p, i)) {
                out[col + i] = dw[p][i];
                out[cols + col + i] = db[p][i];
            }
    }
}

// ---- rows that do not fit in registers: a workgroup a row
constexpr int LN_WIDE_THREADS = 1024;

template <int DT, int PT>
__global__ __launch_bounds__(LN_WIDE_THREADS) void layer_norm_wide_kernel(const uint8_t* __restrict__ x, int64_t ld, int64_t cols, const void* __restrict__ weight,
                                                                          const void* __restrict__ bias, float eps, uint8_t* __restrict__ y, float2* __restrict__ stats) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    __shared__ float2 slots[2][LN_WIDE_THREADS / 64];
    const uint8_t* row = x + blockIdx.x * ld * SIZE;
    float v[V], s = 0.f, none = 0.f;
    for (int64_t col = threadIdx.x * V; col < cols; col += LN_WIDE_THREADS * V) {
        ln_unpack<DT>(ln_load<DT, int64_t>(row, col, cols), v);
#pragma unroll
        for (int i = 0; i < V; i++) s += v[i];
    }
    row_sums<LN_WIDE_THREADS>(s, none, slots[0]);
    const float mean = s / (float)cols;
    s = 0.f;
    for (int64_t col = threadIdx.x * V; col < cols; col += LN_WIDE_THREADS * V) {
        ln_unpack<DT>(ln_load<DT, int64_t>(row, col, cols), v);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (col + i < cols) s = __builtin_fmaf(v[i] - mean, v[i] - mean, s);
    }
    row_sums<LN_WIDE_THREADS>(s, none, slots[1]);
    const float rstd = 1.0f / __builtin_sqrtf(s / (float)cols + eps);
    for (int64_t col = threadIdx.x * V; col < cols; col += LN_WIDE_THREADS * V) {
        float w[V], b[V];
        ln_unpack<DT>(ln_load<DT, int64_t>(row, col, cols), v);
        ln_param<PT, V, int64_t>(weight, col, cols, 1.f, w);
        ln_param<PT, V, int64_t>(bias, col, cols, 0.f, b);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = __builtin_fmaf((v[i] - mean) * rstd, w[i], b[i]);
        ln_store<DT, int64_t>(y + blockIdx.x * cols * SIZE, col, cols, v);
    }
    if (stats && threadIdx.x == 0) stats[blockIdx.x] = make_float2(mean, rstd);
}

template <int DT, int PT>
__global__ __launch_bounds__(LN_WIDE_THREADS) void layer_norm_backward_wide_kernel(const uint8_t* __restrict__ dy, int64_t ld_dy, const uint8_t* __restrict__ x, int64_t ld, int64_t cols,
                                                                                   const void* __restrict__ weight, const float2* __restrict__ stats, uint8_t* __restrict__ dx) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    __shared__ float2 slots[LN_WIDE_THREADS / 64];
    const uint8_t *row = x + blockIdx.x * ld * SIZE, *grow = dy + blockIdx.x * ld_dy * SIZE;
    const float2 st = stats[blockIdx.x];
    float xv[V], g[V], w[V], s1 = 0.f, s2 = 0.f;
    for (int64_t col = threadIdx.x * V; col < cols; col += LN_WIDE_THREADS * V) {
        ln_unpack<DT>(ln_load<DT, int64_t>(row, col, cols), xv);
        ln_unpack<DT>(ln_load<DT, int64_t>(grow, col, cols), g);
        ln_param<PT, V, int64_t>(weight, col, cols, 1.f, w);
#pragma unroll
        for (int i = 0; i < V; i++) {
            g[i] *= w[i];
            s1 += g[i];
            if (col + i < cols) s2 = __builtin_fmaf(g[i], (xv[i] - st.x) * st.y, s2);  // (past the end of a row xhat may be infinite)
        }
    }
    row_sums<LN_WIDE_THREADS>(s1, s2, slots);
    s1 /= (float)cols;
    s2 /= (float)cols;
    for (int64_t col = threadIdx.x * V; col < cols; col += LN_WIDE_THREADS * V) {
        ln_unpack<DT>(ln_load<DT, int64_t>(row, col, cols), xv);
        ln_unpack<DT>(ln_load<DT, int64_t>(grow, col, cols), g);
        ln_param<PT, V, int64_t>(weight, col, cols, 1.f, w);
#pragma unroll
        for (int i = 0; i < V; i++) g[i] = st.y * (g[i] * w[i] - s1 - (xv[i] - st.x) * st.y * s2);
        ln_store<DT, int64_t>(dx + blockIdx.x * cols * SIZE, col, cols, g);
    }
}

// column sums of dy * xhat and dy: 256 lanes' columns of `chunk` rows a workgroup
template <int DT>
__global__ __launch_bounds__(256) void layer_norm_columns_kernel(const uint8_t* __restrict__ dy, int64_t ld_dy, const uint8_t* __restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                                 const float2* __restrict__ stats, int64_t chunk, float* __restrict__ partial) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    const int64_t col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (col >= cols) return;
    float dw[V], db[V], xv[V], g[V];
#pragma unroll
    for (int i = 0; i < V; i++) dw[i] = db[i] = 0.f;
    const int64_t end = std::min<int64_t>(rows, (blockIdx.y + 1) * chunk);
#pragma unroll 4
    for (int64_t r = blockIdx.y * chunk; r < end; r++) {
        const float2 st = stats[r];
        ln_unpack<DT>(ln_load<DT, int64_t>(x + r * ld * SIZE, col, cols), xv);
        ln_unpack<DT>(ln_load<DT, int64_t>(dy + r * ld_dy * SIZE, col, cols), g);
#pragma unroll
        for (int i = 0; i < V; i++) {
            dw[i] = __builtin_fmaf(g[i], (xv[i] - st.x) * st.y, dw[i]);
            db[i] += g[i];
        }
    }
    float* out = partial + (int64_t)blockIdx.y * 2 * cols;
#pragma unroll
    for (int i = 0; i < V; i++)
        if (col + i < cols) {
            out[col + i] = dw[i];
            out[cols + col + i] = db[i];
        }
}

// Adds the `parts` rows of sums: 64 of the 2 * cols columns a workgroup, a wave every 16th row of them
constexpr int LN_FINISH_WAVES = 16;
__global__ __launch_bounds__(64 * LN_FINISH_WAVES) void layer_norm_finish_kernel(const float* __restrict__ partial, int64_t parts, int64_t cols, void* __restrict__ dw,
                                                                                 void* __restrict__ db, int p_dtype) {
    __shared__ float red[LN_FINISH_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (col < 2 * cols) {
#pragma unroll 8
        for (int64_t i = wave; i < parts; i += LN_FINISH_WAVES) s += partial[i * 2 * cols + col];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= 2 * cols) return;
    s = red[0][lane];
#pragma unroll
    for (int i = 1; i < LN_FINISH_WAVES; i++) s += red[i][lane];
    void* out = col < cols ? dw : db;
    const int64_t at = col < cols ? col : col - cols;
    if (!out) return;
    if (p_dtype == F8MI_FP32) ((float*)out)[at] = s;
    else if (p_dtype == F8MI_BF16) ((uint16_t*)out)[at] = (uint16_t)pack2<F8MI_BF16>(s, 0.f);
    else ((uint16_t*)out)[at] = (uint16_t)pack2<F8MI_FP16>(s, 0.f);
}

struct LnArgs {
    const uint8_t *dy, *x;
    int64_t ld_dy, ld, rows, cols;
    const void *weight, *bias;
    float eps;
    uint8_t* out;  // y, dx
    float2* stats;
    float* partial;
    int64_t parts;  // workgroups of the backward kernel
    hipStream_t stream;
};

// Lanes of a row and pieces a lane, by the number of 16-byte pieces of a row; 0: does not fit.  Forward's weight and bias have to fit in LDS
// with it, in backward the column sums of 16-bit rows take the registers of a third piece (with one it spilled and was no faster than by columns: 2048
// rows of 20000 bf16 values, both passes, 169 us, 8192 of them 581).
struct LnShape {
    int t, vpt;
};
constexpr int LN_MAX_LDS = (160 << 10) - 512;
static int64_t ln_pieces(int64_t cols, int dtype) { return (cols + (dtype == F8MI_FP32 ? 3 : 7)) / (dtype == F8MI_FP32 ? 4 : 8); }
// of the parameters that a workgroup of 1024 lanes keeps
static int64_t ln_lds(int64_t cols, int dtype, int p_dtype, bool backward) { return ln_pieces(cols, dtype) * 16 * (dtype == p_dtype ? 1 : 2) * (backward ? 1 : 2); }
static LnShape ln_shape(int64_t cols, int dtype, int p_dtype, bool backward) {
    const int64_t pieces = ln_pieces(cols, dtype);
    for (int t = 64; t <= LN_ROW_LANES; t *= 2)
        if (pieces <= t) return {t, 1};
    // two workgroups a CU, and fewer idle lanes (both passes, us, 1024 lanes / 512: 4099 rows of 4097 96 / 78, 8192 of 4352 169 / 142, 4096 of 5120 97 / 85,
    // 4096 of 6144 108 / 100, 2048 of 4100 71 / 69, 16384 of 6000 398 / 402)
    if (dtype == F8MI_FP32 && pieces <= 3 * 512) return {512, 3};
    const int64_t vpt = (pieces + LN_ROW_LANES - 1) / LN_ROW_LANES;
    if (vpt > (backward && dtype != F8MI_FP32 ? 2 : 4) || ln_lds(cols, dtype, p_dtype, backward) > LN_MAX_LDS) return {0, 0};
    return {LN_ROW_LANES, (int)vpt};
}
// Workgroups of `threads` lanes, `per_cu` of them on every CU, no more than the rows need
static int64_t ln_workgroups(LnShape s, int64_t rows, int threads, int per_cu) {
    const int64_t groups = threads / s.t;
    return std::min<int64_t>((int64_t)cu_count() * per_cu, (rows + groups - 1) / groups);
}
static int64_t ln_chunk_rows(int64_t rows, int64_t cols, int dtype) {  // of the column kernel for wide rows: 1024 workgroups or so
    const int64_t strips = (cols + (dtype == F8MI_FP32 ? 1023 : 2047)) / (dtype == F8MI_FP32 ? 1024 : 2048), want = std::max<int64_t>(1, 1024 / strips);
    return std::max<int64_t>(8, (rows + want - 1) / want);
}
static int64_t ln_parts(int64_t rows, int64_t cols, int dtype) {
    const LnShape s = ln_shape(cols, dtype, F8MI_FP32, true);  // (a weight of fewer bits fits where one of fp32 does, and no row of fp32 ones does not)
    if (s.t) return ln_workgroups(s, rows, ln_backward_threads(s.t, s.vpt), LN_ROW_LANES / ln_backward_threads(s.t, s.vpt));
    const int64_t chunk = ln_chunk_rows(rows, cols, dtype);
    return (rows + chunk - 1) / chunk;
}

template <int DT, int PT, int T, int VPT>
static int launch_ln(const LnArgs& a, bool backward) {
    const int64_t lds = VPT > 1 ? ln_lds(a.cols, DT, PT, backward) : 0;
    if (backward) {
        if constexpr (VPT <= (DT == F8MI_FP32 ? 4 : 2)) {  // (ln_shape)
            const auto kernel = layer_norm_backward_kernel<DT, PT, T, VPT>;
            if constexpr (VPT > 1) {
                static std::atomic<uint64_t> allowed{0};
                if (int rc = allow_big_lds(kernel, LN_MAX_LDS, allowed)) return rc;
            }
            hipLaunchKernelGGL(kernel, dim3((unsigned)a.parts), dim3(ln_backward_threads(T, VPT)), (unsigned)lds, a.stream, a.dy, a.ld_dy, a.x, a.ld, a.rows, (int)a.cols, a.weight, a.stats, a.out, a.partial);
        }
        return check_hip(hipGetLastError(), "layer norm backward kernel launch");
    }
    const auto kernel = layer_norm_kernel<DT, PT, T, VPT>;
    if constexpr (VPT > 1) {
        static std::atomic<uint64_t> allowed{0};
        if (int rc = allow_big_lds(kernel, LN_MAX_LDS, allowed)) return rc;
    }
    const int per_cu = ln_waves_a_simd(T, VPT) * 256 / ln_threads(T);
    hipLaunchKernelGGL(kernel, dim3((unsigned)ln_workgroups({T, VPT}, a.rows, ln_threads(T), per_cu)), dim3(ln_threads(T)), (unsigned)lds, a.stream, a.x, a.ld, a.rows, (int)a.cols, a.weight,
                       a.bias, a.eps, a.out, a.stats);
    return check_hip(hipGetLastError(), "layer norm kernel launch");
}
template <int DT, int PT>
static int launch_ln_wide(const LnArgs& a, bool backward) {
    if (!backward) {
        hipLaunchKernelGGL((layer_norm_wide_kernel<DT, PT>), dim3((unsigned)a.rows), dim3(LN_WIDE_THREADS), 0, a.stream, a.x, a.ld, a.cols, a.weight, a.bias, a.eps, a.out, a.stats);
        return check_hip(hipGetLastError(), "layer norm kernel launch");
    }
    if (a.out)
        hipLaunchKernelGGL((layer_norm_backward_wide_kernel<DT, PT>), dim3((unsigned)a.rows), dim3(LN_WIDE_THREADS), 0, a.stream, a.dy, a.ld_dy, a.x, a.ld, a.cols, a.weight, a.stats, a.out);
    if (a.partial) {
        const unsigned strips = (unsigned)((a.cols + 256 * Ln<DT>::V - 1) / (256 * Ln<DT>::V));
        hipLaunchKernelGGL(layer_norm_columns_kernel<DT>, dim3(strips, (unsigned)a.parts), dim3(256), 0, a.stream, a.dy, a.ld_dy, a.x, a.ld, a.rows, a.cols, a.stats,
                           ln_chunk_rows(a.rows, a.cols, DT), a.partial);
    }
    return check_hip(hipGetLastError(), "layer norm backward kernel launch");
}
template <int DT, int PT>
static int launch_ln_by_size(const LnArgs& a, bool backward) {
    const LnShape s = ln_shape(a.cols, DT, PT, backward);
    if (s.t == 64) return launch_ln<DT, PT, 64, 1>(a, backward);
    if (s.t == 128) return launch_ln<DT, PT, 128, 1>(a, backward);
    if (s.t == 256) return launch_ln<DT, PT, 256, 1>(a, backward);
    if (s.t == 512 && s.vpt == 1) return launch_ln<DT, PT, 512, 1>(a, backward);
    if constexpr (DT == F8MI_FP32)
        if (s.t == 512) return launch_ln<DT, PT, 512, 3>(a, backward);
    if (s.vpt == 1) return launch_ln<DT, PT, LN_ROW_LANES, 1>(a, backward);
    if (s.vpt == 2) return launch_ln<DT, PT, LN_ROW_LANES, 2>(a, backward);
    if (s.vpt == 3) return launch_ln<DT, PT, LN_ROW_LANES, 3>(a, backward);
    if (s.vpt == 4) return launch_ln<DT, PT, LN_ROW_LANES, 4>(a, backward);
    return launch_ln_wide<DT, PT>(a, backward);
}
static int launch_ln_by_type(int dtype, int p_dtype, const LnArgs& a, bool backward) {
    if (dtype == F8MI_BF16) return p_dtype == F8MI_FP32 ? launch_ln_by_size<F8MI_BF16, F8MI_FP32>(a, backward) : launch_ln_by_size<F8MI_BF16, F8MI_BF16>(a, backward);
    if (dtype == F8MI_FP16) return p_dtype == F8MI_FP32 ? launch_ln_by_size<F8MI_FP16, F8MI_FP32>(a, backward) : launch_ln_by_size<F8MI_FP16, F8MI_FP16>(a, backward);
    return launch_ln_by_size<F8MI_FP32, F8MI_FP32>(a, backward);
}

static int ln_check(const char* what, int64_t rows, int64_t cols, int dtype, int p_dtype) {
    if (dtype < 0 || dtype > 2 || (p_dtype != dtype && p_dtype != F8MI_FP32)) { set_error("%s: parameters have x's type or are fp32 (dtype codes %d, %d)", what, dtype, p_dtype); return F8MI_ERR_INVALID_ARG; }
    if (rows < 0 || cols <= 0) { set_error("%s: bad shape rows=%lld cols=%lld", what, (long long)rows, (long long)cols); return F8MI_ERR_INVALID_ARG; }
    if (rows > 0x7fffffff || cols > 0x7fffff00) { set_error("%s: dimension too large", what); return F8MI_ERR_UNSUPPORTED; }
    return F8MI_OK;
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int f8mi_layer_norm(const void* x, int64_t rows, int64_t cols, int64_t ld, int dtype, const void* weight, const void* bias, int p_dtype, float eps, void* y,
                               float* stats, void* stream) {
    if (int rc = ln_check("f8mi_layer_norm", rows, cols, dtype, p_dtype)) return rc;
    if (rows == 0) return F8MI_OK;
    if (!x || !y || ld < 0 || (ld < cols && ld != 0)) { set_error("f8mi_layer_norm: null pointer or ld=%lld < cols=%lld", (long long)ld, (long long)cols); return F8MI_ERR_INVALID_ARG; }
    if ((uintptr_t)stats % 8 != 0) { set_error("f8mi_layer_norm: statistics are 8-byte aligned pairs"); return F8MI_ERR_INVALID_ARG; }
    return launch_ln_by_type(dtype, p_dtype, {nullptr, (const uint8_t*)x, 0, ld, rows, cols, weight, bias, eps, (uint8_t*)y, (float2*)stats, nullptr, 0, (hipStream_t)stream}, false);
}

extern "C" int64_t f8mi_layer_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
    return rows <= 0 || cols <= 0 || dtype < 0 || dtype > 2 ? 0 : ln_parts(rows, cols, dtype) * 2 * cols * 4;
}

extern "C" int f8mi_layer_norm_backward(const void* dy, int64_t ld_dy, const void* x, int64_t ld, int64_t rows, int64_t cols, int dtype, const void* weight, int p_dtype,
                                        const float* stats, void* dx, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = ln_check("f8mi_layer_norm_backward", rows, cols, dtype, p_dtype)) return rc;
    if (!dx && !dweight && !dbias) return F8MI_OK;
    const bool sums = dweight || dbias;
    if (rows > 0 && (!dy || !x || !stats || ld < 0 || (ld < cols && ld != 0) || ld_dy < 0 || (ld_dy < cols && ld_dy != 0))) { set_error("f8mi_layer_norm_backward: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    if ((uintptr_t)stats % 8 != 0) { set_error("f8mi_layer_norm_backward: statistics are 8-byte aligned pairs"); return F8MI_ERR_INVALID_ARG; }
    const int64_t need = sums ? f8mi_layer_norm_workspace_bytes(rows, cols, dtype) : 0;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)) { set_error("f8mi_layer_norm_backward: workspace of %lld bytes needed", (long long)need); return F8MI_ERR_INVALID_ARG; }
    const int64_t parts = rows > 0 ? ln_parts(rows, cols, dtype) : 0;
    if (rows > 0)
        if (int rc = launch_ln_by_type(dtype, p_dtype, {(const uint8_t*)dy, (const uint8_t*)x, ld_dy, ld, rows, cols, weight, nullptr, 0.f, (uint8_t*)dx, (float2*)stats,
                                                         sums ? (float*)workspace : nullptr, parts, stream}, true)) return rc;
    if (sums)
        hipLaunchKernelGGL(layer_norm_finish_kernel, dim3((unsigned)((2 * cols + 63) / 64)), dim3(64 * LN_FINISH_WAVES), 0, stream, (const float*)workspace, parts, cols, dweight, dbias, p_dtype);
    return check_hip(hipGetLastError(), "layer norm column sum kernel launch");
}
