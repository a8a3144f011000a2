// RMS norm over the last dimension, with the addition in front of it: s = x + residual, rounded to their type, and
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps),
// y rounded once to x's type, or kept as e4m3 with a scale for each 128 values of a row (f8mi_block.h), which a product with block scales reads as
// it is.  Backward, with g = dy * w and xhat = s * rstd:
//   dx = ds + rstd * (g - xhat * mean(g * xhat))  (of the residual too),  dw = sum over rows of dy * xhat.
// What is normed is the rounded sum: it is what later layers add to, what a program that adds and norms in two steps gets, and all that backward needs beside
// rstd.  Statistics and sums are fp32 (a row whose mean square no fp32 holds gives zeros).
//
// HBM-bound, as layer norm (f8mi_layer_norm.hip), and built the same way: a row stays in the registers of T lanes between its first read and its
// last use, one barrier a row (there is one sum, where layer norm has two), the next row on its way meanwhile; a workgroup takes every (number of workgroups)-th row, so that the weight is read
// once and, backward, a lane sums the columns it owns over its rows in registers; a second launch adds the workgroups' sums in a fixed order.  The widest rows backward, three pieces a lane of 16-bit values
// and five of fp32, keep those sums in LDS and spill 20 to 112 bytes a lane all the same (1024 lanes leave each 128 registers), addresses mostly.
// Measured, out of HBM (a large copy: 5.1 - 5.4 TB/s): 8192 x 4096 bf16 with a residual and an fp32 weight forward 45 us (6.0 TB/s), backward 45 (5.9) and 4 for the sums;
// 8192 x 8192 bf16 with a residual into e4m3 78 us (6.0 TB/s); 4099 x 4097 fp32 forward 26 us (5.1 TB/s), backward 39 (5.2); 2048 x 20000 bf16 with a residual, both passes, 131 us
// (5.0 TB/s); 16 rows of 8192 into e4m3 5.5 us and one of 4096 2.5 us, latency.  16-bit rows of an odd number of values begin at odd multiples of two bytes: 8192 x 4097
// with a residual takes 132 us both ways where 4096 columns take 94.
#include <algorithm>

#include "f8mi_block.h"
#include "f8mi_row.h"

namespace f8mi {

constexpr int RMS_LANES = 1024;  // of a row, at most
constexpr int rms_threads(int t) { return t < 256 ? 256 : t; }
constexpr int rms_waves_a_simd(int t, int vpt) { return t < RMS_LANES && vpt == 1 ? 8 : 4; }
constexpr int rms_backward_threads(int t, int vpt) { return vpt > 1 ? t : RMS_LANES; }

// The sum over the T lanes of a row, in every one of them.  `slots`: a float for each wave of the workgroup, not in use elsewhere until the next
// barrier but one.
template <int T>
__device__ __forceinline__ float rms_row_sum(float a, float* slots) {
    a = wave_sum(a);
    if constexpr (T > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slots[wave] = a;
        __syncthreads();
        const int first = wave / (T / 64) * (T / 64);
        a = 0.f;
#pragma unroll 4
        for (int i = 0; i < T / 64; i++) a += slots[first + i];
    }
    return a;
}

// Pieces where blocks of 128 need them: piece p of lane t at column (p T + t) V, zeros past the end of the row (LnLane moves the last one back instead).
template <int T, int VPT, int V>
struct BlockLane {
    int t;
    __device__ __forceinline__ BlockLane(int t_, int) : t(t_) {}
    __device__ __forceinline__ int col(int p) const { return (p * T + t) * V; }
    __device__ __forceinline__ bool has(int, int) const { return true; }
    template <int DT>
    __device__ __forceinline__ uint4 load(const uint8_t* row, int p, int cols) const {
        return ln_load<DT, int>(row, col(p), cols);
    }
    template <int DT>
    __device__ __forceinline__ void store(uint8_t* row, int p, int cols, const float (&v)[V]) const {
        if (col(p) < cols) ln_store<DT, int>(row, col(p), cols, v);
    }
};
template <int DT, int T, int VPT, bool CAST>
using RmsLane = std::conditional_t<CAST, BlockLane<T, VPT, Ln<DT>::V>, LnLane<T, VPT, Ln<DT>::V>>;

struct RmsArgs {
    const uint8_t *x, *residual;
    int64_t ld, ld_res, rows, cols;
    const void* weight;
    float eps;
    uint8_t *y, *sum;          // y: or the e4m3 copy
    float* rstd;
    uint8_t* scales;           // of the e4m3 copy
    int64_t padded_rows;       // of its scales
    hipStream_t stream;
};

// V values in block scales: the maximum of their block (128 / V neighbouring lanes), 8 or 4 bytes of e4m3, and the block's exponent.
template <int V>
__device__ __forceinline__ void rms_cast(const float (&v)[V], uint32_t (&q)[V / 4], uint32_t& exponent) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < V; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, true));  // row_ror 1, 2, 4, 8
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, true));
    if constexpr (V == 4) m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    const float f = block_factor(m);
    exponent = block_exponent(m);
#pragma unroll
    for (int h = 0; h < V / 4; h++) q[h] = cvt4_fp8<F8MI_E4M3FN>(v[4 * h] * f, v[4 * h + 1] * f, v[4 * h + 2] * f, v[4 * h + 3] * f);
}

// T lanes a row, VPT pieces of 16 bytes a lane
template <int DT, int PT, int T, int VPT, bool RES, bool CAST>
__global__ __launch_bounds__(rms_threads(T), rms_waves_a_simd(T, VPT)) void rms_norm_kernel(const RmsArgs a) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, GROUPS = rms_threads(T) / T;
    constexpr bool SHARED = VPT > 1;
    __shared__ float slots[2][rms_threads(T) / 64];
    extern __shared__ uint4 rms_shared[];
    const int t = threadIdx.x % T, group = __builtin_amdgcn_readfirstlane(threadIdx.x / T), cols = (int)a.cols;
    const RmsLane<DT, T, VPT, CAST> lane(t, cols);
    const float inv_cols = 1.0f / (float)cols;
    const int64_t rows = a.rows, stride = (int64_t)gridDim.x * GROUPS, first = (int64_t)blockIdx.x * GROUPS;
    struct Next {  // the row after this one: asked for before this one's sum has to wait for the other waves
        uint4 x[VPT], r[RES ? VPT : 1];
    } next;
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            next.x[p] = row < rows ? lane.template load<DT>(a.x + row * a.ld * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (RES) next.r[p] = row < rows ? lane.template load<DT>(a.residual + row * a.ld_res * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    fetch(first + group);
    LnShared<PT, V> ws{rms_shared, (cols + V - 1) / V};
    float w[V];
    if constexpr (SHARED) {
        if constexpr (CAST) {  // pieces where the lanes have them
            for (int i = threadIdx.x; i < ws.pieces * ws.PARTS; i += blockDim.x) {
                const int part = i / ws.pieces, piece = i - part * ws.pieces;
                float one[Ln<PT>::V];
                ln_param<PT, Ln<PT>::V, int>(a.weight, piece * V + part * Ln<PT>::V, cols, 1.f, one);
                rms_shared[i] = ln_pack<PT>(one);
            }
        } else {
            ws.fill(a.weight, cols, 1.f);
        }
        __syncthreads();
    } else {
        ln_param<PT, V, int>(a.weight, CAST ? t * V : lane.col(0), cols, 1.f, w);
    }
    int parity = 0;
    for (int64_t r0 = first; r0 < rows; r0 += stride, parity ^= 1) {
        const int64_t row = r0 + group;
        uint4 q[VPT];  // the row as it is normed: unpacking it again costs less than registers that keep waves from running
        float v[V], s = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            q[p] = next.x[p];
            if constexpr (RES) {
                float r[V];
                ln_unpack<DT>(q[p], v);
                ln_unpack<DT>(next.r[p], r);
#pragma unroll
                for (int i = 0; i < V; i++) v[i] += r[i];
                q[p] = ln_pack<DT>(v);
            }
        }
        if (r0 + stride < rows) fetch(row + stride);
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            ln_unpack<DT>(q[p], v);
            if constexpr (RES)
                if (row < rows) lane.template store<DT>(a.sum + row * cols * SIZE, p, cols, v);
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane.has(p, i)) s = __builtin_fmaf(v[i], v[i], s);
        }
        s = rms_row_sum<T>(s, slots[parity]);
        const float rstd = 1.0f / __builtin_sqrtf(s * inv_cols + a.eps);
        if (row >= rows) continue;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            set_apart<DT>(q[p]);
            ln_unpack<DT>(q[p], v);
            if constexpr (SHARED) ws.read(p * T + t, w);
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = v[i] * rstd * w[i];
            if constexpr (CAST) {
                uint32_t c[V / 4], exponent;
                if (!(V == 4 || p * T * V + (t & ~15) * V < cols)) continue;  // (the 16 lanes of a block together; 32 of fp32 exchange below)
                rms_cast<V>(v, c, exponent);
                const int col = lane.col(p), block = col >> 7;
                if ((block << 7) >= cols) continue;
                uint8_t* at = a.y + ((int64_t)(col >> 6) * rows + row) * 64 + (col & 63);
                if constexpr (V == 8) *(uint2*)at = make_uint2(c[0], c[1]);
                else *(uint32_t*)at = c[0];
                if ((col & 127) == 0) a.scales[block * a.padded_rows + (row & ~(int64_t)127) + block_scale_at((int)(row & 127))] = (uint8_t)exponent;
            } else {
                lane.template store<DT>(a.y + row * cols * SIZE, p, cols, v);
            }
        }
        if (!CAST && a.rstd && t == 0) a.rstd[row] = rstd;
    }
}

struct RmsBackwardArgs {
    const uint8_t *dy, *s, *ds;
    int64_t ld_dy, ld, ld_ds, rows, cols;
    const void* weight;
    const float* rstd;
    uint8_t* dx;
    float* partial;
    int64_t parts;
    hipStream_t stream;
};

// Sums of columns in registers, of more pieces a lane than those have room for in LDS
constexpr bool rms_sums_in_lds(int dtype, int vpt) { return vpt > (dtype == F8MI_FP32 ? 3 : 2); }
template <int DT, int PT, int T, int VPT, bool DS>
__global__ __launch_bounds__(rms_backward_threads(T, VPT), 4) void rms_norm_backward_kernel(const RmsBackwardArgs a) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, GROUPS = rms_backward_threads(T, VPT) / T;
    constexpr bool SHARED = VPT > 1, IN_LDS = rms_sums_in_lds(DT, VPT);
    __shared__ float slots[2][rms_backward_threads(T, VPT) / 64];
    __shared__ float sums[GROUPS > 1 ? (GROUPS - 1) * T * V : 1];
    extern __shared__ uint4 rms_shared[];
    const int t = threadIdx.x % T, group = __builtin_amdgcn_readfirstlane(threadIdx.x / T), cols = (int)a.cols;
    const LnLane<T, VPT, V> lane(t, cols);
    const float inv_cols = 1.0f / (float)cols;
    const int64_t rows = a.rows, stride = (int64_t)gridDim.x * GROUPS, first = (int64_t)blockIdx.x * GROUPS;
    struct Next {  // of the row after this one
        uint4 s[VPT], g[VPT];
        float rstd;
    } next;
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
        const bool in = row < rows;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            next.s[p] = in ? lane.template load<DT>(a.s + row * a.ld * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
            next.g[p] = in ? lane.template load<DT>(a.dy + row * a.ld_dy * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);
        }
        next.rstd = in ? a.rstd[row] : 0.f;
    };
    fetch(first + group);
    LnShared<PT, V> ws{rms_shared, (cols + V - 1) / V};
    float4* const lds_sums = (float4*)(rms_shared + ws.pieces * ws.PARTS);  // of V columns, the four from part * 4 on, at [part][piece]; a lane's own
    float w[V], dw[IN_LDS ? 1 : VPT][V];
    if constexpr (SHARED) {
        ws.fill(a.weight, cols, 1.f);
        __syncthreads();
    } else {
        ln_param<PT, V, int>(a.weight, lane.last, cols, 1.f, w);
    }
#pragma unroll
    for (int p = 0; p < VPT; p++) {
        if constexpr (IN_LDS) {
            if (p * T + t < ws.pieces)
#pragma unroll
                for (int part = 0; part < V / 4; part++) lds_sums[part * ws.pieces + p * T + t] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) dw[p][i] = 0.f;
        }
    }
    int parity = 0;
    for (int64_t r0 = first; r0 < rows; r0 += stride, parity ^= 1) {
        const int64_t row = r0 + group;
        uint4 qs[VPT], qg[VPT], qd[DS ? VPT : 1];
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            qs[p] = next.s[p];
            qg[p] = next.g[p];
            if constexpr (DS && !IN_LDS) qd[p] = row < rows ? lane.template load<DT>(a.ds + row * a.ld_ds * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);  // needed behind the sum
        }
        const float rstd = next.rstd;
        if (r0 + stride < rows) fetch(row + stride);
        float xh[V], g[V], s2 = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);  // one piece at a time: unpacked together they do not fit in registers
            ln_unpack<DT>(qs[p], xh);
            ln_unpack<DT>(qg[p], g);
            if constexpr (SHARED) ws.read(p * T + t, w);
#pragma unroll
            for (int i = 0; i < V; i++) {
                xh[i] *= rstd;
                if (!lane.has(p, i)) g[i] = xh[i] = 0.f;
                s2 = __builtin_fmaf(g[i] * w[i], xh[i], s2);
                if constexpr (!IN_LDS) {
                    dw[p][i] = __builtin_fmaf(g[i], xh[i], dw[p][i]);
                    asm volatile("" : "+v"(dw[p][i]));  // added here, not behind the barrier
                }
            }
            if constexpr (IN_LDS)
                if (p * T + t < ws.pieces)
#pragma unroll
                    for (int part = 0; part < V / 4; part++) {
                        float4& d = lds_sums[part * ws.pieces + p * T + t];
                        const float4 v = d;
                        d = make_float4(__builtin_fmaf(g[4 * part], xh[4 * part], v.x), __builtin_fmaf(g[4 * part + 1], xh[4 * part + 1], v.y),
                                        __builtin_fmaf(g[4 * part + 2], xh[4 * part + 2], v.z), __builtin_fmaf(g[4 * part + 3], xh[4 * part + 3], v.w));
                    }
        }
        if (!a.dx) continue;
        if constexpr (DS && IN_LDS) {  // (no registers for it before)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < VPT; p++) qd[p] = row < rows ? lane.template load<DT>(a.ds + row * a.ld_ds * SIZE, p, cols) : make_uint4(0u, 0u, 0u, 0u);
        }
        s2 = rms_row_sum<T>(s2, slots[parity]) * inv_cols;
        if (row >= rows) continue;
#pragma unroll
        for (int p = 0; p < VPT; p++) {
            if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);
            set_apart<DT>(qs[p]);
            set_apart<DT>(qg[p]);
            ln_unpack<DT>(qs[p], xh);
            ln_unpack<DT>(qg[p], g);
            if constexpr (SHARED) ws.read(p * T + t, w);
            float d[V];
            if constexpr (DS) ln_unpack<DT>(qd[p], d);
#pragma unroll
            for (int i = 0; i < V; i++) {
#pragma clang fp contract(off)  // what two lanes store has the same bits
                g[i] = __builtin_fmaf(rstd, __builtin_fmaf(xh[i] * rstd, -s2, g[i] * w[i]), DS ? d[i] : 0.f);
            }
            lane.template store<DT>(a.dx + row * cols * SIZE, p, cols, g);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (int64_t)blockIdx.x * cols;  // a row of sums a workgroup
#pragma unroll
    for (int p = 0; p < VPT; p++) {
        if constexpr (GROUPS > 1) {
            __syncthreads();
            if (group > 0)
#pragma unroll
                for (int i = 0; i < V; i++) sums[((group - 1) * V + i) * T + t] = dw[p][i];
            __syncthreads();
            if (group > 0) continue;
#pragma unroll 1
            for (int k = 0; k < GROUPS - 1; k++)
#pragma unroll
                for (int i = 0; i < V; i++) dw[p][i] += sums[(k * V + i) * T + t];
        }
        const int col = lane.col(p);
        if constexpr (IN_LDS) {
            if (p * T + t >= ws.pieces) continue;
#pragma unroll
            for (int part = 0; part < V / 4; part++) {
                const float4 d = lds_sums[part * ws.pieces + p * T + t];
                const float v[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (lane.has(p, part * 4 + e)) out[col + part * 4 + e] = v[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane.has(p, i)) out[col + i] = dw[p][i];
        }
    }
}

// ---- rows that do not fit in registers: a workgroup a row, read again for the result (out of the L2), and the column sums by themselves
constexpr int RMS_WIDE_THREADS = 1024;

template <int DT, int PT, bool CAST>
__global__ __launch_bounds__(RMS_WIDE_THREADS) void rms_norm_wide_kernel(const RmsArgs a) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    constexpr int64_t STEP = RMS_WIDE_THREADS * V;
    __shared__ float slots[RMS_WIDE_THREADS / 64];
    const int64_t row = blockIdx.x, cols = a.cols;
    const uint8_t* in = a.x + row * a.ld * SIZE;
    float v[V], s = 0.f;
    auto load = [&](int64_t col) __attribute__((always_inline)) {
        ln_unpack<DT>(ln_load<DT, int64_t>(in, col, cols), v);
        if (a.residual) {
            float r[V];
            ln_unpack<DT>(ln_load<DT, int64_t>(a.residual + row * a.ld_res * SIZE, col, cols), r);
#pragma unroll
            for (int i = 0; i < V; i++) v[i] += r[i];
            ln_unpack<DT>(ln_pack<DT>(v), v);
        }
    };
    for (int64_t col = threadIdx.x * V; col < cols; col += STEP) {
        load(col);
        if (a.residual) ln_store<DT, int64_t>(a.sum + row * cols * SIZE, col, cols, v);
#pragma unroll
        for (int i = 0; i < V; i++) s = __builtin_fmaf(v[i], v[i], s);
    }
    s = rms_row_sum<RMS_WIDE_THREADS>(s, slots);
    const float rstd = 1.0f / __builtin_sqrtf(s / (float)cols + a.eps);
    const int64_t end = CAST ? (cols + 127) & ~(int64_t)127 : cols;
    for (int64_t col = threadIdx.x * V; col < end; col += STEP) {  // (CAST: the lanes of a block leave together)
        float w[V];
        load(col);
        ln_param<PT, V, int64_t>(a.weight, col, cols, 1.f, w);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = v[i] * rstd * w[i];
        if constexpr (CAST) {
            uint32_t c[V / 4], exponent;
            rms_cast<V>(v, c, exponent);
            uint8_t* at = a.y + ((col >> 6) * a.rows + row) * 64 + (col & 63);
            if constexpr (V == 8) *(uint2*)at = make_uint2(c[0], c[1]);
            else *(uint32_t*)at = c[0];
            if ((col & 127) == 0) a.scales[(col >> 7) * a.padded_rows + (row & ~(int64_t)127) + block_scale_at((int)(row & 127))] = (uint8_t)exponent;
        } else {
            ln_store<DT, int64_t>(a.y + row * cols * SIZE, col, cols, v);
        }
    }
    if (!CAST && a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
}

// SUMS: the sums of the columns too, in LDS; a workgroup takes every (number of workgroups)-th row.  Else a workgroup a row, and a kernel of their own.
template <int DT, int PT, bool SUMS>
__global__ __launch_bounds__(RMS_WIDE_THREADS) void rms_norm_backward_wide_kernel(const RmsBackwardArgs a) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    constexpr int64_t STEP = RMS_WIDE_THREADS * V;
    __shared__ float slots[2][RMS_WIDE_THREADS / 64];
    extern __shared__ uint4 rms_shared[];  // SUMS: of V columns, the four from part * 4 on, at [part][piece]
    const int64_t cols = a.cols, pieces = (cols + V - 1) / V;
    float4* sums = (float4*)rms_shared;
    if constexpr (SUMS)
        for (int64_t i = threadIdx.x; i < pieces; i += RMS_WIDE_THREADS)
#pragma unroll
            for (int part = 0; part < V / 4; part++) sums[part * pieces + i] = make_float4(0.f, 0.f, 0.f, 0.f);  // (a lane's own)
    int parity = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        const uint8_t *srow = a.s + row * a.ld * SIZE, *grow = a.dy + row * a.ld_dy * SIZE;
        const float rstd = a.rstd[row];
        float s2 = 0.f;
#pragma unroll 2
        for (int64_t col = threadIdx.x * V; col < cols; col += STEP) {
            float s[V], g[V], w[V];
            ln_unpack<DT>(ln_load<DT, int64_t>(srow, col, cols), s);
            ln_unpack<DT>(ln_load<DT, int64_t>(grow, col, cols), g);
            ln_param<PT, V, int64_t>(a.weight, col, cols, 1.f, w);
#pragma unroll
            for (int i = 0; i < V; i++) {
                s[i] *= rstd;
                if (col + i >= cols) s[i] = 0.f;  // (there g is zero, but rstd may be infinite)
                s2 = __builtin_fmaf(g[i] * w[i], s[i], s2);
            }
            if constexpr (SUMS)
#pragma unroll
                for (int part = 0; part < V / 4; part++) {
                    float4& d = sums[part * pieces + col / V];
                    d = make_float4(__builtin_fmaf(g[4 * part], s[4 * part], d.x), __builtin_fmaf(g[4 * part + 1], s[4 * part + 1], d.y), __builtin_fmaf(g[4 * part + 2], s[4 * part + 2], d.z),
                                    __builtin_fmaf(g[4 * part + 3], s[4 * part + 3], d.w));
                }
        }
        if (!a.dx) continue;
        s2 = rms_row_sum<RMS_WIDE_THREADS>(s2, slots[parity]) / (float)cols;
#pragma unroll 2
        for (int64_t col = threadIdx.x * V; col < cols; col += STEP) {
            float s[V], g[V], w[V], d[V] = {};
            ln_unpack<DT>(ln_load<DT, int64_t>(srow, col, cols), s);
            ln_unpack<DT>(ln_load<DT, int64_t>(grow, col, cols), g);
            ln_param<PT, V, int64_t>(a.weight, col, cols, 1.f, w);
            if (a.ds) ln_unpack<DT>(ln_load<DT, int64_t>(a.ds + row * a.ld_ds * SIZE, col, cols), d);
#pragma unroll
            for (int i = 0; i < V; i++) g[i] = __builtin_fmaf(rstd, __builtin_fmaf(s[i] * rstd, -s2, g[i] * w[i]), d[i]);
            ln_store<DT, int64_t>(a.dx + row * cols * SIZE, col, cols, g);
        }
    }
    if constexpr (SUMS) {
        float* out = a.partial + (int64_t)blockIdx.x * cols;
        for (int64_t i = threadIdx.x; i < pieces; i += RMS_WIDE_THREADS)
#pragma unroll
            for (int part = 0; part < V / 4; part++) {
                const float4 d = sums[part * pieces + i];
                const float v[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i * V + part * 4 + e < cols) out[i * V + part * 4 + e] = v[e];
            }
    }
}

// column sums of dy * xhat: 256 lanes' columns of `chunk` rows a workgroup
template <int DT>
__global__ __launch_bounds__(256) void rms_norm_columns_kernel(const RmsBackwardArgs a, int64_t chunk) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    const int64_t col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, cols = a.cols;
    if (col >= cols) return;
    float dw[V] = {}, s[V], g[V];
    const int64_t end = std::min<int64_t>(a.rows, (blockIdx.y + 1) * chunk);
#pragma unroll 4
    for (int64_t r = blockIdx.y * chunk; r < end; r++) {
        const float rstd = a.rstd[r];
        ln_unpack<DT>(ln_load<DT, int64_t>(a.s + r * a.ld * SIZE, col, cols), s);
        ln_unpack<DT>(ln_load<DT, int64_t>(a.dy + r * a.ld_dy * SIZE, col, cols), g);
#pragma unroll
        for (int i = 0; i < V; i++) dw[i] = __builtin_fmaf(g[i], s[i] * rstd, dw[i]);
    }
    float* out = a.partial + (int64_t)blockIdx.y * cols;
#pragma unroll
    for (int i = 0; i < V; i++)
        if (col + i < cols) out[col + i] = dw[i];
}

// Adds the `parts` rows of sums: 64 columns a workgroup, a wave every 16th row of them
constexpr int RMS_FINISH_WAVES = 16;
__global__ __launch_bounds__(64 * RMS_FINISH_WAVES) void rms_norm_finish_kernel(const float* __restrict__ partial, int64_t parts, int64_t cols, void* __restrict__ dw, int p_dtype) {
    __shared__ float red[RMS_FINISH_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (col < cols) {
#pragma unroll 8
        for (int64_t i = wave; i < parts; i += RMS_FINISH_WAVES) s += partial[i * cols + col];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= cols) return;
    s = red[0][lane];
#pragma unroll
    for (int i = 1; i < RMS_FINISH_WAVES; i++) s += red[i][lane];
    if (p_dtype == F8MI_FP32) ((float*)dw)[col] = s;
    else if (p_dtype == F8MI_BF16) ((uint16_t*)dw)[col] = (uint16_t)pack2<F8MI_BF16>(s, 0.f);
    else ((uint16_t*)dw)[col] = (uint16_t)pack2<F8MI_FP16>(s, 0.f);
}

// ---- launches

// Lanes of a row and pieces a lane, by the number of 16-byte pieces of a row; 0: does not fit.  The weight has to fit in LDS, and a lane's pieces in 128 registers: with
// the conversion to block scales three of them, in backward three of 16-bit values.
struct RmsShape {
    int t, vpt;
};
constexpr int RMS_MAX_LDS = (160 << 10) - 512;
static int64_t rms_pieces(int64_t cols, int dtype) { return (cols + (dtype == F8MI_FP32 ? 3 : 7)) / (dtype == F8MI_FP32 ? 4 : 8); }
static int64_t rms_lds(int64_t cols, int dtype, int p_dtype) { return rms_pieces(cols, dtype) * 16 * (dtype == p_dtype ? 1 : 2); }
constexpr int rms_forward_pieces(int dtype, bool cast) { return cast ? 3 : dtype == F8MI_FP32 ? 5 : 4; }
constexpr int rms_backward_pieces(int dtype) { return dtype == F8MI_FP32 ? 5 : 3; }
static int64_t rms_sums_lds(int64_t cols, int dtype) { return rms_pieces(cols, dtype) * (dtype == F8MI_FP32 ? 16 : 32); }  // of the columns' sums
static RmsShape rms_shape(int64_t cols, int dtype, int p_dtype, int most, bool sums) {
    const int64_t pieces = rms_pieces(cols, dtype);
    for (int t = 64; t <= 512; t *= 2)
        if (pieces <= t) return {t, 1};
    // two workgroups a CU instead of one whose lanes are half idle (both passes, us, 1024 lanes / 512: 8192 rows of 4352 bf16 107 / 102, of 5120 118 / 113, 4096 of 6000 78 / 76, of 7000
    // 87 / 88, of 8192 94 / 96; 4099 of 2050 fp32 45 / 42, of 3000 53 / 52, of 4096 62 / 65)
    if (pieces <= 768) return {512, 2};
    if (pieces <= RMS_LANES) return {RMS_LANES, 1};
    const int64_t vpt = (pieces + RMS_LANES - 1) / RMS_LANES;
    if (vpt > most || rms_lds(cols, dtype, p_dtype) + (sums && rms_sums_in_lds(dtype, (int)vpt) ? rms_sums_lds(cols, dtype) : 0) > RMS_MAX_LDS) return {0, 0};
    return {RMS_LANES, (int)vpt};
}
// Workgroups of `threads` lanes, `per_cu` of them on every CU, no more than the rows need
static int64_t rms_workgroups(RmsShape s, int64_t rows, int threads, int per_cu) {
    const int64_t groups = threads / s.t;
    return std::min<int64_t>((int64_t)cu_count() * per_cu, (rows + groups - 1) / groups);
}
static int64_t rms_chunk_rows(int64_t rows, int64_t cols, int dtype) {  // of the column kernel for wide rows: 1024 workgroups or so
    const int64_t strip = dtype == F8MI_FP32 ? 1024 : 2048, strips = (cols + strip - 1) / strip, want = std::max<int64_t>(1, 1024 / strips);
    return std::max<int64_t>(8, (rows + want - 1) / want);
}
static int64_t rms_parts(int64_t rows, int64_t cols, int dtype, int p_dtype) {
    const RmsShape s = rms_shape(cols, dtype, p_dtype, rms_backward_pieces(dtype), true);
    if (s.t) return rms_workgroups(s, rows, rms_backward_threads(s.t, s.vpt), RMS_LANES / rms_backward_threads(s.t, s.vpt));
    if (rms_sums_lds(cols, dtype) <= RMS_MAX_LDS) return std::min<int64_t>(cu_count(), rows);
    const int64_t chunk = rms_chunk_rows(rows, cols, dtype);
    return (rows + chunk - 1) / chunk;
}

template <int DT, int PT, int T, int VPT, bool RES, bool CAST>
static int launch_rms(const RmsArgs& a) {
    const auto kernel = rms_norm_kernel<DT, PT, T, VPT, RES, CAST>;
    if constexpr (VPT > 1) {
        static std::atomic<uint64_t> allowed{0};
        if (int rc = allow_big_lds(kernel, RMS_MAX_LDS, allowed)) return rc;
    }
    const int per_cu = rms_waves_a_simd(T, VPT) * 256 / rms_threads(T);
    hipLaunchKernelGGL(kernel, dim3((unsigned)rms_workgroups({T, VPT}, a.rows, rms_threads(T), per_cu)), dim3(rms_threads(T)), (unsigned)(VPT > 1 ? rms_lds(a.cols, DT, PT) : 0), a.stream, a);
    return check_hip(hipGetLastError(), "RMS norm kernel launch");
}
template <int DT, int PT, bool CAST>
static int launch_rms_wide(const RmsArgs& a) {
    hipLaunchKernelGGL((rms_norm_wide_kernel<DT, PT, CAST>), dim3((unsigned)a.rows), dim3(RMS_WIDE_THREADS), 0, a.stream, a);
    return check_hip(hipGetLastError(), "RMS norm kernel launch");
}
template <int DT, int PT, bool RES, bool CAST>
static int launch_rms_by_size(const RmsArgs& a) {
    const RmsShape s = rms_shape(CAST ? (a.cols + 127) & ~(int64_t)127 : a.cols, DT, PT, rms_forward_pieces(DT, CAST), false);
    if (s.t == 64) return launch_rms<DT, PT, 64, 1, RES, CAST>(a);
    if (s.t == 128) return launch_rms<DT, PT, 128, 1, RES, CAST>(a);
    if (s.t == 256) return launch_rms<DT, PT, 256, 1, RES, CAST>(a);
    if (s.t == 512 && s.vpt == 1) return launch_rms<DT, PT, 512, 1, RES, CAST>(a);
    if (s.t == 512) return launch_rms<DT, PT, 512, 2, RES, CAST>(a);
    if (s.vpt == 1) return launch_rms<DT, PT, RMS_LANES, 1, RES, CAST>(a);
    if (s.vpt == 2) return launch_rms<DT, PT, RMS_LANES, 2, RES, CAST>(a);
    if (s.vpt == 3) return launch_rms<DT, PT, RMS_LANES, 3, RES, CAST>(a);
    if constexpr (rms_forward_pieces(DT, CAST) >= 4)
        if (s.vpt == 4) return launch_rms<DT, PT, RMS_LANES, 4, RES, CAST>(a);
    if constexpr (rms_forward_pieces(DT, CAST) == 5)
        if (s.vpt == 5) return launch_rms<DT, PT, RMS_LANES, 5, RES, CAST>(a);
    return launch_rms_wide<DT, PT, CAST>(a);
}
template <bool CAST>
static int launch_rms_by_type(int dtype, int p_dtype, const RmsArgs& a) {
    auto with = [&](auto dt, auto pt) {
        constexpr int DT = decltype(dt)::value, PT = decltype(pt)::value;
        return a.residual ? launch_rms_by_size<DT, PT, true, CAST>(a) : launch_rms_by_size<DT, PT, false, CAST>(a);
    };
    using BF16 = std::integral_constant<int, F8MI_BF16>;
    using FP16 = std::integral_constant<int, F8MI_FP16>;
    using FP32 = std::integral_constant<int, F8MI_FP32>;
    if (dtype == F8MI_BF16) return p_dtype == F8MI_FP32 ? with(BF16{}, FP32{}) : with(BF16{}, BF16{});
    if (dtype == F8MI_FP16) return p_dtype == F8MI_FP32 ? with(FP16{}, FP32{}) : with(FP16{}, FP16{});
    return with(FP32{}, FP32{});
}

template <int DT, int PT, int T, int VPT, bool DS>
static int launch_rms_backward(const RmsBackwardArgs& a) {
    const auto kernel = rms_norm_backward_kernel<DT, PT, T, VPT, DS>;
    if constexpr (VPT > 1) {
        static std::atomic<uint64_t> allowed{0};
        if (int rc = allow_big_lds(kernel, RMS_MAX_LDS, allowed)) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)a.parts), dim3(rms_backward_threads(T, VPT)),
                       (unsigned)((VPT > 1 ? rms_lds(a.cols, DT, PT) : 0) + (rms_sums_in_lds(DT, VPT) ? rms_sums_lds(a.cols, DT) : 0)), a.stream, a);
    return check_hip(hipGetLastError(), "RMS norm backward kernel launch");
}
template <int DT, int PT>
static int launch_rms_backward_wide(const RmsBackwardArgs& a) {
    if (a.partial && rms_sums_lds(a.cols, DT) <= RMS_MAX_LDS) {
        const auto kernel = rms_norm_backward_wide_kernel<DT, PT, true>;
        static std::atomic<uint64_t> allowed{0};
        if (int rc = allow_big_lds(kernel, RMS_MAX_LDS, allowed)) return rc;
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.parts), dim3(RMS_WIDE_THREADS), (unsigned)rms_sums_lds(a.cols, DT), a.stream, a);
        return check_hip(hipGetLastError(), "RMS norm backward kernel launch");
    }
    if (a.dx) hipLaunchKernelGGL((rms_norm_backward_wide_kernel<DT, PT, false>), dim3((unsigned)a.rows), dim3(RMS_WIDE_THREADS), 0, a.stream, a);
    if (a.partial) {
        const unsigned strips = (unsigned)((a.cols + 256 * Ln<DT>::V - 1) / (256 * Ln<DT>::V));
        hipLaunchKernelGGL(rms_norm_columns_kernel<DT>, dim3(strips, (unsigned)a.parts), dim3(256), 0, a.stream, a, rms_chunk_rows(a.rows, a.cols, DT));
    }
    return check_hip(hipGetLastError(), "RMS norm backward kernel launch");
}
template <int DT, int PT, bool DS>
static int launch_rms_backward_by_size(const RmsBackwardArgs& a) {
    const RmsShape s = rms_shape(a.cols, DT, PT, rms_backward_pieces(DT), true);
    if (s.t == 64) return launch_rms_backward<DT, PT, 64, 1, DS>(a);
    if (s.t == 128) return launch_rms_backward<DT, PT, 128, 1, DS>(a);
    if (s.t == 256) return launch_rms_backward<DT, PT, 256, 1, DS>(a);
    if (s.t == 512 && s.vpt == 1) return launch_rms_backward<DT, PT, 512, 1, DS>(a);
    if (s.t == 512) return launch_rms_backward<DT, PT, 512, 2, DS>(a);
    if (s.vpt == 1) return launch_rms_backward<DT, PT, RMS_LANES, 1, DS>(a);
    if (s.vpt == 2) return launch_rms_backward<DT, PT, RMS_LANES, 2, DS>(a);
    if (s.vpt == 3) return launch_rms_backward<DT, PT, RMS_LANES, 3, DS>(a);
    if constexpr (rms_backward_pieces(DT) == 5) {
        if (s.vpt == 4) return launch_rms_backward<DT, PT, RMS_LANES, 4, DS>(a);
        if (s.vpt == 5) return launch_rms_backward<DT, PT, RMS_LANES, 5, DS>(a);
    }
    return launch_rms_backward_wide<DT, PT>(a);
}
static int launch_rms_backward_by_type(int dtype, int p_dtype, const RmsBackwardArgs& a) {
    auto with = [&](auto dt, auto pt) {
        constexpr int DT = decltype(dt)::value, PT = decltype(pt)::value;
        return a.ds ? launch_rms_backward_by_size<DT, PT, true>(a) : launch_rms_backward_by_size<DT, PT, false>(a);
    };
    using BF16 = std::integral_constant<int, F8MI_BF16>;
    using FP16 = std::integral_constant<int, F8MI_FP16>;
    using FP32 = std::integral_constant<int, F8MI_FP32>;
    if (dtype == F8MI_BF16) return p_dtype == F8MI_FP32 ? with(BF16{}, FP32{}) : with(BF16{}, BF16{});
    if (dtype == F8MI_FP16) return p_dtype == F8MI_FP32 ? with(FP16{}, FP32{}) : with(FP16{}, FP16{});
    return with(FP32{}, FP32{});
}

static int rms_check(const char* what, int64_t rows, int64_t cols, int dtype, int p_dtype) {
    if (dtype < 0 || dtype > 2 || (p_dtype != dtype && p_dtype != F8MI_FP32)) { set_error("%s: the weight has x's type or is fp32 (dtype codes %d, %d)", what, dtype, p_dtype); return F8MI_ERR_INVALID_ARG; }
    if (rows < 0 || cols <= 0) { set_error("%s: bad shape rows=%lld cols=%lld", what, (long long)rows, (long long)cols); return F8MI_ERR_INVALID_ARG; }
    if (rows > 0x7fffffff || cols > 0x7fffff00) { set_error("%s: dimension too large", what); return F8MI_ERR_UNSUPPORTED; }
    return F8MI_OK;
}
static bool bad_ld(int64_t ld, int64_t cols) { return ld < 0 || (ld < cols && ld != 0); }

}  // namespace f8mi

using namespace f8mi;

extern "C" int f8mi_rms_norm(const void* x, int64_t ld, const void* residual, int64_t ld_residual, int64_t rows, int64_t cols, int dtype, const void* weight, int p_dtype, float eps,
                             void* y, void* sum, float* rstd, void* stream) {
    if (int rc = rms_check("f8mi_rms_norm", rows, cols, dtype, p_dtype)) return rc;
    if (rows == 0) return F8MI_OK;
    if (!x || !y || bad_ld(ld, cols) || (residual && (!sum || bad_ld(ld_residual, cols)))) { set_error("f8mi_rms_norm: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    return launch_rms_by_type<false>(dtype, p_dtype, {(const uint8_t*)x, (const uint8_t*)residual, ld, ld_residual, rows, cols, weight, eps, (uint8_t*)y, (uint8_t*)sum, rstd, nullptr, 0, (hipStream_t)stream});
}

extern "C" int f8mi_rms_norm_block(const void* x, int64_t ld, const void* residual, int64_t ld_residual, int64_t rows, int64_t cols, int dtype, const void* weight, int p_dtype, float eps,
                                   void* out, void* out_scales, void* sum, void* stream) {
    if (int rc = rms_check("f8mi_rms_norm_block", rows, cols, dtype, p_dtype)) return rc;
    if (rows == 0) return F8MI_OK;
    if (!x || !out || !out_scales || bad_ld(ld, cols) || (residual && (!sum || bad_ld(ld_residual, cols)))) { set_error("f8mi_rms_norm_block: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    if ((uintptr_t)out % 16 != 0 || (uintptr_t)out_scales % 16 != 0) { set_error("f8mi_rms_norm_block: the copy and its scales are 16-byte aligned"); return F8MI_ERR_INVALID_ARG; }
    return launch_rms_by_type<true>(dtype, p_dtype, {(const uint8_t*)x, (const uint8_t*)residual, ld, ld_residual, rows, cols, weight, eps, (uint8_t*)out, (uint8_t*)sum, nullptr,
                                                     (uint8_t*)out_scales, block_rows_padded(rows), (hipStream_t)stream});
}

extern "C" int64_t f8mi_rms_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype, int p_dtype) {
    return rows <= 0 || cols <= 0 || dtype < 0 || dtype > 2 || (p_dtype != dtype && p_dtype != F8MI_FP32) ? 0 : rms_parts(rows, cols, dtype, p_dtype) * cols * 4;
}

extern "C" int f8mi_rms_norm_backward(const void* dy, int64_t ld_dy, const void* s, int64_t ld, const void* ds, int64_t ld_ds, int64_t rows, int64_t cols, int dtype, const void* weight,
                                      int p_dtype, const float* rstd, void* dx, void* dweight, void* workspace, int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = rms_check("f8mi_rms_norm_backward", rows, cols, dtype, p_dtype)) return rc;
    if (!dx && !dweight) return F8MI_OK;
    if (rows > 0 && (!dy || !s || !rstd || bad_ld(ld, cols) || bad_ld(ld_dy, cols) || (ds && bad_ld(ld_ds, cols)))) { set_error("f8mi_rms_norm_backward: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    const int64_t need = dweight ? f8mi_rms_norm_workspace_bytes(rows, cols, dtype, p_dtype) : 0;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)) { set_error("f8mi_rms_norm_backward: workspace of %lld bytes needed", (long long)need); return F8MI_ERR_INVALID_ARG; }
    const int64_t parts = rows > 0 ? rms_parts(rows, cols, dtype, p_dtype) : 0;
    if (rows > 0)
        if (int rc = launch_rms_backward_by_type(dtype, p_dtype, {(const uint8_t*)dy, (const uint8_t*)s, (const uint8_t*)ds, ld_dy, ld, ld_ds, rows, cols, weight, rstd, (uint8_t*)dx,
                                                                   dweight ? (float*)workspace : nullptr, parts, stream})) return rc;
    if (dweight)
        hipLaunchKernelGGL(rms_norm_finish_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(64 * RMS_FINISH_WAVES), 0, stream, (const float*)workspace, parts, cols, dweight, p_dtype);
    return check_hip(hipGetLastError(), "RMS norm column sum kernel launch");
}
