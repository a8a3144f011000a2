// Low-rank adapters of many requests beside one projection (f8mi_adapters.h), forward and backward:
//   h_i = A_e x_i,  out_i = y_i + scale_e B_e h_i,
//   dh_i = B_e^T dout_i,  dx_i = scale_e A_e^T dh_i,  dA_e = scale_e sum_i dh_i x_i^T,  dB_e = scale_e sum_i dout_i h_i^T.
// Three kernels: `shrink` (h from x and A, dh from dout and B^T), `expand` (out from y, h and B; dx from dh and A^T) and `outer` (dA, dB).  The
// transposed copies of the adapters that backward needs are made by a fourth; they are small beside x.
//
// HBM-bound: x, y and dout are read once each, out and dx written, an adapter is read by each of its tiles out of the L2.  The products run
// on the matrix cores straight from registers: a lane's 16 bytes of a row, loaded as they lie, are its operand.  The order of a contraction is free as long
// as both operands have the same one, so a lane takes 32 neighbouring bytes of a row and four lanes whole lines of the cache.
//
// h and dh are sums and stay in 32 bits: 16-bit matrix instructions get them as the sum of two 16-bit values (an error of 2^-17 of h, where one alone
// would be off by as much as the rounding of the result), fp16 ones after a power of two for each row, so that nothing overflows or falls among the
// subnormals.
#include <algorithm>

#include "f8mi_adapters.h"

namespace f8mi {

typedef float v4f_l __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fp16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ v4f_l mfma_16(uint4 a, uint4 b, v4f_l acc) {
    if constexpr (DT == F8MI_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    else if constexpr (DT == F8MI_FP16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), acc, 0, 0, 0);
    else {
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
    }
}
__device__ __forceinline__ uint4 load16_any(const uint8_t* p) {
    const u32x4 v = *(const u32x4_any*)p;
    return make_uint4(v.x, v.y, v.z, v.w);
}

struct AdapterArgs {
    const uint8_t* x;  // [m][k], k: contracted (shrink)
    int64_t ld;
    const uint8_t* a;  // [count][r][k]
    const int32_t* table;
    float* partial;    // [splits][m][rp]: h in the table's order, parts of the contraction
    int64_t m;
    int k, r, rp, count, splits;
    // expand
    const uint8_t* b;  // [count][n][r]
    const float* scale;  // [count] or null: 1
    float factor;        // scale_e = factor * scale[e]
    const uint8_t* y;  // [m][n] or null
    int64_t ld_y;
    uint8_t* out;      // [m][n]
    float* h;          // [m][rp]: the parts added up, or null
    int n, cols;       // cols: of out that a workgroup has, a multiple of 256
};

// ---- shrink: a wave has 16 MT rows of one adapter, 16 RT of its rank and a part of the contraction
template <int DT, int MT, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void adapter_shrink_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2, STEP = 128 / SIZE;  // values of a step: a line of the cache of each row
    constexpr int DEPTH = MT * RT >= 8 ? 1 : 2;                       // steps in flight
    __shared__ float4 part[WAVES][MT * RT][64];
    const AdapterTile tile = tiles[blockIdx.x];
    if (tile.rows == 0 || tile.group >= g.count) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lm = lane & 15, lq = lane >> 4;
    const int j0 = blockIdx.z * (16 * RT);
    const int32_t* order = g.table + AdapterTable(g.m, g.count).order() + tile.first;
    const int64_t steps = g.k / STEP, unit = (int64_t)blockIdx.y * WAVES + wave, units = (int64_t)g.splits * WAVES;
    const int s0 = (int)(steps * unit / units), s1 = (int)(steps * (unit + 1) / units);
    const uint8_t *px[MT], *pa[RT];
#pragma unroll
    for (int i = 0; i < MT; i++) px[i] = g.x + (int64_t)order[min(i * 16 + lm, tile.rows - 1)] * g.ld * SIZE;
#pragma unroll
    for (int i = 0; i < RT; i++) pa[i] = g.a + ((int64_t)tile.group * g.r + min(j0 + i * 16 + lm, g.r - 1)) * g.k * SIZE;

    v4f_l acc[RT][MT];
#pragma unroll
    for (int i = 0; i < RT * MT; i++) acc[i / MT][i % MT] = (v4f_l){0.f, 0.f, 0.f, 0.f};
    uint4 fx[DEPTH][MT][2], fa[DEPTH][RT][2];
    auto load = [&](int d, int s) __attribute__((always_inline)) {
        const int64_t at = (int64_t)s * 128 + lq * 32;
#pragma unroll
        for (int i = 0; i < RT; i++) {
            fa[d][i][0] = load16_any(pa[i] + at);
            fa[d][i][1] = load16_any(pa[i] + at + 16);
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
            fx[d][i][0] = load16_any(px[i] + at);
            fx[d][i][1] = load16_any(px[i] + at + 16);
        }
    };
    auto multiply = [&](int d) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = mfma_16<DT>(fa[d][i][h], fx[d][j][h], acc[i][j]);
    };
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) load(d, min(s0 + d, s1 - 1));
        int s = s0;
        for (; s + DEPTH < s1; s += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                multiply(d);
                load(d, min(s + DEPTH + d, s1 - 1));
            }
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (s + d < s1) multiply(d);
    }
    if (unit == units - 1 && steps * STEP < g.k) {  // what is left of the rows
        const int at = (int)steps * STEP + lq * (STEP / 4);
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
            uint4 ta[RT], tx[MT];
#pragma unroll
            for (int i = 0; i < RT; i++) ta[i] = ln_load<DT, int>(pa[i], at + h * (STEP / 8), g.k);
#pragma unroll
            for (int i = 0; i < MT; i++) tx[i] = ln_load<DT, int>(px[i], at + h * (STEP / 8), g.k);
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = mfma_16<DT>(ta[i], tx[j], acc[i][j]);
        }
    }
    // lane l: row l % 16, 4 (l / 16) + e of the rank
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) part[wave][i * MT + j][lane] = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
    __syncthreads();
    for (int item = threadIdx.x; item < RT * MT * 64; item += 64 * WAVES) {
        const int at = item >> 6, l = item & 63, row = (at % MT) * 16 + (l & 15), j = j0 + (at / MT) * 16 + 4 * (l >> 4);
        float4 s = part[0][at][l];
#pragma unroll
        for (int w = 1; w < WAVES; w++) {
            const float4 p = part[w][at][l];
            s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
        }
        if (row < tile.rows && j < g.rp) *(float4*)(g.partial + ((int64_t)blockIdx.y * g.m + tile.first + row) * g.rp + j) = s;
    }
}

// ---- expand: a workgroup has 16 MT rows of one adapter and `cols` columns of out
constexpr int EXPAND_THREADS = 256;
template <int DT>
constexpr int expand_pitch(int rp) { return DT == F8MI_FP32 ? rp + 4 : (rp <= 16 ? 16 : (rp + 31) / 32 * 32) * 2 + 8; }  // elements of a row of h in LDS: high parts, then low ones

template <int DT, int MT>
__global__ __launch_bounds__(EXPAND_THREADS) void adapter_expand_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, ROWS = 16 * MT;
    extern __shared__ __align__(16) uint8_t expand_lds[];  // h [ROWS][pitch], then fp32 [ROWS][rp] while it is converted
    __shared__ float row_factor[ROWS];
    const AdapterTile tile = tiles[blockIdx.x];
    if (tile.rows == 0) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lm = lane & 15, lq = lane >> 4;
    const bool none = tile.group >= g.count;
    const int32_t* order = g.table + AdapterTable(g.m, g.count).order() + tile.first;
    const int rp = g.rp, pitch = expand_pitch<DT>(rp), half = (pitch - 8) / 2;  // half: of a row's high parts (16-bit types)
    float* sums = DT == F8MI_FP32 ? (float*)expand_lds : (float*)(expand_lds + ROWS * pitch * 2);
    const int sums_pitch = DT == F8MI_FP32 ? pitch : rp;
    if (!none) {
        const float scale = g.factor * (g.scale ? g.scale[tile.group] : 1.f);
        for (int item = t; item < ROWS * (rp / 4); item += EXPAND_THREADS) {
            const int row = item / (rp / 4), j = (item % (rp / 4)) * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < tile.rows) {
                const float* p = g.partial + ((int64_t)tile.first + row) * rp + j;
#pragma unroll 4
                for (int i = 0; i < g.splits; i++) {
                    const float4 q = *(const float4*)(p + i * g.m * rp);
                    s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
                }
                if (j >= g.r) s.x = 0.f;  // (rows of A past the last are the last again)
                if (j + 1 >= g.r) s.y = 0.f;
                if (j + 2 >= g.r) s.z = 0.f;
                if (j + 3 >= g.r) s.w = 0.f;
                if (g.h && blockIdx.y == 0) *(float4*)(g.h + ((int64_t)tile.first + row) * rp + j) = s;
            }
            *(float4*)(sums + row * sums_pitch + j) = make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale);
        }
        __syncthreads();
        if constexpr (DT != F8MI_FP32) {
            if constexpr (DT == F8MI_FP16) {  // a power of two that brings the row's largest to [1, 2)
                if (t < ROWS) {
                    uint32_t most = 0u;
                    for (int j = 0; j < g.r; j++) most = max(most, __float_as_uint(sums[t * rp + j]) & 0x7fffffffu);
                    const int e = min(max((int)(most >> 23), 1), 253);
                    row_factor[t] = __uint_as_float((uint32_t)e << 23);  // 2^(e - 127)
                }
                __syncthreads();
            }
            uint16_t* kept = (uint16_t*)expand_lds;
            for (int item = t; item < ROWS * half; item += EXPAND_THREADS) {
                const int row = item / half, j = item % half;
                float v = j < rp ? sums[row * rp + j] : 0.f;
                if constexpr (DT == F8MI_FP16) v *= __uint_as_float((254u << 23) - __float_as_uint(row_factor[row]));  // times 2^(127 - e)
                const uint32_t high = pack2<DT>(v, 0.f) & 0xffffu;
                float back, zero;
                unpack2<DT>(high, back, zero);
                kept[row * pitch + j] = (uint16_t)high;
                kept[row * pitch + half + j] = (uint16_t)pack2<DT>(back - back == 0.f ? v - back : 0.f, 0.f);  // (nothing is left of an infinity)
            }
            __syncthreads();
        }
    }
    const uint8_t* hrow[MT];  // of the lane's row in LDS
    float factor[MT];
    int64_t at_row[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        hrow[i] = expand_lds + (i * 16 + lm) * pitch * SIZE;
        factor[i] = DT == F8MI_FP16 && !none ? row_factor[i * 16 + lm] : 1.f;
        at_row[i] = order[min(i * 16 + lm, tile.rows - 1)];
    }
    const int end = min(g.n, (int)(blockIdx.y + 1) * g.cols);
    for (int n0 = blockIdx.y * g.cols + wave * 64; n0 < end; n0 += 256) {
        const int col = n0 + lq * 16;  // of out: 16 neighbouring ones of each of the lane's rows
        uint4 fy[MT][16 / V];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int p = 0; p < 16 / V; p++)
                fy[i][p] = g.y ? ln_load<DT, int>(g.y + at_row[i] * g.ld_y * SIZE, col + p * V, g.n) : make_uint4(0u, 0u, 0u, 0u);
        v4f_l acc[MT][4];
#pragma unroll
        for (int i = 0; i < MT * 4; i++) acc[i / 4][i % 4] = (v4f_l){0.f, 0.f, 0.f, 0.f};
        if (!none) {
            // tile c's row q of B: column n0 + 16 (q / 4) + 4 c + q % 4, so that a lane's four tiles give it neighbours
            const uint8_t* pb[4];
#pragma unroll
            for (int c = 0; c < 4; c++) pb[c] = g.b + ((int64_t)tile.group * g.n + min(n0 + 16 * (lm >> 2) + 4 * c + (lm & 3), g.n - 1)) * g.r * SIZE;
            if constexpr (DT == F8MI_FP32) {
                for (int j = 0; j < rp; j += 16) {
                    uint4 fb[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) fb[c] = ln_load<DT, int>(pb[c], j + lq * 4, g.r);
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        const uint4 fh = *(const uint4*)(hrow[i] + (j + lq * 4) * 4);
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[i][c] = mfma_16<DT>(fb[c], fh, acc[i][c]);
                    }
                }
            } else if (half == 16) {  // both parts of h in one instruction, B twice
                uint4 fb[4];
#pragma unroll
                for (int c = 0; c < 4; c++) fb[c] = ln_load<DT, int>(pb[c], (lq & 1) * 8, g.r);
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const uint4 fh = *(const uint4*)(hrow[i] + lq * 16);
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[i][c] = mfma_16<DT>(fb[c], fh, acc[i][c]);
                }
            } else {
                for (int j = 0; j < half; j += 32) {
                    uint4 fb[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) fb[c] = ln_load<DT, int>(pb[c], j + lq * 8, g.r);
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        const uint4 high = *(const uint4*)(hrow[i] + (j + lq * 8) * 2), low = *(const uint4*)(hrow[i] + (half + j + lq * 8) * 2);
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[i][c] = mfma_16<DT>(fb[c], low, mfma_16<DT>(fb[c], high, acc[i][c]));
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
            if (i * 16 + lm >= tile.rows) continue;
#pragma unroll
            for (int p = 0; p < 16 / V; p++) {
                if (col + p * V >= g.n) continue;
                float v[V];
                ln_unpack<DT>(fy[i][p], v);
                if (!none)  // (-0 + 0 is 0: a row without an adapter keeps its bits)
#pragma unroll
                    for (int e = 0; e < V; e++) v[e] = __builtin_fmaf(acc[i][(p * V + e) / 4][e % 4], factor[i], v[e]);
                ln_store<DT, int>(g.out + at_row[i] * g.n * SIZE, col + p * V, g.n, v);
            }
        }
    }
}

// ---- outer: of the rows of a chunk, small [row][j] times big [row][c]: 128 columns c and 64 of the rank j a workgroup
struct OuterArgs {
    const uint8_t* big;   // [m][cols], as the batch has its rows
    int64_t ld;
    const float* small;   // [m][rp], in the table's order
    const int32_t* table;
    int64_t m;
    int cols, r, rp, count, cols_first;  // cols_first: sums [cols][r], else [r][cols]
    float* partial;       // a matrix of sums for each chunk
};
constexpr int OUTER_COLS = 128, OUTER_ROWS = 16, OUTER_RANK = 64, OUTER_THREADS = 256;

template <int DT>
__global__ __launch_bounds__(OUTER_THREADS) void adapter_outer_kernel(const OuterArgs g, const AdapterTile* __restrict__ chunks) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    __shared__ __align__(16) float big[OUTER_ROWS][OUTER_COLS + 4];
    __shared__ __align__(16) float small[OUTER_ROWS][OUTER_RANK + 4];
    const AdapterTile chunk = chunks[blockIdx.x];
    if (chunk.rows == 0 || chunk.group >= g.count) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lm = lane & 15, lq = lane >> 4;
    const int c0 = blockIdx.y * OUTER_COLS, j0 = blockIdx.z * OUTER_RANK, rank_tiles = min((g.rp - j0) / 16, OUTER_RANK / 16);
    const int32_t* order = g.table + AdapterTable(g.m, g.count).order() + chunk.first;
    v4f_l acc[2][4];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i / 4][i % 4] = (v4f_l){0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < chunk.rows; r0 += OUTER_ROWS) {
        __syncthreads();
        for (int item = t; item < OUTER_ROWS * OUTER_COLS / V; item += OUTER_THREADS) {
            const int row = item / (OUTER_COLS / V), c = (item % (OUTER_COLS / V)) * V;
            float v[V] = {};
            if (r0 + row < chunk.rows) ln_unpack<DT>(ln_load<DT, int>(g.big + (int64_t)order[r0 + row] * g.ld * SIZE, c0 + c, g.cols), v);
#pragma unroll
            for (int e = 0; e < V; e += 4) *(float4*)&big[row][c + e] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
        for (int item = t; item < OUTER_ROWS * rank_tiles * 4; item += OUTER_THREADS) {
            const int row = item / (rank_tiles * 4), j = (item % (rank_tiles * 4)) * 4;
            *(float4*)&small[row][j] = r0 + row < chunk.rows ? *(const float4*)(g.small + ((int64_t)chunk.first + r0 + row) * g.rp + j0 + j) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < OUTER_ROWS; kk += 4) {
            float fb[2], fs[4];
#pragma unroll
            for (int c = 0; c < 2; c++) fb[c] = big[kk + lq][wave * 32 + c * 16 + lm];
#pragma unroll
            for (int j = 0; j < 4; j++) fs[j] = j < rank_tiles ? small[kk + lq][j * 16 + lm] : 0.f;
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (j < rank_tiles) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[c], fs[j], acc[c][j], 0, 0, 0);  // lane: j lm, c 4 lq + e
        }
    }
    float* out = g.partial + (int64_t)blockIdx.x * g.cols * g.r;
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int col = c0 + wave * 32 + c * 16 + 4 * lq + e, rank = j0 + j * 16 + lm;
                if (col < g.cols && rank < g.r) out[g.cols_first ? (int64_t)col * g.r + rank : (int64_t)rank * g.cols + col] = acc[c][j][e];
            }
}

// the chunks of an adapter added up in their order; no chunk: zeros
__global__ __launch_bounds__(256) void adapter_outer_finish_kernel(const float* __restrict__ partial, const int32_t* __restrict__ chunk_start, const float* __restrict__ scale, float factor, int64_t size,
                                                                   void* __restrict__ out, int dtype) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int e = blockIdx.y, first = chunk_start[e], end = chunk_start[e + 1];
    if (at >= size) return;
    float s = 0.f;
#pragma unroll 8
    for (int i = first; i < end; i++) s += partial[(int64_t)i * size + at];
    if (first < end) s *= factor * (scale ? scale[e] : 1.f);
    const int64_t to = (int64_t)e * size + at;
    if (dtype == F8MI_FP32) ((float*)out)[to] = s;
    else if (dtype == F8MI_BF16) ((uint16_t*)out)[to] = (uint16_t)pack2<F8MI_BF16>(s, 0.f);
    else ((uint16_t*)out)[to] = (uint16_t)pack2<F8MI_FP16>(s, 0.f);
}

// ---- [batch][rows][cols] -> [batch][cols][rows]
template <typename T>
__global__ __launch_bounds__(256) void adapter_transpose_kernel(const T* __restrict__ in, T* __restrict__ out, int rows, int cols, int tiles_c) {
    __shared__ T tile[32][33];
    const int64_t base = (int64_t)blockIdx.y * rows * cols;
    const int r0 = blockIdx.x / tiles_c * 32, c0 = blockIdx.x % tiles_c * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int i = ty; i < 32; i += 8)
        if (r0 + i < rows && c0 + tx < cols) tile[i][tx] = in[base + (int64_t)(r0 + i) * cols + c0 + tx];
    __syncthreads();
    for (int i = ty; i < 32; i += 8)
        if (c0 + i < cols && r0 + tx < rows) out[base + (int64_t)(c0 + i) * rows + r0 + tx] = tile[tx][i];
}
static int launch_transpose(const void* in, void* out, int64_t batch, int rows, int cols, int dtype, hipStream_t stream) {
    const int tiles_c = (cols + 31) / 32;
    const dim3 grid((unsigned)(((rows + 31) / 32) * tiles_c), (unsigned)batch);
    if (dtype == F8MI_FP32) hipLaunchKernelGGL(adapter_transpose_kernel<uint32_t>, grid, dim3(256), 0, stream, (const uint32_t*)in, (uint32_t*)out, rows, cols, tiles_c);
    else hipLaunchKernelGGL(adapter_transpose_kernel<uint16_t>, grid, dim3(256), 0, stream, (const uint16_t*)in, (uint16_t*)out, rows, cols, tiles_c);
    return check_hip(hipGetLastError(), "adapter transpose kernel launch");
}

// ---- launches
struct AdapterShape {
    int64_t m, k, n, r, count;
    int dtype;
    int64_t rp() const { return (r + 15) / 16 * 16; }
    AdapterTable table() const { return {m, count}; }
    // Tiles of 64 rows where an adapter has that many on average: x is read once for each 64 of the rank, an adapter once a tile.
    bool tall() const { return m >= 48 * (count < m ? count : m); }
    int64_t tiles() const { return table().tiles(tall() ? 64 : 16); }
    // Parts of a contraction of this length: two workgroups a CU, and two steps a wave
    int64_t splits(int64_t contracted) const {
        const int64_t steps = contracted * (dtype == F8MI_FP32 ? 4 : 2) / 128, waves = tall() ? 4 : 8, want = 2 * (int64_t)cu_count() / std::max<int64_t>(1, tiles() * ((rp() + 63) / 64));
        return std::max<int64_t>(1, std::min({want, steps / (2 * waves), (int64_t)32}));
    }
    int64_t partial_bytes(int64_t contracted) const { return splits(contracted) * m * rp() * 4; }
};
static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

template <int DT, int MT, int WAVES>
static int launch_shrink3(const AdapterArgs& g, const AdapterTile* tiles, int64_t n_tiles, hipStream_t stream) {
    const int rt = g.rp / 16;
    const dim3 grid((unsigned)n_tiles, (unsigned)g.splits, (unsigned)(rt <= 4 ? 1 : (rt + 3) / 4));
    if (rt == 1) hipLaunchKernelGGL((adapter_shrink_kernel<DT, MT, 1, WAVES>), grid, dim3(64 * WAVES), 0, stream, g, tiles);
    else if (rt == 2) hipLaunchKernelGGL((adapter_shrink_kernel<DT, MT, 2, WAVES>), grid, dim3(64 * WAVES), 0, stream, g, tiles);
    else hipLaunchKernelGGL((adapter_shrink_kernel<DT, MT, 4, WAVES>), grid, dim3(64 * WAVES), 0, stream, g, tiles);
    return check_hip(hipGetLastError(), "adapter shrink kernel launch");
}
template <int DT>
static int launch_shrink2(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    const AdapterTable table = s.table();
    if (s.tall()) return launch_shrink3<DT, 4, 4>(g, (const AdapterTile*)(g.table + table.tiles64()), s.tiles(), stream);
    return launch_shrink3<DT, 1, 8>(g, (const AdapterTile*)(g.table + table.tiles16()), s.tiles(), stream);
}
static int launch_shrink(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    if (s.dtype == F8MI_BF16) return launch_shrink2<F8MI_BF16>(g, s, stream);
    if (s.dtype == F8MI_FP16) return launch_shrink2<F8MI_FP16>(g, s, stream);
    return launch_shrink2<F8MI_FP32>(g, s, stream);
}

template <int DT, int MT>
static int launch_expand3(AdapterArgs g, const AdapterTile* tiles, int64_t n_tiles, hipStream_t stream) {
    // four workgroups a CU, each with as many columns as that leaves
    const int64_t want = std::max<int64_t>(1, 4 * (int64_t)cu_count() / n_tiles), blocks = std::max(1, (g.n + 255) / 256);  // (one, without columns, where h alone is asked for)
    g.cols = (int)((blocks + want - 1) / want * 256);
    const int lds = 16 * MT * (DT == F8MI_FP32 ? expand_pitch<DT>(g.rp) * 4 : expand_pitch<DT>(g.rp) * 2 + g.rp * 4);
    const auto kernel = adapter_expand_kernel<DT, MT>;
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_big_lds(kernel, (160 << 10) - 1024, allowed)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_tiles, (unsigned)((blocks * 256 + g.cols - 1) / g.cols)), dim3(EXPAND_THREADS), (unsigned)lds, stream, g, tiles);
    return check_hip(hipGetLastError(), "adapter expand kernel launch");
}
template <int DT>
static int launch_expand2(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    const AdapterTable table = s.table();
    if (s.tall()) return launch_expand3<DT, 4>(g, (const AdapterTile*)(g.table + table.tiles64()), s.tiles(), stream);
    return launch_expand3<DT, 1>(g, (const AdapterTile*)(g.table + table.tiles16()), s.tiles(), stream);
}
static int launch_expand(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    if (s.dtype == F8MI_BF16) return launch_expand2<F8MI_BF16>(g, s, stream);
    if (s.dtype == F8MI_FP16) return launch_expand2<F8MI_FP16>(g, s, stream);
    return launch_expand2<F8MI_FP32>(g, s, stream);
}
static int launch_outer(const OuterArgs& g, int dtype, const float* scale, float factor, void* out, int out_dtype, hipStream_t stream) {
    const AdapterTable table(g.m, g.count);
    const int64_t chunks = table.tiles(adapter_chunk_rows(g.m)), size = (int64_t)g.cols * g.r;
    const AdapterTile* list = (const AdapterTile*)(g.table + table.chunks());
    const dim3 grid((unsigned)chunks, (unsigned)((g.cols + OUTER_COLS - 1) / OUTER_COLS), (unsigned)((g.rp + OUTER_RANK - 1) / OUTER_RANK));
    if (dtype == F8MI_BF16) hipLaunchKernelGGL(adapter_outer_kernel<F8MI_BF16>, grid, dim3(OUTER_THREADS), 0, stream, g, list);
    else if (dtype == F8MI_FP16) hipLaunchKernelGGL(adapter_outer_kernel<F8MI_FP16>, grid, dim3(OUTER_THREADS), 0, stream, g, list);
    else hipLaunchKernelGGL(adapter_outer_kernel<F8MI_FP32>, grid, dim3(OUTER_THREADS), 0, stream, g, list);
    if (int rc = check_hip(hipGetLastError(), "adapter gradient kernel launch")) return rc;
    hipLaunchKernelGGL(adapter_outer_finish_kernel, dim3((unsigned)((size + 255) / 256), (unsigned)g.count), dim3(256), 0, stream, g.partial, g.table + table.chunk_start(), scale, factor, size, out, out_dtype);
    return check_hip(hipGetLastError(), "adapter gradient sum kernel launch");
}

static int adapters_check(const char* what, const AdapterShape& s) {
    if (s.dtype < 0 || s.dtype > 2) { set_error("%s: unknown dtype code %d", what, s.dtype); return F8MI_ERR_INVALID_ARG; }
    if (s.m < 0 || s.k < 1 || s.n < 1 || s.r < 1 || s.count < 1) { set_error("%s: bad shape m=%lld k=%lld n=%lld r=%lld count=%lld", what, (long long)s.m, (long long)s.k, (long long)s.n, (long long)s.r, (long long)s.count); return F8MI_ERR_INVALID_ARG; }
    if (s.m > F8MI_ADAPTER_MAX_ROWS || s.count > F8MI_ADAPTER_MAX_COUNT || s.r > F8MI_ADAPTER_MAX_RANK || s.k > (1 << 24) || s.n > (1 << 24)) {
        set_error("%s: at most %d rows, %d adapters of rank %d and 2^24 features", what, F8MI_ADAPTER_MAX_ROWS, F8MI_ADAPTER_MAX_COUNT, F8MI_ADAPTER_MAX_RANK);
        return F8MI_ERR_UNSUPPORTED;
    }
    return F8MI_OK;
}
static bool bad_stride(int64_t ld, int64_t cols) { return ld < 0 || (ld < cols && ld != 0); }

// parts of backward's workspace
struct AdapterBackwardSpace {
    int64_t partial, dh, at, bt, sums, bytes;
    AdapterBackwardSpace(const AdapterShape& s, bool need_dx, bool need_da, bool need_db) {
        const int64_t size = s.dtype == F8MI_FP32 ? 4 : 2, chunks = s.table().tiles(adapter_chunk_rows(s.m));
        const bool inner = need_dx || need_da;
        int64_t at_byte = 0;
        auto take = [&](int64_t n) { const int64_t o = at_byte; at_byte += up256(n); return o; };
        partial = take(inner ? s.partial_bytes(s.n) : 0);
        dh = take(inner ? s.m * s.rp() * 4 : 0);
        bt = take(inner ? s.count * s.n * s.r * size : 0);
        at = take(need_dx ? s.count * s.k * s.r * size : 0);
        sums = take(std::max(need_da ? chunks * s.k * s.r * 4 : 0, need_db ? chunks * s.n * s.r * 4 : 0));
        bytes = at_byte;
    }
};

}  // namespace f8mi

using namespace f8mi;

extern "C" int64_t f8mi_adapters_workspace_bytes(int64_t m, int64_t k, int64_t n, int64_t r, int64_t count, int dtype) {
    const AdapterShape s{m, k, n, r, count, dtype};
    return adapters_check("f8mi_adapters_workspace_bytes", s) || m == 0 ? 0 : s.partial_bytes(k);
}
extern "C" int64_t f8mi_adapters_backward_workspace_bytes(int64_t m, int64_t k, int64_t n, int64_t r, int64_t count, int dtype, int need_dx, int need_da, int need_db) {
    const AdapterShape s{m, k, n, r, count, dtype};
    return adapters_check("f8mi_adapters_backward_workspace_bytes", s) || m == 0 ? 0 : AdapterBackwardSpace(s, need_dx, need_da, need_db).bytes;
}

extern "C" int f8mi_adapters(const void* x, int64_t ldx, const void* a, const void* b, const float* scale, float factor, const void* table, int64_t m, int64_t k, int64_t n, int64_t r, int64_t count,
                             int dtype, const void* y, int64_t ldy, void* out, float* h, void* workspace, int64_t workspace_bytes, void* stream_) {
    const AdapterShape s{m, k, n, r, count, dtype};
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = adapters_check("f8mi_adapters", s)) return rc;
    if (m == 0) return F8MI_OK;
    if (!x || !a || !b || !table || !out || bad_stride(ldx, k) || (y && bad_stride(ldy, n))) { set_error("f8mi_adapters: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    const int64_t need = s.partial_bytes(k);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0 || (uintptr_t)table % 16 != 0 || (uintptr_t)h % 16 != 0) { set_error("f8mi_adapters: 16-byte aligned workspace of %lld bytes, table and h", (long long)need); return F8MI_ERR_INVALID_ARG; }
    const AdapterArgs g{(const uint8_t*)x, ldx, (const uint8_t*)a, (const int32_t*)table, (float*)workspace, m, (int)k, (int)r, (int)s.rp(), (int)count, (int)s.splits(k),
                        (const uint8_t*)b, scale, factor, (const uint8_t*)y, ldy, (uint8_t*)out, h, (int)n, 0};
    if (int rc = launch_shrink(g, s, stream)) return rc;
    return launch_expand(g, s, stream);
}

extern "C" int f8mi_adapters_backward(const void* dout, int64_t ld_dout, const void* x, int64_t ldx, const void* a, const void* b, const float* scale, float factor, const void* table, const float* h, int64_t m,
                                      int64_t k, int64_t n, int64_t r, int64_t count, int dtype, void* dx, void* da, void* db, int p_dtype, void* workspace, int64_t workspace_bytes, void* stream_) {
    const AdapterShape s{m, k, n, r, count, dtype};
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = adapters_check("f8mi_adapters_backward", s)) return rc;
    if (m == 0 || (!dx && !da && !db)) return F8MI_OK;
    if (p_dtype < 0 || p_dtype > 2) { set_error("f8mi_adapters_backward: unknown dtype code %d", p_dtype); return F8MI_ERR_INVALID_ARG; }
    if (!dout || !table || bad_stride(ld_dout, n) || (da && (!x || bad_stride(ldx, k))) || (dx && !a) || ((dx || da) && !b) || (db && !h)) { set_error("f8mi_adapters_backward: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    const AdapterBackwardSpace space(s, dx, da, db);
    if (space.bytes && (!workspace || workspace_bytes < space.bytes || (uintptr_t)workspace % 256 != 0)) { set_error("f8mi_adapters_backward: 256-byte aligned workspace of %lld bytes needed", (long long)space.bytes); return F8MI_ERR_INVALID_ARG; }
    if ((uintptr_t)table % 16 != 0 || (uintptr_t)h % 16 != 0) { set_error("f8mi_adapters_backward: table and h are 16-byte aligned"); return F8MI_ERR_INVALID_ARG; }
    uint8_t* ws = (uint8_t*)workspace;
    float* dh = (float*)(ws + space.dh);
    if (dx || da) {
        if (int rc = launch_transpose(b, ws + space.bt, count, (int)n, (int)r, dtype, stream)) return rc;
        if (dx)
            if (int rc = launch_transpose(a, ws + space.at, count, (int)r, (int)k, dtype, stream)) return rc;
        const AdapterArgs g{(const uint8_t*)dout, ld_dout, ws + space.bt, (const int32_t*)table, (float*)(ws + space.partial), m, (int)n, (int)r, (int)s.rp(), (int)count, (int)s.splits(n),
                            dx ? ws + space.at : nullptr, scale, factor, nullptr, 0, (uint8_t*)dx, dh, dx ? (int)k : 0, 0};
        if (int rc = launch_shrink(g, s, stream)) return rc;
        if (int rc = launch_expand(g, s, stream)) return rc;
    }
    const OuterArgs o{nullptr, 0, nullptr, (const int32_t*)table, m, 0, (int)r, (int)s.rp(), (int)count, 0, (float*)(ws + space.sums)};
    if (da) {
        OuterArgs q = o;
        q.big = (const uint8_t*)x; q.ld = ldx; q.small = dh; q.cols = (int)k;
        if (int rc = launch_outer(q, dtype, scale, factor, da, p_dtype, stream)) return rc;
    }
    if (db) {
        OuterArgs q = o;
        q.big = (const uint8_t*)dout; q.ld = ld_dout; q.small = h; q.cols = (int)n; q.cols_first = 1;
        if (int rc = launch_outer(q, dtype, scale, factor, db, p_dtype, stream)) return rc;
    }
    return F8MI_OK;
}
