// Casts with block scales (f8mi_block.h): one pass over a tensor writes its e4m3 copy for the product that contracts the columns
// (blocks of 1 x 128), the transposed copy for the one that contracts the rows (blocks of 128 x 1), or both with one scale for each
// 128 x 128 (weights), each in the k-blocked placement [k/64][rows][64] with the contraction zero-padded to a multiple of 128.
//
// HBM-bound: 2 or 4 bytes read and one written per value and copy.  No amax pass in front, unlike a cast with one scale for the
// tensor: a workgroup of 256 lanes holds a tile of 128 x 128, which is whole blocks of every kind, in registers.  Lane t has
// columns 8 * (t % 16) .. + 7 of the rows 64 h + 4 * (t / 16) .. + 3.  The 16 lanes of a row find its maximum with four DPP steps (16-bit types: two
// rows in one register); the column maxima cross the waves through LDS.  The row copy leaves from registers as 8-byte stores; for the
// transposed one each lane turns its 4 x 8 blocks (v_perm), parks them in a swizzled LDS tile and the tile leaves as 16-byte stores that
// are contiguous over 4 KB.  A tile of 128 x 128 and not more: its 8 words a lane (fp32: 16) beside the converted ones let six workgroups be on a
// CU, and every kind of block is whole in it.
//
// Measured: 8192 x 28672 bf16 to both copies 161 us (5.8 TB/s; a copy: 4.9), with 8192 x 8192 to both and 28672 x 8192 to one 170 us (5.7), 2048 x 4096 12 us
// (launch and latency), 11007 x 4097 29 us.
#include "f8mi_block.h"
#include "f8mi_gemm_util.h"

namespace f8mi {

constexpr int BC_THREADS = 256;

struct BlockCastItem {
    const uint8_t* x;
    int64_t rows, cols, ld;  // ld in elements
    uint8_t *out, *out_scales, *out_t, *out_t_scales;
    float* sums;  // [rows / 128][cols]: the columns of each tile added up (the first half of a bias's gradient), or null
    int square;  // one scale for each 128 x 128
    int tiles_c;
};

template <int DT>
struct Eight {  // eight neighbouring elements
    uint32_t w[DT == F8MI_FP32 ? 8 : 4];
};

template <int DT>
__device__ __forceinline__ float value(const Eight<DT>& r, int i) {
    if constexpr (DT == F8MI_FP32) return __uint_as_float(r.w[i]);
    const uint32_t h = (i & 1) ? r.w[i >> 1] >> 16 : r.w[i >> 1] & 0xffffu;
    if constexpr (DT == F8MI_BF16) return bf16_bits_to_float(h);
    else return fp16_bits_to_float(h);
}

// Elements col .. + 7 of a row, zeros past `cols`.  Rows that start at multiples of 16 bytes are streamed.  Others (not ALIGNED) share a line of the
// cache wherever two tiles meet in a row: neighbouring tiles go to the same XCD and the lines are left in its L2 (11007 x 4097 bf16: 34.6 -> 29.0 us; the
// same tile with aligned rows: 27.2).
template <int DT, bool ALIGNED>
__device__ __forceinline__ Eight<DT> load_eight(const uint8_t* row, int64_t col, int64_t cols, bool in) {
    constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2, W = SIZE * 2;  // words of eight elements
    Eight<DT> r;
#pragma unroll
    for (uint32_t& w : r.w) w = 0u;
    if (in && col + 8 <= cols) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint8_t* p = row + col * SIZE + 4 * i;
            const u32x4 v = ALIGNED ? __builtin_nontemporal_load((const u32x4*)p) : *(const u32x4_any*)p;
            r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
        }
    } else if (in && col < cols) {
#pragma unroll 1
        for (int64_t c = cols - 1; c >= col; c--) {  // from the last one: each moves those behind it up by one place
#pragma unroll
            for (int i = W - 1; i > 0; i--) r.w[i] = DT == F8MI_FP32 ? r.w[i - 1] : r.w[i] << 16 | r.w[i - 1] >> 16;
            if constexpr (DT == F8MI_FP32) r.w[0] = ((const uint32_t*)row)[c];
            else r.w[0] = r.w[0] << 16 | ((const uint16_t*)row)[c];
        }
    }
    return r;
}
// What is unpacked after this is not kept from before.
template <int DT>
__device__ __forceinline__ void set_apart(Eight<DT>& r) {
    if constexpr (DT != F8MI_FP32)
#pragma unroll
        for (uint32_t& w : r.w) asm("" : "+v"(w));
}

// maximum over the 16 lanes that hold a row; two 16-bit maxima side by side, or one of 32 bits
template <int DT>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (DT == F8MI_FP32) return a > b ? a : b;
    else return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int DT>
__device__ __forceinline__ uint32_t max_of_16_lanes(uint32_t v) {
    v = larger<DT>(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));  // row_ror 1, 2, 4, 8
    v = larger<DT>(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
    v = larger<DT>(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    return larger<DT>(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));
}
// fp32 bits of the magnitude whose bits in its own type these are
template <int DT>
__device__ __forceinline__ uint32_t widen_bits(uint32_t bits) { return __float_as_uint(abs_bits_to_float(bits, DT)); }

__device__ __forceinline__ void transpose4x4(const uint32_t (&r)[4], uint32_t (&c)[4]) {  // c[j]: byte j of the four rows
    const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
    const uint32_t d = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), e = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
    c[0] = __builtin_amdgcn_perm(d, a, 0x05040100u);
    c[1] = __builtin_amdgcn_perm(d, a, 0x07060302u);
    c[2] = __builtin_amdgcn_perm(e, b, 0x05040100u);
    c[3] = __builtin_amdgcn_perm(e, b, 0x07060302u);
}

// v and that of the lanes 16 and 32 further on and back: over the four rows of 16 lanes, in all of them
__device__ __forceinline__ float sum_of_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

template <int DT, bool ALIGNED>
__global__ __launch_bounds__(BC_THREADS) void block_cast_kernel(const BlockCastItem first, const BlockCastItem second, int tiles_first) {
    constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2;
    constexpr int CW = DT == F8MI_FP32 ? 8 : 4;  // words of a lane's column maxima
    __shared__ __align__(16) uint8_t turned[BLOCK * BLOCK];
    __shared__ __align__(16) uint32_t col_max[4][16 * CW];
    __shared__ __align__(16) uint8_t row_bytes[BLOCK], col_bytes[BLOCK];
    __shared__ __align__(16) float col_sum[4][BLOCK];
    const int bid = ALIGNED ? (int)blockIdx.x : xcd_contiguous_id(blockIdx.x, gridDim.x);
    const bool in_first = bid < tiles_first;
    BlockCastItem it = first;  // (field by field: a choice of the whole went through memory)
    if (!in_first) {
        it.x = second.x; it.rows = second.rows; it.cols = second.cols; it.ld = second.ld;
        it.out = second.out; it.out_scales = second.out_scales; it.out_t = second.out_t; it.out_t_scales = second.out_t_scales;
        it.sums = second.sums; it.square = second.square; it.tiles_c = second.tiles_c;
    }
    const int tile = bid - (in_first ? 0 : tiles_first);
    const int tr = tile / it.tiles_c, tc = tile % it.tiles_c;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, tx = t & 15, ty = t >> 4;
    const int64_t r0 = (int64_t)tr * BLOCK, c0 = (int64_t)tc * BLOCK, col = c0 + 8 * tx;

    Eight<DT> v[8];  // rows 64 h + 4 ty + i at 4 h + i
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int64_t row = r0 + 64 * (i >> 2) + 4 * ty + (i & 3);
        v[i] = load_eight<DT, ALIGNED>(it.x + row * it.ld * SIZE, col, it.cols, row < it.rows);
    }

    // maxima of the rows, in every lane of a row: row i in half i % 2 of word i / 2 (fp32: a word each)
    uint32_t rmax[DT == F8MI_FP32 ? 8 : 4];
    if constexpr (DT == F8MI_FP32) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t m = 0u;
#pragma unroll
            for (int j = 0; j < 8; j++) m = max(m, v[i].w[j] & 0x7fffffffu);
            rmax[i] = m;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t m[2] = {0u, 0u};
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int j = 0; j < 4; j++) m[h] = absmax16x2(v[2 * i + h].w[j], m[h]);
                m[h] = fold16(m[h]);
            }
            rmax[i] = m[0] | (m[1] << 16);
        }
    }
#pragma unroll
    for (uint32_t& m : rmax) m = max_of_16_lanes<DT>(m);
    auto row_max = [&](int i) __attribute__((always_inline)) {
        if constexpr (DT == F8MI_FP32) return rmax[i];
        else return widen_bits<DT>((rmax[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    };

    if (it.sums) {  // the same for the whole workgroup, as all of `it`
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            float s[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                s[c] = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) s[c] += value(v[i], j + c);
                s[c] = sum_of_rows(s[c]);
            }
            if (lane < 16) *(float4*)&col_sum[wave][8 * tx + j] = make_float4(s[0], s[1], s[2], s[3]);
        }
    }
    const bool by_cols = it.out_t_scales || it.square;  // the same for the whole workgroup
    uint32_t cmax[CW];
    if (by_cols) {
#pragma unroll
        for (int j = 0; j < CW; j++) {
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 8; i++) m = DT == F8MI_FP32 ? max(m, v[i].w[j] & 0x7fffffffu) : absmax16x2(v[i].w[j], m);
            m = larger<DT>(m, (uint32_t)__shfl_xor((int)m, 16, 64));
            cmax[j] = larger<DT>(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        }
        if (lane < 16) {
#pragma unroll
            for (int j = 0; j < CW; j += 4) *(uint4*)&col_max[wave][lane * CW + j] = make_uint4(cmax[j], cmax[j + 1], cmax[j + 2], cmax[j + 3]);
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int j = 0; j < CW; j++) cmax[j] = larger<DT>(cmax[j], col_max[w][tx * CW + j]);
    }
    uint32_t all = 0u;  // fp32 bits of the tile's maximum
    if (it.square) {
#pragma unroll
        for (int j = 0; j < CW; j++) all = larger<DT>(all, cmax[j]);
        all = max_of_16_lanes<DT>(all);
        all = DT == F8MI_FP32 ? all : widen_bits<DT>(fold16(all));
    }

    if (it.out) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int in_tile = 64 * (i >> 2) + 4 * ty + (i & 3);
            const uint32_t m = it.square ? all : row_max(i);
            const float f = block_factor(m);
            if (tx == 0) row_bytes[block_scale_at(in_tile)] = (uint8_t)block_exponent(m);
            const uint32_t lo = cvt4_fp8<F8MI_E4M3FN>(value(v[i], 0) * f, value(v[i], 1) * f, value(v[i], 2) * f, value(v[i], 3) * f);
            const uint32_t hi = cvt4_fp8<F8MI_E4M3FN>(value(v[i], 4) * f, value(v[i], 5) * f, value(v[i], 6) * f, value(v[i], 7) * f);
            const int64_t row = r0 + in_tile;
            if (row < it.rows) *(uint2*)(it.out + ((col >> 6) * it.rows + row) * 64 + (col & 63)) = make_uint2(lo, hi);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) set_apart<DT>(v[i]);
    if (it.out_t_scales) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t m = all;
            if (!it.square) m = DT == F8MI_FP32 ? cmax[j < CW ? j : 0] : widen_bits<DT>((cmax[(j >> 1) & (CW - 1)] >> (16 * (j & 1))) & 0xffffu);
            f[j] = block_factor(m);
            if (ty == 0) col_bytes[block_scale_at(8 * tx + j)] = (uint8_t)block_exponent(m);
        }
        if (it.out_t)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t r[4], c[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const Eight<DT>& e = v[4 * h + i];
                    r[i] = cvt4_fp8<F8MI_E4M3FN>(value(e, 4 * q) * f[4 * q], value(e, 4 * q + 1) * f[4 * q + 1], value(e, 4 * q + 2) * f[4 * q + 2], value(e, 4 * q + 3) * f[4 * q + 3]);
                }
                transpose4x4(r, c);
                // column 8 tx + 4 q + j, rows 64 h + 4 ty .. + 3: dword 16 h + ty of its 32, swizzled by the column's group of 8
#pragma unroll
                for (int j = 0; j < 4; j++) *(uint32_t*)&turned[(8 * tx + 4 * q + j) * BLOCK + 4 * ((16 * h + ty) ^ ((tx & 7) << 2))] = c[j];
            }
    }
    __syncthreads();
    if (it.sums && t < BLOCK && c0 + t < it.cols) it.sums[tr * it.cols + c0 + t] = (col_sum[0][t] + col_sum[1][t]) + (col_sum[2][t] + col_sum[3][t]);
    if (it.out_t) {
        const int64_t rows_kept = it.cols;  // of the transposed copy
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const int u = p >> 1, c = 64 * (p & 1) + (t >> 2), piece = 4 * u + (t & 3);
            if (c0 + c < rows_kept) {
                const uint4 d = *(const uint4*)&turned[c * BLOCK + 16 * (piece ^ ((c >> 3) & 7))];
                *(uint4*)(it.out_t + ((2 * (int64_t)tr + u) * rows_kept + c0 + c) * 64 + 16 * (t & 3)) = d;
            }
        }
    }
    if (it.out_t_scales && t >= 64 && t < 96) *(uint32_t*)(it.out_t_scales + tr * block_rows_padded(it.cols) + c0 + 4 * (t - 64)) = *(const uint32_t*)&col_bytes[4 * (t - 64)];
    if (it.out && t < 32) *(uint32_t*)(it.out_scales + tc * block_rows_padded(it.rows) + r0 + 4 * t) = *(const uint32_t*)&row_bytes[4 * t];
}

template <int DT>
static int launch_block_cast(const BlockCastItem& a, const BlockCastItem& b, int tiles_a, int tiles, bool aligned, hipStream_t stream) {
    if (aligned) hipLaunchKernelGGL((block_cast_kernel<DT, true>), dim3((unsigned)tiles), dim3(BC_THREADS), 0, stream, a, b, tiles_a);
    else hipLaunchKernelGGL((block_cast_kernel<DT, false>), dim3((unsigned)tiles), dim3(BC_THREADS), 0, stream, a, b, tiles_a);
    return check_hip(hipGetLastError(), "block cast kernel launch");
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int64_t f8mi_block_scale_bytes(int64_t rows, int64_t k) { return rows <= 0 || k <= 0 ? 0 : f8mi_padded_k(k) / BLOCK * block_rows_padded(rows); }

extern "C" int f8mi_block_cast(const f8mi_block_cast_job* jobs, int count, void* stream) {
    if (!jobs || count < 1 || count > 2) { set_error("f8mi_block_cast: one or two tensors"); return F8MI_ERR_INVALID_ARG; }
    BlockCastItem items[2];
    int64_t tiles[2] = {0, 0};
    for (int i = 0; i < count; i++) {
        const f8mi_block_cast_job& j = jobs[i];
        if (j.rows <= 0 || j.cols <= 0 || (j.ld < j.cols && j.ld != 0)) { set_error("f8mi_block_cast: bad shape rows=%lld cols=%lld ld=%lld", (long long)j.rows, (long long)j.cols, (long long)j.ld); return F8MI_ERR_INVALID_ARG; }
        if (j.dtype < 0 || j.dtype > 2) { set_error("f8mi_block_cast: unknown dtype code %d", j.dtype); return F8MI_ERR_INVALID_ARG; }
        if (!j.x || (!j.out && !j.out_t && !j.col_sums) || !j.out != !j.out_scales || (j.out_t && !j.out_t_scales) || (j.out_t_scales && !j.out_t && !(j.square && j.out))) { set_error("f8mi_block_cast: null pointer, or a copy without its scales"); return F8MI_ERR_INVALID_ARG; }
        for (const void* p : {(const void*)j.out, (const void*)j.out_scales, (const void*)j.out_t, (const void*)j.out_t_scales})
            if ((uintptr_t)p % 16 != 0) { set_error("f8mi_block_cast: copies and scales are 16-byte aligned"); return F8MI_ERR_INVALID_ARG; }
        if ((uintptr_t)j.col_sums % 4 != 0) { set_error("f8mi_block_cast: column sums not aligned to a float"); return F8MI_ERR_INVALID_ARG; }
        if ((uintptr_t)j.x % (j.dtype == F8MI_FP32 ? 4 : 2) != 0) { set_error("f8mi_block_cast: input not aligned to its elements"); return F8MI_ERR_INVALID_ARG; }
        const int64_t tiles_c = (j.cols + BLOCK - 1) / BLOCK;
        tiles[i] = tiles_c * ((j.rows + BLOCK - 1) / BLOCK);
        if (tiles_c > 0x3fffffff || tiles[i] > 0x3fffffff) { set_error("f8mi_block_cast: more than 2^30 tiles of 128 x 128"); return F8MI_ERR_UNSUPPORTED; }
        items[i] = {(const uint8_t*)j.x, j.rows, j.cols, j.ld, (uint8_t*)j.out, (uint8_t*)j.out_scales, (uint8_t*)j.out_t, (uint8_t*)j.out_t_scales, j.col_sums, j.square != 0, (int)tiles_c};
    }
    hipStream_t s = (hipStream_t)stream;
    if (count == 2 && jobs[0].dtype != jobs[1].dtype) {
        if (int rc = f8mi_block_cast(jobs, 1, stream)) return rc;
        return f8mi_block_cast(jobs + 1, 1, stream);
    }
    double elements = 0.0;
    for (int i = 0; i < count; i++) elements += (double)jobs[i].rows * (double)jobs[i].cols;
    ProfScope prof(F8MI_K_CAST, elements * (jobs[0].dtype == F8MI_FP32 ? 4 : 2), s);
    const int total = (int)(tiles[0] + tiles[1]);
    if (count == 1) items[1] = items[0];
    bool aligned = true;
    for (const BlockCastItem& it : items) aligned &= (uintptr_t)it.x % 16 == 0 && it.ld * (jobs[0].dtype == F8MI_FP32 ? 4 : 2) % 16 == 0;
    if (jobs[0].dtype == F8MI_BF16) return launch_block_cast<F8MI_BF16>(items[0], items[1], (int)tiles[0], total, aligned, s);
    if (jobs[0].dtype == F8MI_FP16) return launch_block_cast<F8MI_FP16>(items[0], items[1], (int)tiles[0], total, aligned, s);
    return launch_block_cast<F8MI_FP32>(items[0], items[1], (int)tiles[0], total, aligned, s);
}
