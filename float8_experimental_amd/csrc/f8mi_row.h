// Rows of a matrix in registers, for the norms over the last dimension: a row lies in the registers of T lanes, VPT pieces of 16 bytes a lane.
#pragma once
#include <type_traits>

#include "f8mi_gemm_util.h"

namespace f8mi {

template <int DT>
struct Ln {
    static constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2, V = 16 / SIZE;  // values of a lane's 16 bytes
};

template <int DT>
__device__ __forceinline__ void ln_unpack(uint4 q, float (&v)[Ln<DT>::V]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == F8MI_FP32) v[i] = __uint_as_float(w[i]);
        else unpack2<DT>(w[i], v[2 * i], v[2 * i + 1]);
    }
}
// Values col .. col + V - 1 of a row zeros past its end: there the last V values of the row are read and shifted (element by element that
// part held 30 registers more, in every lane).  I: int, or int64_t where columns may need it.
template <int DT, typename I>
__device__ __forceinline__ uint4 ln_load(const uint8_t* row, I col, I cols) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    if (col + V <= cols) return load_nt16_any(row + std::make_unsigned_t<I>(col * SIZE));
    uint64_t lo = 0, hi = 0;
    if (col < cols && cols >= V) {
        const uint4 q = load_nt16_any(row + (cols - V) * SIZE);
        const int shift = (int)(col + V - cols) * SIZE * 8;  // 0 < shift < 128
        lo = q.x | (uint64_t)q.y << 32;
        hi = q.z | (uint64_t)q.w << 32;
        lo = shift >= 64 ? hi >> (shift - 64) : (lo >> shift) | (hi << (64 - shift));
        hi = shift >= 64 ? 0 : hi >> shift;
    } else {
#pragma unroll 1
        for (I i = col; i < cols; i++) {  // a row of less than V values
            const uint64_t e = DT == F8MI_FP32 ? ((const uint32_t*)row)[i] : ((const uint16_t*)row)[i];
            const int at = (int)(i - col) * SIZE * 8;
            if (at < 64) lo |= e << at;
            else hi |= e << (at - 64);
        }
    }
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}
template <int DT>
__device__ __forceinline__ uint4 ln_pack(const float (&v)[Ln<DT>::V]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == F8MI_FP32) w[i] = __float_as_uint(v[i]);
        else w[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT, typename I>
__device__ __forceinline__ void ln_store(uint8_t* row, I col, I cols, const float (&v)[Ln<DT>::V]) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    const uint4 w = ln_pack<DT>(v);
    if (col + V <= cols) {
        store16_any(row + std::make_unsigned_t<I>(col * SIZE), w);
        return;
    }
    uint64_t lo = w.x | (uint64_t)w.y << 32, hi = w.z | (uint64_t)w.w << 32;
#pragma unroll 1
    for (; col < cols; col++) {
        if constexpr (DT == F8MI_FP32) ((uint32_t*)row)[col] = (uint32_t)lo;
        else ((uint16_t*)row)[col] = (uint16_t)lo;
        lo = lo >> (SIZE * 8) | hi << (64 - SIZE * 8);
        hi >>= SIZE * 8;
    }
}
// What is unpacked after this is not kept from before: 16-bit rows stay packed while their sums are waited for.
template <int DT>
__device__ __forceinline__ void set_apart(uint4& q) {
    if constexpr (DT != F8MI_FP32) asm("" : "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w));
}
// V values of a parameter (`otherwise` without one)
template <int PT, int V, typename I>
__device__ __forceinline__ void ln_param(const void* p, I col, I cols, float otherwise, float (&v)[V]) {
    constexpr int PV = Ln<PT>::V;
#pragma unroll
    for (int i = 0; i < V; i += PV) {
        float f[PV];
        if (p) {
            ln_unpack<PT>(ln_load<PT, I>((const uint8_t*)p, col + i, cols), f);
        } else {
#pragma unroll
            for (int j = 0; j < PV; j++) f[j] = otherwise;
        }
#pragma unroll
        for (int j = 0; j < PV; j++) v[i + j] = f[j];
    }
}

// The sum over a wave, in every lane: rotations inside the rows of 16 lanes, then exchanges of rows and halves
template <int CTRL>
__device__ __forceinline__ float plus_rotated(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = plus_rotated<0x128>(plus_rotated<0x124>(plus_rotated<0x122>(plus_rotated<0x121>(v))));  // row_ror 1, 2, 4, 8
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}
// Two sums over the T lanes of a row, in every one of them.  `slots`: two floats for each wave of the workgroup, not in use elsewhere
// until the next barrier but one.
template <int T>
__device__ __forceinline__ void row_sums(float& a, float& b, float2* slots) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (T > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slots[wave] = make_float2(a, b);
        __syncthreads();
        const int first = wave / (T / 64) * (T / 64);
        a = b = 0.f;
#pragma unroll 4
        for (int i = 0; i < T / 64; i++) {
            const float2 s = slots[first + i];
            a += s.x;
            b += s.y;
        }
    }
}

// What a lane holds of a row: VPT pieces of V values, T * V apart.  The last may lie past the end of the row: it is moved back to end there
// (no branch, nothing shifted; with those a lane's addresses and shifts took the registers of a piece), and `off` counts the values at
// its start that the lane before holds too: they stay out of sums, and are stored twice, the same.  With 64 lanes a row may be shorter than a
// piece: there values past the end are zeros, and `off` counts the others.
template <int T, int VPT, int V>
struct LnLane {
    int t, last, off;
    __device__ __forceinline__ LnLane(int t_, int cols) : t(t_), last(((VPT - 1) * T + t_) * V) {
        if constexpr (T == 64) {
            off = min(max(cols - last, 0), V);
        } else {
            const int col = last;
            last = min(col, cols - V);
            off = min(col - last, V);
        }
    }
    __device__ __forceinline__ int col(int p) const { return p < VPT - 1 ? (p * T + t) * V : last; }
    __device__ __forceinline__ bool has(int p, int i) const { return p < VPT - 1 || (T == 64 ? i < off : i >= off); }
    __device__ __forceinline__ bool any(int p) const { return p < VPT - 1 || (T == 64 ? off > 0 : off < V); }
    // row: the same in a wave, and kept apart from the lane's offset, or each piece has its own 64-bit address in registers for the whole loop
    template <int DT>
    __device__ __forceinline__ uint4 load(const uint8_t* row, int p, int cols) const {
        if constexpr (T == 64) return ln_load<DT, int>(row, last, cols);
        asm("" : "+s"(row));
        return load_nt16_any(row + (uint32_t)(col(p) * Ln<DT>::SIZE));
    }
    template <int DT>
    __device__ __forceinline__ void store(uint8_t* row, int p, int cols, const float (&v)[V]) const {
        if (!any(p)) return;
        if constexpr (T == 64) return ln_store<DT, int>(row, last, cols, v);
        asm("" : "+s"(row));
        store16_any(row + (uint32_t)(col(p) * Ln<DT>::SIZE), ln_pack<DT>(v));
    }
};

// A parameter in LDS: 16-byte parts of a piece of V values lie `pieces` apart, so that lanes next to each other read without conflicts.
template <int PT, int V>
struct LnShared {
    static constexpr int PV = Ln<PT>::V, PARTS = V / PV;
    uint4* at;
    int pieces;
    __device__ __forceinline__ void fill(const void* p, int cols, float otherwise) {
        for (int i = threadIdx.x; i < pieces * PARTS; i += blockDim.x) {
            const int part = i / pieces, piece = i - part * pieces;
            uint4 q;
            if (p) {
                q = load_nt16_any((const uint8_t*)p + (uint32_t)((min(piece * V, cols - V) + part * PV) * Ln<PT>::SIZE));
            } else {
                const uint32_t one = PT == F8MI_FP32 ? __float_as_uint(otherwise) : pack2<PT == F8MI_FP32 ? F8MI_BF16 : PT>(otherwise, otherwise);
                q = make_uint4(one, one, one, one);
            }
            at[i] = q;
        }
    }
    __device__ __forceinline__ void read(int piece, float (&v)[V]) const {
        piece = min(piece, pieces - 1);
#pragma unroll
        for (int part = 0; part < PARTS; part++) {
            float f[PV];
            ln_unpack<PT>(at[part * pieces + piece], f);
#pragma unroll
            for (int j = 0; j < PV; j++) v[part * PV + j] = f[j];
        }
    }
};

}  // namespace f8mi
