// Low-rank adapters of many requests beside one projection (f8mi_adapters.h), forward and backward:
//   h_i = A_e x_i,  out_i = y_i + scale_e B_e h_i,
//   dh_i = B_e^T dout_i,  dx_i = scale_e A_e^T dh_i,  dA_e = scale_e sum_i dh_i x_i^T,  dB_e = scale_e sum_i dout_i h_i^T.
// Three kernels: `shrink` (h from x and A, dh from dout and B^T), `expand` (out from y, h and B; dx from dh and A^T) and `outer` (dA, dB); for few rows `whole`, the first two in one.  The
// transposed copies of the adapters that backward needs of short tiles and in fp32 are made by a fourth; they are small beside x.
//
// HBM-bound: x, y and dout are read once each, out and dx written, an adapter is read by each of its tiles out of the L2.  The products run
// on the matrix cores straight from registers: a lane's 16 bytes of a row, loaded as they lie, are its operand.  The order of a contraction is free as long
// as both operands have the same one, so the four lanes that share a row take 64 neighbouring bytes of it, two instructions a line of the cache.
//
// h and dh are sums and stay in 32 bits: 16-bit matrix instructions get them as the sum of two 16-bit values (an error of 2^-17 of h, where one alone
// would be off by as much as the rounding of the result), fp16 ones after a power of two for each row, so that nothing overflows, and of the row's largest no more
// than 2^-39 is lost among the subnormals.
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

typedef short s16x4 __attribute__((ext_vector_type(4)));
// ds_read_b64_tr_b16: the 16 lanes of a group address 8 bytes each, lane l row l / 4 of four and four of its columns; a lane gets the four rows of one column, that of lane l / 4's
// bytes l % 4.  Two of them, of rows and of the four rows after, are a lane's operand.
__device__ __forceinline__ uint4 read_turned(const uint8_t* rows, const uint8_t* after) {
    typedef __attribute__((address_space(3))) s16x4* at;
    const uint2 l = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)rows)), h = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)after));
    return make_uint4(l.x, l.y, h.x, h.y);
}
// Rows of 16-bit values with an odd pitch begin at odd multiples of two bytes every other time, where an access of 16 bytes takes three times as long (4099 x 4097: 32 us to read instead
// of 10).  ODD: the words around them instead, moved by half a word.  No word is read that holds none of the 16 bytes.
template <bool ODD>
__device__ __forceinline__ uint4 load16_at(const uint8_t* p) {
    if constexpr (!ODD) return load16_any(p);
    const uint32_t off = (uint32_t)(uintptr_t)p & 2u, shift = off * 8;
    const uint4 q = load16_any(p - off);
    const uint32_t next = *(const u32_any*)(p - off + (off ? 16 : 12));
    return make_uint4(__builtin_amdgcn_alignbit(q.y, q.x, shift), __builtin_amdgcn_alignbit(q.z, q.y, shift), __builtin_amdgcn_alignbit(q.w, q.z, shift),
                      __builtin_amdgcn_alignbit(off ? next : 0u, q.w, shift));
}

// V values of a row of r, from column col on, zeros past its end: `from` is their place in a tensor of `total` values.  WHOLE: r is a multiple of V, so that they all lie in the
// row or none does.  No branch, so that many are on their way at once: past the end of the tensor its last 16 bytes are read and shifted.
template <int DT, bool WHOLE>
__device__ __forceinline__ uint4 load_of_row(const uint8_t* base, int64_t from, int64_t total, int col, int r) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE;
    if constexpr (WHOLE) {
        const bool in = col < r;
        const uint4 q = load16_any(base + (in ? from : from - col) * SIZE);
        return in ? q : make_uint4(0u, 0u, 0u, 0u);
    } else {
        if (total < V) return ln_load<DT, int>(base + (from - col) * SIZE, col, r);  // (nothing to read 16 bytes of)
        const int64_t at = min(from, total - V);
        const uint4 q = load16_any(base + at * SIZE);
        uint64_t lo = q.x | (uint64_t)q.y << 32, hi = q.z | (uint64_t)q.w << 32;
        const int shift = (int)min(from - at, (int64_t)V) * SIZE * 8, keep = min(max(r - col, 0), V) * SIZE * 8;  // bits
        if (shift) {
            lo = shift >= 64 ? (shift >= 128 ? 0 : hi >> (shift - 64)) : lo >> shift | hi << (64 - shift);
            hi = shift >= 64 ? 0 : hi >> shift;
        }
        lo = keep >= 64 ? lo : keep ? lo & ~0ull >> (64 - keep) : 0;
        hi = keep >= 128 ? hi : keep > 64 ? hi & ~0ull >> (128 - keep) : 0;
        return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    }
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
    int n, cols, chunks;  // cols: of out that a workgroup has; chunks: workgroups a tile
    bool a_turned, b_turned;  // a is [count][k][r], b [count][r][n]: the adapters' other matrices as they lie
};

// ---- shrink: a wave has 16 rows of one adapter, 16 RT of its rank and a part of the contraction; those of a workgroup's waves are added up in LDS
// (16 rows a tile: an adapter of few rows.  64 rows with an adapter each, 8192 values, rank 16: 6.6 us out of HBM; latency.)
constexpr int SHRINK_WAVES = 8;
// The sums of part `split` of `splits` over the workgroup, of the rank from j0 on, to h [tile.rows][rp]
template <int DT, int RT, int DEPTH, int WAVES>  // DEPTH: steps in flight
__device__ __forceinline__ void shrink_rows(const AdapterArgs& g, const AdapterTile& tile, int split, int splits, int j0, float4 (&part)[WAVES][RT][64], float* h_out) {
    constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2, STEP = 128 / SIZE;  // values of a step: a line of the cache of each row
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lm = lane & 15, lq = lane >> 4;
    const int32_t* order = g.table + AdapterTable(g.m, g.count).order() + tile.first;
    const int64_t steps = g.k / STEP, unit = (int64_t)split * WAVES + wave, units = (int64_t)splits * WAVES;
    const int s0 = (int)(steps * unit / units), s1 = (int)(steps * (unit + 1) / units);
    const int at_row = order[min(lm, tile.rows - 1)];  // (waited for behind the first loads of A)
    const uint8_t *px = nullptr, *pa[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) pa[i] = g.a + ((int64_t)tile.group * g.r + min(j0 + i * 16 + lm, g.r - 1)) * g.k * SIZE;

    v4f_l acc[RT] = {};
    uint4 fx[DEPTH][2], fa[DEPTH][RT][2];
    auto load_a = [&](int d, int h, int s) __attribute__((always_inline)) {
        const int64_t at = (int64_t)s * 128 + h * 64 + lq * 16;
#pragma unroll
        for (int i = 0; i < RT; i++) fa[d][i][h] = load16_any(pa[i] + at);
    };
    auto load_x = [&](int d, int h, int s) __attribute__((always_inline)) { fx[d][h] = load16_any(px + (int64_t)s * 128 + h * 64 + lq * 16); };
    auto multiply = [&](int d, int h) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < RT; i++) acc[i] = mfma_16<DT>(fa[d][i][h], fx[d][h], acc[i]);
    };
    if (s0 < s1)
#pragma unroll
        for (int i = 0; i < 2 * DEPTH; i++) load_a(i / 2, i % 2, min(s0 + i / 2, s1 - 1));
    __builtin_amdgcn_sched_barrier(0);
    px = g.x + (int64_t)at_row * g.ld * SIZE;
    if (s0 < s1) {
#pragma unroll
        for (int i = 0; i < 2 * DEPTH; i++) load_x(i / 2, i % 2, min(s0 + i / 2, s1 - 1));
        int s = s0;
        for (; s + DEPTH < s1; s += DEPTH) {
#pragma unroll
            for (int i = 0; i < 2 * DEPTH; i++) {  // what has been multiplied is asked for again at once
                multiply(i / 2, i % 2);
                load_a(i / 2, i % 2, min(s + DEPTH + i / 2, s1 - 1));
                load_x(i / 2, i % 2, min(s + DEPTH + i / 2, s1 - 1));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * DEPTH; i++)
            if (s + i / 2 < s1) multiply(i / 2, i % 2);
    }
    if (unit == units - 1 && steps * STEP < g.k) {  // what is left of the rows
        const int at = (int)steps * STEP + lq * (STEP / 8);
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
            const uint4 tx = ln_load<DT, int>(px, at + h * (STEP / 2), g.k);
#pragma unroll
            for (int i = 0; i < RT; i++) acc[i] = mfma_16<DT>(ln_load<DT, int>(pa[i], at + h * (STEP / 2), g.k), tx, acc[i]);
        }
    }
    // lane l: row l % 16, 4 (l / 16) + e of the rank
#pragma unroll
    for (int i = 0; i < RT; i++) part[wave][i][lane] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    __syncthreads();
    for (int item = threadIdx.x; item < RT * 64; item += 64 * WAVES) {
        const int at = item >> 6, l = item & 63, row = l & 15, j = j0 + at * 16 + 4 * (l >> 4);
        float4 s = part[0][at][l];
#pragma unroll
        for (int w = 1; w < WAVES; w++) {
            const float4 p = part[w][at][l];
            s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
        }
        if (row < tile.rows && j < g.rp) *(float4*)(h_out + row * g.rp + j) = s;
    }
}
template <int DT, int RT>
__global__ __launch_bounds__(64 * SHRINK_WAVES, 4) void adapter_shrink_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    __shared__ float4 part[SHRINK_WAVES][RT][64];
    const int id = xcd_contiguous_id(blockIdx.x, gridDim.x), split = id % g.splits;  // a tile's workgroups, and those of the next ones, on one XCD: A stays in its L2
    const AdapterTile tile = tiles[id / g.splits];
    if (tile.rows == 0 || tile.group >= g.count) return;
    shrink_rows<DT, RT, 2, SHRINK_WAVES>(g, tile, split, g.splits, blockIdx.y * (16 * RT), part, g.partial + ((int64_t)split * g.m + tile.first) * g.rp);
}

// 64 rows of one adapter and 16 RT of its rank a workgroup: a wave has 16 of the rows and brings them itself, all four multiply them by the same part of A, which goes through LDS: BYTES
// of each of its rows at a time, the next ones (and the next ones of x) on their way meanwhile.  A workgroup has a part of the contraction; nothing is left to add up inside it.
// Measured: 8192 rows of 4096 bf16 values, rank 16 22 us (3.0 TB/s), rank 64 24; of 8192, rank 16 37 us (3.6 TB/s).  Two to six workgroups a CU instead of one and a half: no faster.
constexpr int TALL_THREADS = 256;
// ODD: some rows of x begin at odd multiples of two bytes (load16_at): the words around a lane's values are brought, and the last one is the first of the lane that has the next 16 bytes, but for
// one word a step.  TURNED (16-bit types): A is [count][k][r], the other matrix of an adapter as it lies, and is turned on the way out of LDS.
template <int DT, int RT, int BYTES, bool ODD, bool TURNED>
__global__ __launch_bounds__(TALL_THREADS, ODD || (TURNED && RT == 1) ? 3 : 4) void adapter_shrink_tall_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, PIECES = BYTES / 16, KP = RT * 16 * PIECES / TALL_THREADS, STEP = BYTES / SIZE;
    // turned, the rows of 32 RT bytes that 32 lanes read at a time (0 .. 3 and 8 .. 11) lie in different banks: by a half turn of every second eight, or by padding (two of eight meet)
    constexpr int PITCH = !TURNED ? BYTES + 16 : RT == 4 ? 160 : RT * 32;
    __shared__ __align__(16) uint8_t lds_a[2][(TURNED ? STEP : RT * 16) * PITCH];
    auto turned_at = [](int row, int byte) __attribute__((always_inline)) { return (row * PITCH + byte) ^ (RT == 4 ? 0 : (row >> 3 & 1) * (RT == 1 ? 128 : 32)); };
    const int id = xcd_contiguous_id(blockIdx.x, gridDim.x), split = id % g.splits;  // a tile's workgroups, and those of the next ones, on one XCD: A stays in its L2
    const AdapterTile tile = tiles[id / g.splits];
    if (tile.rows == 0 || tile.group >= g.count) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lm = lane & 15, lq = lane >> 4, j0 = blockIdx.y * (16 * RT);
    const int steps = (g.k + STEP - 1) / STEP, s0 = (int)((int64_t)steps * split / g.splits), s1 = (int)((int64_t)steps * (split + 1) / g.splits);
    const int64_t x_row = (int64_t)g.table[AdapterTable(g.m, g.count).order() + tile.first + min(wave * 16 + lm, tile.rows - 1)] * g.ld, x_total = (g.m - 1) * g.ld + g.k;
    const int64_t a_first = TURNED ? (int64_t)tile.group * g.k * g.r : ((int64_t)tile.group * g.r + j0) * g.k, a_total = (int64_t)g.count * g.r * g.k;
    const bool whole = g.r % V == 0;
    v4f_l acc[RT] = {};
    uint4 fa[KP], fx[PIECES / 4], next_x[PIECES / 4];
    const uint32_t off = ODD ? (uint32_t)(uintptr_t)(g.x + x_row * SIZE) & 2u : 0u;
    uint32_t edge = 0u, next_edge = 0u;  // the word behind the step's values of the row
    // (a step that ends with the row or before it, the same for the workgroup, needs no edges)
    auto load_x = [&](int s, uint4 (&q)[PIECES / 4], uint32_t& e) __attribute__((always_inline)) {
        const int k0 = s * STEP + lq * V;
        if ((s + 1) * STEP <= g.k) {
#pragma unroll
            for (int i = 0; i < PIECES / 4; i++) q[i] = load16_any(g.x + (x_row + k0 + i * 4 * V) * SIZE - off);
            if constexpr (ODD)
                if (off && lq == 3) e = *(const u32_any*)(g.x + (x_row + (s + 1) * STEP) * SIZE - off);
        } else {
#pragma unroll
            for (int i = 0; i < PIECES / 4; i++) q[i] = load_of_row<DT, false>(g.x, x_row + k0 + i * 4 * V, x_total, k0 + i * 4 * V, g.k);
        }
    };
    auto load_a = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const int item = i * TALL_THREADS + t;
            if constexpr (TURNED) {  // (zeros behind the last row)
                const int row = s * STEP + item / (2 * RT), j = j0 + item % (2 * RT) * 8;
                fa[i] = make_uint4(0u, 0u, 0u, 0u);
                if (row < g.k) {
                    if (whole) fa[i] = j < g.r ? load16_any(g.a + (a_first + (int64_t)row * g.r + j) * SIZE) : fa[i];
                    else fa[i] = load_of_row<DT, false>(g.a, a_first + (int64_t)row * g.r + j, a_total, j, g.r);
                }
                continue;
            }
            const int row = min(item / PIECES, g.r - 1 - j0), k = s * STEP + item % PIECES * V;
            if ((s + 1) * STEP <= g.k) fa[i] = load16_any(g.a + (a_first + (int64_t)row * g.k + k) * SIZE);
            else fa[i] = load_of_row<DT, false>(g.a, a_first + (int64_t)row * g.k + k, a_total, k, g.k);
        }
    };
    auto keep_a = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const int item = i * TALL_THREADS + t;
            *(uint4*)(lds_a[buffer] + (TURNED ? turned_at(item / (2 * RT), item % (2 * RT) * 16) : item / PIECES * PITCH + item % PIECES * 16)) = fa[i];
        }
    };
    if (s0 < s1) {
        load_a(s0);
        load_x(s0, fx, edge);
        keep_a(0);
        __syncthreads();
    }
    for (int s = s0, buffer = 0; s < s1; s++, buffer ^= 1) {
        const bool more = s + 1 < s1;
        if (more) {
            load_x(s + 1, next_x, next_edge);
            load_a(s + 1);
        }
        if constexpr (ODD)
            if ((s + 1) * STEP <= g.k) {  // (the same for the workgroup)
                const uint32_t shift = off * 8;
                uint32_t got[PIECES / 4 + 1];
#pragma unroll
                for (int i = 0; i < PIECES / 4; i++) got[i] = (uint32_t)__builtin_amdgcn_ds_bpermute((lane + 16) * 4, (int)fx[i].x);
                got[PIECES / 4] = edge;
#pragma unroll
                for (int i = 0; i < PIECES / 4; i++) {
                    const uint4 q = fx[i];
                    const uint32_t next = lq == 3 ? got[i + 1] : got[i];
                    fx[i] = make_uint4(__builtin_amdgcn_alignbit(q.y, q.x, shift), __builtin_amdgcn_alignbit(q.z, q.y, shift), __builtin_amdgcn_alignbit(q.w, q.z, shift),
                                       __builtin_amdgcn_alignbit(next, q.w, shift));
                }
            }
#pragma unroll
        for (int i = 0; i < PIECES / 4; i++)
#pragma unroll
            for (int j = 0; j < RT; j++) {
                uint4 q;
                if constexpr (TURNED) {
                    const int row = i * 32 + lq * 8 + (lm >> 2), byte = j * 32 + (lm & 3) * 8;
                    q = read_turned(lds_a[buffer] + turned_at(row, byte), lds_a[buffer] + turned_at(row + 4, byte));
                } else {
                    q = *(const uint4*)(lds_a[buffer] + (j * 16 + lm) * PITCH + i * 64 + lq * 16);
                }
                acc[j] = mfma_16<DT>(q, fx[i], acc[j]);
            }
        if (more) {
            keep_a(buffer ^ 1);
            lds_barrier();
#pragma unroll
            for (int i = 0; i < PIECES / 4; i++) fx[i] = next_x[i];
            edge = next_edge;
        }
    }
    const int row = wave * 16 + lm;
    if (row < tile.rows)
#pragma unroll
        for (int j = 0; j < RT; j++)
            if (j0 + j * 16 < g.rp) *(float4*)(g.partial + ((int64_t)split * g.m + tile.first + row) * g.rp + j0 + j * 16 + 4 * lq) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
}

// ---- expand: a workgroup has 16 WR rows of one adapter and `cols` columns of out
constexpr int EXPAND_THREADS = 256;
// Columns that the kernel for 64 rows needs: a whole block
constexpr int expand_least(int rp) { return rp <= 32 ? 128 : 64; }
// Of a row of h in LDS: 16-bit types have its high parts, then its low ones, `half` elements each: whole instructions of 32, or 16, where one instruction takes both.
__host__ __device__ constexpr int expand_half(int rp) { return rp <= 16 ? 16 : (rp + 31) / 32 * 32; }
template <int DT>
__host__ __device__ constexpr int expand_pitch(int rp) { return DT == F8MI_FP32 ? rp + 4 : expand_half(rp) * 2 + 8; }

// The parts of h that the contraction's parts gave, added up, scaled and kept in LDS as the products take them: rows first .. of the table's order.  `sums` (fp16 alone): fp32
// [ROWS][half] beside them, free afterwards.
template <int DT, int ROWS, int THREADS = EXPAND_THREADS>
__device__ __forceinline__ void stage_h(const AdapterArgs& g, const AdapterTile& tile, const float* parts, int splits, bool first, uint8_t* kept_bytes, float* sums, uint32_t* row_most, float& factor, int my_row) {
    const int t = threadIdx.x, rp = g.rp, pitch = expand_pitch<DT>(rp), half = DT == F8MI_FP32 ? rp : expand_half(rp), quads = half / 4;
    const float scale = g.factor * (g.scale ? g.scale[tile.group] : 1.f);
    auto keep = [&](int row, int j, const float (&v)[4]) __attribute__((always_inline)) {
        uint32_t high[2], low[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float a, b;
            high[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
            unpack2<DT>(high[i], a, b);
            low[i] = pack2<DT>(a - a == 0.f ? v[2 * i] - a : 0.f, b - b == 0.f ? v[2 * i + 1] - b : 0.f);  // (nothing is left of an infinity)
        }
        uint16_t* at = (uint16_t*)kept_bytes + row * pitch + j;
        *(uint2*)at = make_uint2(high[0], high[1]);
        *(uint2*)(at + half) = make_uint2(low[0], low[1]);
    };
    if constexpr (DT == F8MI_FP16) {
        if (t < ROWS) row_most[t] = 0u;
        __syncthreads();
    }
    for (int item = t; item < ROWS * quads; item += THREADS) {
        const int row = item / quads, j = (item - row * quads) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (row < tile.rows && j < rp) {
            const float* p = parts + row * rp + j;
#pragma unroll 4
            for (int i = 0; i < splits; i++) {
                const float4 q = *(const float4*)(p + i * g.m * rp);
                v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (j + e >= g.r) v[e] = 0.f;  // (rows of A past the last are the last again)
            if (g.h && first) *(float4*)(g.h + ((int64_t)tile.first + row) * rp + j) = make_float4(v[0], v[1], v[2], v[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] *= scale;
        if constexpr (DT == F8MI_BF16) keep(row, j, v);
        else *(float4*)(DT == F8MI_FP32 ? (float*)kept_bytes + row * pitch + j : sums + item * 4) = make_float4(v[0], v[1], v[2], v[3]);
        if constexpr (DT == F8MI_FP16) {
            uint32_t most = 0u;
#pragma unroll
            for (int e = 0; e < 4; e++) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
            atomicMax(&row_most[row], most);  // (in LDS; a maximum has no order)
        }
    }
    __syncthreads();
    factor = 1.f;
    if constexpr (DT == F8MI_FP16) {  // a power of two, 2^(141 - e), that brings the row's largest to [2^14, 2^15): the low parts of values down to 2^-23 of it have their bits (brought
        // to [1, 2), those of 2^-9 had lost some, and where B takes no part of the large ones, that was the result); 2^39 at most, of 256 of the rank, in the sums
        auto exponent = [&](int row) __attribute__((always_inline)) { return (uint32_t)min(max((int)(row_most[row] >> 23), 15), 254); };
        for (int item = t; item < ROWS * quads; item += THREADS) {
            const int row = item / quads;
            const float4 q = *(const float4*)(sums + item * 4);
            const float f = __uint_as_float((268u - exponent(row)) << 23);
            const float v[4] = {q.x * f, q.y * f, q.z * f, q.w * f};
            keep(row, (item - row * quads) * 4, v);
        }
        factor = __uint_as_float((exponent(my_row) - 14u) << 23);
        __syncthreads();
    }
}

// Of out and y, 64 columns from n0: a lane's pieces of 16 bytes of its row, those of the four lanes that share it next to each other, so that an instruction takes 64 bytes of each row.
// (Not past the caches: these are half lines; a copy of 8192 x 14336 in such pieces takes 95 us, past the caches 122.)
// EDGE: some may lie past the last.  ODD: load16_at, and stores of whole words, a value moved on from lane to lane, where a row begins at an odd multiple of two bytes.
template <int DT, bool EDGE, bool ODD = false>
struct ExpandCols {
    static constexpr int V = Ln<DT>::V, SIZE = Ln<DT>::SIZE, PIECES = 16 / V;
    int n0, n, lq, lm;
    __device__ __forceinline__ int col(int p) const { return n0 + p * 4 * V + lq * V; }
    // row q of the matrix instructions' tile c: four columns of piece c / (V / 4) of the lane q / 4
    __device__ __forceinline__ int of_tile(int c) const { return n0 + c / (V / 4) * 4 * V + (lm >> 2) * V + c % (V / 4) * 4 + (lm & 3); }
    __device__ __forceinline__ bool inside() const { return !EDGE || n0 + 64 <= n; }  // the same for the wave
    __device__ __forceinline__ void load(const uint8_t* row, uint4 (&q)[PIECES]) const {
        if (inside()) {
#pragma unroll
            for (int p = 0; p < PIECES; p++) q[p] = load16_at<ODD>(row + (int64_t)col(p) * SIZE);
        } else {
#pragma unroll
            for (int p = 0; p < PIECES; p++) q[p] = ln_load<DT, int>(row, col(p), n);
        }
    }
    // y + acc * factor (adapted: a row without an adapter keeps y's bits)
    __device__ __forceinline__ void store(uint8_t* row, const uint4 (&q)[PIECES], const v4f_l* acc, float factor, bool adapted) const {
        uint32_t before = 0u;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            float v[V];
            ln_unpack<DT>(q[p], v);
            if (adapted)
#pragma unroll
                for (int e = 0; e < V; e++) v[e] = __builtin_fmaf(acc[(p * V + e) / 4][e % 4], factor, v[e]);
            if constexpr (ODD) {
                uint4 w = ln_pack<DT>(v);
                const bool odd = (uintptr_t)row & 2;
                const bool first = odd && p == 0 && lq == 0, last = odd && p == PIECES - 1 && lq == 3;
                // the value before these eight: of the lane 16 before, or that of the piece before 48 after
                const uint32_t got = (uint32_t)__builtin_amdgcn_ds_bpermute((int)((threadIdx.x & 63) - 16) * 4, (int)w.w), own = w.w;
                const uint32_t prev = lq == 0 ? before : got;
                before = got;
                uint8_t* at = row + (int64_t)col(p) * SIZE;
                if (first) *(uint16_t*)at = (uint16_t)w.x;
                if (odd) w = make_uint4(w.x << 16 | prev >> 16, __builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16), __builtin_amdgcn_alignbit(w.w, w.z, 16));
                if (first) {
                    store8_any(at + 2, w.y, w.z);
                    *(u32_any*)(at + 10) = w.w;
                } else {
                    store16_any(at - (odd ? 2 : 0), w);
                }
                if (last) *(uint16_t*)(at + 14) = (uint16_t)(own >> 16);
            } else if (inside()) store16_any(row + (int64_t)col(p) * SIZE, ln_pack<DT>(v));
            else if (col(p) < n) ln_store<DT, int>(row, col(p), n, v);
        }
    }
};

// A wave has 16 rows and 64 columns at a time, the waves below each other (WR 4) or side by side (1); B straight out of the caches.
// The last 64 columns are moved back to end with the last one (those before are computed twice, the same); EDGE: there are less than 64.
template <int DT, int WR, bool WHOLE, bool EDGE>
__global__ __launch_bounds__(EXPAND_THREADS, WHOLE && !EDGE ? 4 : 1) void adapter_expand_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    constexpr int SIZE = Ln<DT>::SIZE, ROWS = 16 * WR, STEP = WR > 1 ? 64 : 256;
    extern __shared__ __align__(16) uint8_t expand_lds[];  // h [ROWS][pitch], then (fp16) fp32 [ROWS][half] while it is converted
    __shared__ uint32_t row_most[DT == F8MI_FP16 ? ROWS : 1];
    const int id = xcd_contiguous_id(blockIdx.x, gridDim.x), chunk = id % g.chunks;  // a tile's workgroups, and those of the next ones, on one XCD: B stays in its L2
    const AdapterTile tile = tiles[id / g.chunks];
    if (tile.rows == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lm = lane & 15, lq = lane >> 4;
    const bool none = tile.group >= g.count;
    const int rp = g.rp, pitch = expand_pitch<DT>(rp), half = expand_half(rp);
    const int my_row = (WR > 1 ? wave * 16 : 0) + lm;
    float factor = 1.f;
    if (!none) stage_h<DT, ROWS>(g, tile, g.partial + (int64_t)tile.first * rp, g.splits, chunk == 0, expand_lds, (float*)(expand_lds + ROWS * pitch * SIZE), row_most, factor, my_row);
    if (WR > 1 && wave * 16 >= tile.rows) return;
    const int64_t at_row = g.table[AdapterTable(g.m, g.count).order() + tile.first + min(my_row, tile.rows - 1)];
    const uint8_t *hrow = expand_lds + my_row * pitch * SIZE, *y_row = g.y + at_row * g.ld_y * SIZE;
    uint8_t* out_row = g.out + at_row * g.n * SIZE;
    const int end = min(g.n, (chunk + 1) * g.cols);
    const int64_t b_total = (int64_t)g.count * g.n * g.r;
    for (int n0 = chunk * g.cols + (WR > 1 ? 0 : wave * 64); n0 < end; n0 += STEP) {
        const ExpandCols<DT, EDGE> at{EDGE ? n0 : min(n0, g.n - 64), g.n, lq, lm};
        uint4 fy[ExpandCols<DT, EDGE>::PIECES] = {};
        if (g.y) at.load(y_row, fy);
        v4f_l acc[4] = {};
        if (!none) {
            int64_t pb[4];
#pragma unroll
            for (int c = 0; c < 4; c++) pb[c] = ((int64_t)tile.group * g.n + (EDGE ? min(at.of_tile(c), g.n - 1) : at.of_tile(c))) * g.r;
            auto load_b = [&](uint4 (&fb)[4], int j) __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c < 4; c++) fb[c] = load_of_row<DT, WHOLE>(g.b, pb[c] + j, b_total, j, g.r);
            };
            if constexpr (DT == F8MI_FP32) {
                for (int j = 0; j < rp; j += 16) {
                    uint4 fb[4];
                    load_b(fb, j + lq * 4);
                    const uint4 fh = *(const uint4*)(hrow + (j + lq * 4) * 4);
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c] = mfma_16<DT>(fb[c], fh, acc[c]);
                }
            } else if (half == 16) {  // both parts of h in one instruction, B twice
                uint4 fb[4];
                load_b(fb, (lq & 1) * 8);
                const uint4 fh = *(const uint4*)(hrow + lq * 16);
#pragma unroll
                for (int c = 0; c < 4; c++) acc[c] = mfma_16<DT>(fb[c], fh, acc[c]);
            } else {
                uint4 fb[2][4];  // the next part of the rank is on its way while one is multiplied
                load_b(fb[0], lq * 8);
                for (int j = 0; j < half; j += 64) {
#pragma unroll
                    for (int d = 0; d < 2; d++) {
                        const int k = j + d * 32;
                        if (k >= half) break;
                        if (k + 32 < half) load_b(fb[d ^ 1], k + 32 + lq * 8);
                        const uint4 high = *(const uint4*)(hrow + (k + lq * 8) * 2), low = *(const uint4*)(hrow + (half + k + lq * 8) * 2);
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[c] = mfma_16<DT>(fb[d][c], low, mfma_16<DT>(fb[d][c], high, acc[c]));
                    }
                }
            }
        }
        if (my_row < tile.rows) at.store(out_row, fy, acc, factor, !none);
    }
}

// Both products of 16 rows of one adapter of rank 16 or less in one launch: each workgroup of a tile has 64 columns a wave and finds all of h for itself, A out of the L2 but for the first of
// them.  B and y are on their way meanwhile.
constexpr int WHOLE_COLS = 64 * SHRINK_WAVES;
template <int DT, bool WHOLE>
__global__ __launch_bounds__(64 * SHRINK_WAVES, 4) void adapter_whole_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    constexpr int SIZE = Ln<DT>::SIZE, ROWS = 16, PITCH = expand_pitch<DT>(16);
    __shared__ float4 part[SHRINK_WAVES][1][64];
    __shared__ __align__(16) float h[ROWS * 16], sums[DT == F8MI_FP16 ? ROWS * 16 : 4];
    __shared__ __align__(16) uint8_t kept[ROWS * PITCH * SIZE];
    __shared__ uint32_t row_most[DT == F8MI_FP16 ? ROWS : 1];
    const int id = xcd_contiguous_id(blockIdx.x, gridDim.x), chunk = id % g.chunks;
    const AdapterTile tile = tiles[id / g.chunks];
    if (tile.rows == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lm = lane & 15, lq = lane >> 4;
    const bool none = tile.group >= g.count;
    const int64_t at_row = g.table[AdapterTable(g.m, g.count).order() + tile.first + min(lm, tile.rows - 1)];
    const int n0 = chunk * WHOLE_COLS + wave * 64;
    const ExpandCols<DT, false> at{min(n0, g.n - 64), g.n, lq, lm};  // (the last 64 columns are moved back as in the other kernels)
    uint4 fy[ExpandCols<DT, false>::PIECES] = {}, fb[4] = {};
    if (n0 < g.n) {
        if (!none)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int j = DT == F8MI_FP32 ? lq * 4 : (lq & 1) * 8;  // (16-bit types: both parts of h in one instruction, B twice)
                fb[c] = load_of_row<DT, WHOLE>(g.b, ((int64_t)tile.group * g.n + at.of_tile(c)) * g.r + j, (int64_t)g.count * g.n * g.r, j, g.r);
            }
        if (g.y) at.load(g.y + at_row * g.ld_y * SIZE, fy);
    }
    float factor = 1.f;
    v4f_l acc[4] = {};
    if (!none) {
        shrink_rows<DT, 1, 4, SHRINK_WAVES>(g, tile, 0, 1, 0, part, h);
        __syncthreads();
        stage_h<DT, ROWS, 64 * SHRINK_WAVES>(g, tile, h, 1, chunk == 0, kept, sums, row_most, factor, lm);
        const uint4 fh = *(const uint4*)(kept + lm * PITCH * SIZE + lq * 16);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] = mfma_16<DT>(fb[c], fh, acc[c]);
    }
    if (n0 < g.n && lm < tile.rows) at.store(g.out + at_row * g.n * SIZE, fy, acc, factor, !none);
}

// 64 rows and B through LDS, 16-bit types: the four waves have 16 rows each and the same columns, CB of them at a time, so that B is read once a workgroup.  The next
// CB columns of B and of y are on their way while these are multiplied.  The last of them are moved back to end with the last column (their first are
// then computed twice, the same): no access has an edge.  Measured: 8192 rows of eight adapters of rank 64, to 14336 columns: 138 us (3.4 TB/s of y and out; a copy in the same pieces 97 - 110,
// B out of the L2 16), of four of rank 16, to 4096 columns: 37 us.  y two steps ahead instead of one: the same, or 1 us more.  MOST: the largest expand_half.  TURNED: B is
// [count][r][n], the other matrix of an adapter as it lies: CB values of each of its rows go to LDS and are turned on the way out.
template <int DT, int MOST, int CB, bool WHOLE, bool ODD, bool TURNED>
__global__ __launch_bounds__(EXPAND_THREADS) void adapter_expand_tall_kernel(const AdapterArgs g, const AdapterTile* __restrict__ tiles) {
    constexpr int SIZE = 2, ROWS = 64, SUB = CB / 64, PIECES = ExpandCols<DT, false, ODD>::PIECES;
    constexpr int KP = CB * MOST / 8 / EXPAND_THREADS;  // pieces of 16 bytes of B that a lane brings
    constexpr int KH = MOST <= 64 ? (MOST + 31) / 32 : 0;  // of a rank of up to 64 the wave's h stays in registers
    extern __shared__ __align__(16) uint8_t expand_lds[];  // h [ROWS][pitch], then (fp16) fp32 [ROWS][half] while it is converted and B [2][CB][half + 8] from then on
    __shared__ uint32_t row_most[DT == F8MI_FP16 ? ROWS : 1];
    const int id = xcd_contiguous_id(blockIdx.x, gridDim.x), chunk = id % g.chunks;  // a tile's workgroups, and those of the next ones, on one XCD: B stays in its L2
    const AdapterTile tile = tiles[id / g.chunks];
    if (tile.rows == 0) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lm = lane & 15, lq = lane >> 4;
    const bool none = tile.group >= g.count;
    const int rp = g.rp, half = KH ? MOST : expand_half(rp), pitch = 2 * half + 8, b_pitch = TURNED ? CB + 32 : half + 8, row_pieces = TURNED ? CB / 8 : half / 8, pieces = CB / 8 * half;
    const int buffer_values = TURNED ? half * b_pitch : CB * b_pitch;
    uint8_t* const behind = expand_lds + ROWS * pitch * 2;
    uint16_t* const lds_b = (uint16_t*)behind;
    const int my_row = wave * 16 + lm;
    const int64_t at_row = g.table[AdapterTable(g.m, g.count).order() + tile.first + min(my_row, tile.rows - 1)];
    const uint8_t* y_row = g.y + at_row * g.ld_y * SIZE;
    uint8_t* out_row = g.out + at_row * g.n * SIZE;
    const int begin = chunk * g.cols, end = min(g.n, begin + g.cols), last = g.n - CB;
    const int64_t b_total = (int64_t)g.count * g.n * g.r;
    uint4 fb[KP], fy[SUB][PIECES] = {}, next_y[SUB][PIECES] = {};
    auto load_b = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const int item = i * EXPAND_THREADS + t, row = item / row_pieces, j = (item - row * row_pieces) * 8;
            if (item >= pieces) continue;
            if constexpr (TURNED) fb[i] = row < g.r ? load16_any(g.b + (((int64_t)tile.group * g.r + row) * g.n + n0 + j) * SIZE) : make_uint4(0u, 0u, 0u, 0u);
            else fb[i] = load_of_row<DT, WHOLE>(g.b, ((int64_t)tile.group * g.n + n0 + row) * g.r + j, b_total, j, g.r);
        }
    };
    auto keep_b = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const int item = i * EXPAND_THREADS + t, row = item / row_pieces, j = (item - row * row_pieces) * 8;
            if (item >= pieces) continue;
            uint4 q = fb[i];
            if (TURNED && (row >> 3 & 1)) q = make_uint4(q.z, q.w, q.x, q.y);  // (every second eight rows: 32 lanes read the first or the second half of 16 bytes of rows 0 .. 3, and the other of 8 .. 11)
            *(uint4*)(lds_b + buffer * buffer_values + row * b_pitch + j) = q;
        }
    };
    auto load_y = [&](int n0, uint4 (&q)[SUB][PIECES]) __attribute__((always_inline)) {
        if (g.y)
#pragma unroll
            for (int u = 0; u < SUB; u++) ExpandCols<DT, false, ODD>{n0 + u * 64, g.n, lq, lm}.load(y_row, q[u]);
    };
    load_y(min(begin, last), fy);
    float factor = 1.f;
    if (!none) {
        load_b(min(begin, last));
        stage_h<DT, ROWS>(g, tile, g.partial + (int64_t)tile.first * rp, g.splits, chunk == 0, expand_lds, (float*)behind, row_most, factor, my_row);
        keep_b(0);
        __syncthreads();
    }
    const uint16_t* hrow = (const uint16_t*)expand_lds + my_row * pitch;
    uint4 fh[KH ? KH : 1][2] = {};
    if (!none)
#pragma unroll
        for (int k = 0; k < KH; k++) {
            fh[k][0] = *(const uint4*)(hrow + k * 32 + lq * 8);
            if constexpr (MOST > 16) fh[k][1] = *(const uint4*)(hrow + half + k * 32 + lq * 8);
        }
    int buffer = 0;
    for (int n0 = begin; n0 < end; n0 += CB, buffer ^= 1) {
        const bool more = n0 + CB < end;  // the same for the workgroup
        if (more) {
            load_y(min(n0 + CB, last), next_y);
            if (!none) load_b(min(n0 + CB, last));
        }
#pragma unroll
        for (int u = 0; u < SUB; u++) {
            const ExpandCols<DT, false, ODD> at{min(n0, last) + u * 64, g.n, lq, lm};
            v4f_l acc[4] = {};
            if (!none) {
                const uint16_t* pb[4];
                if constexpr (!TURNED)
#pragma unroll
                    for (int c = 0; c < 4; c++) pb[c] = lds_b + buffer * buffer_values + (at.of_tile(c) - min(n0, last)) * b_pitch;
                auto read_b = [&](int c, int k) __attribute__((always_inline)) {  // eight of the rank from k on, k a multiple of 8, of column c of the lane
                    if constexpr (TURNED) {
                        const uint8_t* rows = (const uint8_t*)(lds_b + buffer * buffer_values + (k + (lm >> 2)) * b_pitch + u * 64 + c / 2 * 32 + (lm & 3) * 8) + ((c & 1) ^ (k >> 3 & 1)) * 8;
                        return read_turned(rows, rows + 4 * b_pitch * 2);
                    } else {
                        return *(const uint4*)(pb[c] + k);
                    }
                };
                if constexpr (MOST == 16) {  // a rank of up to 16: both parts of h in one instruction, B twice
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c] = mfma_16<DT>(read_b(c, (lq & 1) * 8), fh[0][0], acc[c]);
                } else if constexpr (KH > 0) {
#pragma unroll
                    for (int k = 0; k < KH; k++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const uint4 q = read_b(c, k * 32 + lq * 8);
                            acc[c] = mfma_16<DT>(q, fh[k][1], mfma_16<DT>(q, fh[k][0], acc[c]));
                        }
                } else {
#pragma unroll 1
                    for (int k = lq * 8; k < half; k += 32) {
                        const uint4 high = *(const uint4*)(hrow + k), low = *(const uint4*)(hrow + half + k);
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const uint4 q = read_b(c, k);
                            acc[c] = mfma_16<DT>(q, low, mfma_16<DT>(q, high, acc[c]));
                        }
                    }
                }
            }
            if (my_row < tile.rows) at.store(out_row, fy[u], acc, factor, !none);
        }
        if (more) {
            if (!none) {
                keep_b(buffer ^ 1);
                lds_barrier();
            }
#pragma unroll
            for (int u = 0; u < SUB; u++)
#pragma unroll
                for (int p = 0; p < PIECES; p++) fy[u][p] = next_y[u][p];
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

// The same for 16-bit types on their matrix instructions.  Both operands are wanted eight rows a lane and lie in LDS by rows: the reads turn them (ds_read_b64_tr_b16: of 4 rows x 16 columns
// each of 16 lanes gets a column).  small goes in as two bf16 values, high and low; fp16 values of big too, exactly, so that neither overflows or falls among the subnormals: bf16 has the
// exponents of fp32.  A row of 128 columns is 256 bytes; a pitch of 288 and rows 8 .. 15 of 16 turned by half a row let the 32 lanes that read at a time reach all banks.
// Measured: 8192 rows of 4096 bf16 columns, rank 16, 22 us out of HBM and 15.5 of what the memory-side cache has; with fp32 matrix instructions, which fp32 takes, 39.
// COLS_FIRST: sums [cols][r], so that a lane has four neighbours of the rank, else of the columns.
constexpr int OUTER_STEP = 64, OUTER_PITCH = 288;
__device__ __forceinline__ int outer_at(int row, int byte) { return row * OUTER_PITCH + (byte ^ ((row >> 3 & 1) * 128)); }
// rows row .. row + 7 of the lane's column of the 16 from `byte` on
__device__ __forceinline__ uint4 outer_read(const uint8_t* lds, int row, int byte, int lm) {
    return read_turned(lds + outer_at(row + (lm >> 2), byte + (lm & 3) * 8), lds + outer_at(row + 4 + (lm >> 2), byte + (lm & 3) * 8));
}
// two values as two bf16 each
__device__ __forceinline__ void split2(float a, float b, uint32_t& high, uint32_t& low) {
    high = pack_bf16x2(a, b);
    const float x = __uint_as_float(high << 16), y = __uint_as_float(high & 0xffff0000u);
    low = pack_bf16x2(x - x == 0.f ? a - x : 0.f, y - y == 0.f ? b - y : 0.f);  // (nothing is left of an infinity)
}
template <int DT, int RT, bool COLS_FIRST>
__global__ __launch_bounds__(OUTER_THREADS) void adapter_outer16_kernel(const OuterArgs g, const AdapterTile* __restrict__ chunks, int col_blocks) {
    constexpr int PARTS = DT == F8MI_FP16 ? 2 : 1;  // of big
    __shared__ __align__(16) uint8_t big[PARTS][OUTER_STEP * OUTER_PITCH], small[RT == 4 ? OUTER_STEP * OUTER_PITCH : OUTER_STEP * 64 * RT];
    // of a row of small the high parts (0) or the low ones: of up to 32 of the rank apart and without gaps, so that five workgroups fit a CU (of 8192 rows of 4096 columns all run at once: 21.4 us, of a pitch as big's has 22.2; fp16 four instead of two)
    auto small_at = [](int row, int part, int byte) __attribute__((always_inline)) {
        if constexpr (RT == 4) return outer_at(row, part * 128 + byte);
        return part * OUTER_STEP * 32 * RT + ((row * 32 * RT + byte) ^ ((row >> 3 & 1) * (RT == 1 ? 128 : 32)));
    };
    const int id = xcd_contiguous_id(blockIdx.x, gridDim.x);  // a chunk's workgroups on one XCD: small stays in its L2
    const AdapterTile chunk = chunks[id / col_blocks];
    if (chunk.rows == 0 || chunk.group >= g.count) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lm = lane & 15, lq = lane >> 4;
    const int c0 = min(id % col_blocks * OUTER_COLS, g.cols - OUTER_COLS), j0 = blockIdx.y * OUTER_RANK;  // (the last columns are moved back: some are computed twice, the same)
    const int32_t* order = g.table + AdapterTable(g.m, g.count).order() + chunk.first;
    const int my_row = t >> 4, my_col = (t & 15) * 8;
    int at_row[4];
    uint4 fb[4];
    float4 fs[RT];
    auto load_order = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) at_row[i] = order[min(r0 + my_row + 16 * i, chunk.rows - 1)];
    };
    auto load = [&](int r0) __attribute__((always_inline)) {  // of rows past the last: that one again, not kept
#pragma unroll
        for (int i = 0; i < 4; i++) fb[i] = load16_any(g.big + (at_row[i] * g.ld + c0 + my_col) * 2);
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int item = i * OUTER_THREADS + t, row = min(r0 + item / (RT * 4), chunk.rows - 1), j = min(j0 + item % (RT * 4) * 4, g.rp - 4);
            fs[i] = *(const float4*)(g.small + ((int64_t)chunk.first + row) * g.rp + j);
        }
    };
    auto keep = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = my_row + 16 * i, at = outer_at(row, my_col * 2);
            const uint4 q = r0 + row < chunk.rows ? fb[i] : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (DT == F8MI_BF16) {
                *(uint4*)(big[0] + at) = q;
            } else {
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
                uint32_t high[4], low[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x, y;
                    unpack2<F8MI_FP16>(w[e], x, y);
                    split2(x, y, high[e], low[e]);
                }
                *(uint4*)(big[0] + at) = make_uint4(high[0], high[1], high[2], high[3]);
                *(uint4*)(big[PARTS - 1] + at) = make_uint4(low[0], low[1], low[2], low[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int item = i * OUTER_THREADS + t, row = item / (RT * 4), j = item % (RT * 4) * 4;
            const bool in = r0 + row < chunk.rows && j0 + j < g.rp;
            uint32_t high[2], low[2];
            split2(in ? fs[i].x : 0.f, in ? fs[i].y : 0.f, high[0], low[0]);
            split2(in ? fs[i].z : 0.f, in ? fs[i].w : 0.f, high[1], low[1]);
            *(uint2*)(small + small_at(row, 0, j * 2)) = make_uint2(high[0], high[1]);
            *(uint2*)(small + small_at(row, 1, j * 2)) = make_uint2(low[0], low[1]);
        }
    };
    v4f_l acc[2][RT] = {};
    load_order(0);
    load(0);
    load_order(OUTER_STEP);
    for (int r0 = 0; r0 < chunk.rows; r0 += OUTER_STEP) {
        lds_barrier();  // (what was kept has been read)
        keep(r0);
        lds_barrier();
        if (r0 + OUTER_STEP < chunk.rows) {
            load(r0 + OUTER_STEP);
            load_order(r0 + 2 * OUTER_STEP);
        }
#pragma unroll
        for (int k = 0; k < OUTER_STEP; k += 32) {
            const int row = k + lq * 8;
            uint4 b[PARTS][2];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int p = 0; p < PARTS; p++) b[p][u] = outer_read(big[p], row, (wave * 32 + u * 16) * 2, lm);
#pragma unroll
            for (int j = 0; j < RT; j++) {
                auto read_small = [&](int part) __attribute__((always_inline)) {
                    return read_turned(small + small_at(row + (lm >> 2), part, j * 32 + (lm & 3) * 8), small + small_at(row + 4 + (lm >> 2), part, j * 32 + (lm & 3) * 8));
                };
                const uint4 high = read_small(0), low = read_small(1);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    auto add = [&](uint4 x, uint4 y) __attribute__((always_inline)) { acc[u][j] = COLS_FIRST ? mfma_16<F8MI_BF16>(y, x, acc[u][j]) : mfma_16<F8MI_BF16>(x, y, acc[u][j]); };
                    add(b[0][u], high);
                    add(b[0][u], low);
                    if constexpr (PARTS == 2) add(b[1][u], high);
                }
            }
        }
    }
    float* out = g.partial + (int64_t)(id / col_blocks) * g.cols * g.r;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < RT; j++) {
            const int col = c0 + wave * 32 + u * 16 + (COLS_FIRST ? lm : 4 * lq), rank = j0 + j * 16 + (COLS_FIRST ? 4 * lq : lm);
            if (rank >= g.r) continue;
            float* at = out + (COLS_FIRST ? (int64_t)col * g.r + rank : (int64_t)rank * g.cols + col);
            const v4f_l v = acc[u][j];
            if (!COLS_FIRST || rank + 4 <= g.r) store16_any(at, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (rank + e < g.r) at[e] = v[e];
        }
}

// The chunks of an adapter added up in their order; no chunk: zeros.  Both gradients in one launch.
struct OuterSums {
    const float* partial;
    int64_t size;  // of one adapter's gradient; 0: not asked for
    void* out;
};
__global__ __launch_bounds__(256) void adapter_outer_finish_kernel(const OuterSums first, const OuterSums second, int first_blocks, const int32_t* __restrict__ chunk_start, const float* __restrict__ scale,
                                                                   float factor, int dtype) {
    const bool in_first = (int)blockIdx.x < first_blocks;
    const OuterSums g{in_first ? first.partial : second.partial, in_first ? first.size : second.size, in_first ? first.out : second.out};
    const int64_t at = (int64_t)(blockIdx.x - (in_first ? 0 : first_blocks)) * 256 + threadIdx.x;
    const int e = blockIdx.y, begin = chunk_start[e], end = chunk_start[e + 1];
    if (at >= g.size) return;
    float s = 0.f;
#pragma unroll 8
    for (int i = begin; i < end; i++) s += g.partial[(int64_t)i * g.size + at];
    if (begin < end) s *= factor * (scale ? scale[e] : 1.f);
    const int64_t to = (int64_t)e * g.size + at;
    if (dtype == F8MI_FP32) ((float*)g.out)[to] = s;
    else if (dtype == F8MI_BF16) ((uint16_t*)g.out)[to] = (uint16_t)pack2<F8MI_BF16>(s, 0.f);
    else ((uint16_t*)g.out)[to] = (uint16_t)pack2<F8MI_FP16>(s, 0.f);
}

// The gradients of a batch without rows.  (Its table holds nothing, so that the kernel above has no chunks to look up.)
template <typename T>
__global__ __launch_bounds__(256) void adapter_zeros_kernel(T* __restrict__ first, int64_t first_size, T* __restrict__ second, int64_t second_size) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < first_size + second_size; i += (int64_t)gridDim.x * 256) {
        if (i < first_size) first[i] = 0;
        else second[i - first_size] = 0;
    }
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
    // Parts of a contraction that two workgroups a CU want
    int64_t wanted_splits() const { return std::max<int64_t>(1, 2 * (int64_t)cu_count() / std::max<int64_t>(1, tiles() * ((rp() + 63) / 64))); }
    int64_t row_bytes(int64_t contracted) const { return contracted * (dtype == F8MI_FP32 ? 4 : 2); }
    // Bytes of a row that a step of 64 rows takes: 512 where a rank of up to 16 leaves the registers and each part has two such steps, else 256
    int shrink_bytes(int64_t contracted) const { return rp() <= 16 && row_bytes(contracted) >= 2 * 512 * wanted_splits() ? 512 : 256; }
    // No more parts than steps (4099 tokens of 1000 fp16 values, 68 tiles: 11.5 us with one part, 7.0 with as many as there are steps); of short tiles two steps for each wave
    int64_t splits(int64_t contracted) const {
        const int64_t steps = tall() ? (row_bytes(contracted) + shrink_bytes(contracted) - 1) / shrink_bytes(contracted) : row_bytes(contracted) / (128 * SHRINK_WAVES) / 2;
        return std::max<int64_t>(1, std::min({wanted_splits(), steps, (int64_t)32}));
    }
    // Backward reads the adapters' matrices as they lie; short tiles and fp32 have their transposes made (4.6 us each for four adapters of 4096 x 16)
    bool turns_b() const { return tall() && dtype != F8MI_FP32; }
    bool turns_a() const { return turns_b() && rp() <= 128 && k >= expand_least((int)rp()); }  // (of a larger rank the rows of two blocks do not fit in LDS beside h)
    // Both products in one launch, where an adapter's rank and rows are few, its side of the contraction is short enough for each workgroup to read all of it and there is a workgroup a CU at most.
    // Eager calls are bound by the host, 9.3 us with two launches and a workspace, 5.2 - 7 with one.  On the GPU (us a call in a captured graph, two launches / one): one row 2048 -> 2048 of rank 8
    // 6.5 / 5.7, 4096 -> 4096 (128 KB) 6.7 / 7.3; 16 rows of 16 adapters 2048 -> 2048 8.1 / 7.0; 256 KB: one row 7.0 / 13; more workgroups: 64 rows of 64 adapters 1024 -> 4096 10.8 / 11.5.
    bool whole(int64_t contracted, int64_t columns) const {
        return !tall() && rp() <= 16 && 16 * row_bytes(contracted) <= (128 << 10) && (columns == 0 || columns >= 64) && tiles() * ((columns + WHOLE_COLS - 1) / WHOLE_COLS) <= cu_count();
    }
    int64_t partial_bytes(int64_t contracted, int64_t columns) const { return whole(contracted, columns) ? 0 : splits(contracted) * m * rp() * 4; }
};
static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// 16-bit rows that begin at odd multiples of two bytes
static bool odd_rows(const void* p, int64_t ld, int dtype) { return dtype != F8MI_FP32 && ((ld & 1) || ((uintptr_t)p & 2)); }
template <int DT, bool ODD, bool TURNED>
static int launch_shrink3(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    const AdapterTable table = s.table();
    const int rt = g.rp / 16;
    const dim3 grid((unsigned)(s.tiles() * g.splits), (unsigned)(rt <= 4 ? 1 : (rt + 3) / 4));
    if (s.tall()) {
        const AdapterTile* tiles = (const AdapterTile*)(g.table + table.tiles64());
        if (rt == 1 && s.shrink_bytes(g.k) == 512) hipLaunchKernelGGL((adapter_shrink_tall_kernel<DT, 1, 512, ODD, TURNED>), grid, dim3(TALL_THREADS), 0, stream, g, tiles);
        else if (rt == 1) hipLaunchKernelGGL((adapter_shrink_tall_kernel<DT, 1, 256, ODD, TURNED>), grid, dim3(TALL_THREADS), 0, stream, g, tiles);
        else if (rt == 2) hipLaunchKernelGGL((adapter_shrink_tall_kernel<DT, 2, 256, ODD, TURNED>), grid, dim3(TALL_THREADS), 0, stream, g, tiles);
        else hipLaunchKernelGGL((adapter_shrink_tall_kernel<DT, 4, 256, ODD, TURNED>), grid, dim3(TALL_THREADS), 0, stream, g, tiles);
    } else {
        const AdapterTile* tiles = (const AdapterTile*)(g.table + table.tiles16());
        if (rt == 1) hipLaunchKernelGGL((adapter_shrink_kernel<DT, 1>), grid, dim3(64 * SHRINK_WAVES), 0, stream, g, tiles);
        else if (rt == 2) hipLaunchKernelGGL((adapter_shrink_kernel<DT, 2>), grid, dim3(64 * SHRINK_WAVES), 0, stream, g, tiles);
        else hipLaunchKernelGGL((adapter_shrink_kernel<DT, 4>), grid, dim3(64 * SHRINK_WAVES), 0, stream, g, tiles);
    }
    return check_hip(hipGetLastError(), "adapter shrink kernel launch");
}
template <int DT>
static int launch_shrink2(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    if constexpr (DT != F8MI_FP32)
        if (odd_rows(g.x, g.ld, DT)) return g.a_turned ? launch_shrink3<DT, true, true>(g, s, stream) : launch_shrink3<DT, true, false>(g, s, stream);
    if constexpr (DT != F8MI_FP32)
        if (g.a_turned) return launch_shrink3<DT, false, true>(g, s, stream);
    return launch_shrink3<DT, false, false>(g, s, stream);
}
static int launch_shrink(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    if (s.dtype == F8MI_BF16) return launch_shrink2<F8MI_BF16>(g, s, stream);
    if (s.dtype == F8MI_FP16) return launch_shrink2<F8MI_FP16>(g, s, stream);
    return launch_shrink2<F8MI_FP32>(g, s, stream);
}

// Columns of out a workgroup: `per_cu` workgroups a CU in all, whole blocks of `block` columns
static int expand_cols(const AdapterArgs& g, int64_t n_tiles, int per_cu, int block) {
    const int64_t want = std::max<int64_t>(1, per_cu * (int64_t)cu_count() / n_tiles), blocks = std::max(1, (g.n + block - 1) / block);  // (one where h alone is asked for)
    return (int)((blocks + want - 1) / want * block);
}
// The same for 64 rows, of which four workgroups run on a CU at once: eight a CU or four, whichever takes less by an estimate in blocks of columns.  A workgroup costs its blocks and what h costs it
// (`before`: half a block for each block's bytes of parts, out of the L2, and one for the latency); a round that is less than a quarter full takes as long as a full one; a tenth of a workgroup is
// lost at the end.  (us of the kernel, eight / four: 2048 rows of rank 16 to 4096 columns 15.0 / 12.8, 4099 fp16 of rank 12 to 4097 31 / 27, 4096 of rank 64 to 4096 36 / 30; 8192 of rank 16 to 4096 36 / 37, to 8192
// 60.6 / 61.8, of rank 64 to 14336 140 / 147.)
static int expand_tall_cols(const AdapterArgs& g, int64_t n_tiles, int block) {
    auto cost = [&](int cols) {
        const double blocks = cols / block, before = 1.0 + 0.5 * g.splits * g.rp / block, slots = 4.0 * cu_count();
        const double rounds = std::max(1.0, (double)n_tiles * ((g.n + cols - 1) / cols) / slots), rest = rounds - (int64_t)rounds;
        return (rest > 0.0 && rest < 0.25 ? (int64_t)rounds + 1.0 : rounds) * (blocks + before) + 0.1 * blocks;
    };
    const int eight = expand_cols(g, n_tiles, 8, block), four = expand_cols(g, n_tiles, 4, block);
    return cost(four) < cost(eight) ? four : eight;
}
template <typename K>
static int launch_expand_kernel(K kernel, std::atomic<uint64_t>& allowed, AdapterArgs g, const AdapterTile* tiles, int64_t n_tiles, int lds, hipStream_t stream) {
    if (int rc = allow_big_lds(kernel, (160 << 10) - 1024, allowed)) return rc;
    g.chunks = std::max(1, (g.n + g.cols - 1) / g.cols);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(n_tiles * g.chunks)), dim3(EXPAND_THREADS), (unsigned)lds, stream, g, tiles);
    return check_hip(hipGetLastError(), "adapter expand kernel launch");
}
template <int DT, int WR, bool WHOLE, bool EDGE>
static int launch_expand_direct2(AdapterArgs g, const AdapterTile* tiles, int64_t n_tiles, hipStream_t stream) {
    static std::atomic<uint64_t> allowed{0};
    g.cols = expand_cols(g, n_tiles, 4, 256);
    return launch_expand_kernel(adapter_expand_kernel<DT, WR, WHOLE, EDGE>, allowed, g, tiles, n_tiles, 16 * WR * (expand_pitch<DT>(g.rp) * Ln<DT>::SIZE + (DT == F8MI_FP16 ? expand_half(g.rp) * 4 : 0)), stream);
}
template <int DT, int WR, bool WHOLE>
static int launch_expand_direct(const AdapterArgs& g, const AdapterTile* tiles, int64_t n_tiles, hipStream_t stream) {
    return g.n < 64 ? launch_expand_direct2<DT, WR, WHOLE, true>(g, tiles, n_tiles, stream) : launch_expand_direct2<DT, WR, WHOLE, false>(g, tiles, n_tiles, stream);
}
template <int DT, int MOST, int CB, bool WHOLE, bool ODD, bool TURNED>
static int launch_expand_tall2(AdapterArgs g, const AdapterTile* tiles, int64_t n_tiles, hipStream_t stream) {
    static std::atomic<uint64_t> allowed{0};
    g.cols = expand_tall_cols(g, n_tiles, CB);
    const int lds = 64 * expand_pitch<DT>(g.rp) * 2 + std::max(DT == F8MI_FP16 ? 64 * expand_half(g.rp) * 4 : 0, 2 * 2 * (TURNED ? expand_half(g.rp) * (CB + 32) : CB * (expand_half(g.rp) + 8)));
    return launch_expand_kernel(adapter_expand_tall_kernel<DT, MOST, CB, WHOLE, ODD, TURNED>, allowed, g, tiles, n_tiles, lds, stream);
}
template <int DT, int MOST, int CB, bool WHOLE>
static int launch_expand_tall(const AdapterArgs& g, const AdapterTile* tiles, int64_t n_tiles, hipStream_t stream) {
    const bool odd = odd_rows(g.out, g.n, DT) || (g.y && odd_rows(g.y, g.ld_y, DT));
    if constexpr (WHOLE && MOST <= 128)  // (turned, it is not asked)
        if (g.b_turned) return odd ? launch_expand_tall2<DT, MOST, CB, true, true, true>(g, tiles, n_tiles, stream) : launch_expand_tall2<DT, MOST, CB, true, false, true>(g, tiles, n_tiles, stream);
    return odd ? launch_expand_tall2<DT, MOST, CB, WHOLE, true, false>(g, tiles, n_tiles, stream) : launch_expand_tall2<DT, MOST, CB, WHOLE, false, false>(g, tiles, n_tiles, stream);
}
template <int DT, bool WHOLE>
static int launch_expand3(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    const AdapterTable table = s.table();
    const AdapterTile *short_tiles = (const AdapterTile*)(g.table + table.tiles16()), *tall_tiles = (const AdapterTile*)(g.table + table.tiles64());
    if (!s.tall()) return launch_expand_direct<DT, 1, WHOLE>(g, short_tiles, s.tiles(), stream);
    const int half = expand_half(g.rp);
    if (DT == F8MI_FP32 || g.n < expand_least(g.rp)) return launch_expand_direct<DT, 4, WHOLE>(g, tall_tiles, s.tiles(), stream);
    if constexpr (DT != F8MI_FP32) {
        if (half == 16) return launch_expand_tall<DT, 16, 128, WHOLE>(g, tall_tiles, s.tiles(), stream);
        if (half == 32) return launch_expand_tall<DT, 32, 128, WHOLE>(g, tall_tiles, s.tiles(), stream);
        if (half == 64) return launch_expand_tall<DT, 64, 64, WHOLE>(g, tall_tiles, s.tiles(), stream);
        if (half <= 128) return launch_expand_tall<DT, 128, 64, WHOLE>(g, tall_tiles, s.tiles(), stream);
        return launch_expand_tall<DT, 256, 64, WHOLE>(g, tall_tiles, s.tiles(), stream);
    }
    return F8MI_ERR_UNSUPPORTED;  // (not reached)
}
template <int DT>
static int launch_expand2(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    return g.b_turned || g.r % Ln<DT>::V == 0 ? launch_expand3<DT, true>(g, s, stream) : launch_expand3<DT, false>(g, s, stream);
}
static int launch_expand(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    if (s.dtype == F8MI_BF16) return launch_expand2<F8MI_BF16>(g, s, stream);
    if (s.dtype == F8MI_FP16) return launch_expand2<F8MI_FP16>(g, s, stream);
    return launch_expand2<F8MI_FP32>(g, s, stream);
}
template <int DT, bool WHOLE>
static int launch_whole2(AdapterArgs g, const AdapterShape& s, hipStream_t stream) {
    g.chunks = std::max(1, (g.n + WHOLE_COLS - 1) / WHOLE_COLS);
    hipLaunchKernelGGL((adapter_whole_kernel<DT, WHOLE>), dim3((unsigned)(s.tiles() * g.chunks)), dim3(64 * SHRINK_WAVES), 0, stream, g, (const AdapterTile*)(g.table + s.table().tiles16()));
    return check_hip(hipGetLastError(), "adapter kernel launch");
}
template <int DT>
static int launch_whole(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    return g.r % Ln<DT>::V == 0 ? launch_whole2<DT, true>(g, s, stream) : launch_whole2<DT, false>(g, s, stream);
}
// h and out
static int launch_products(const AdapterArgs& g, const AdapterShape& s, hipStream_t stream) {
    if (s.whole(g.k, g.n)) return s.dtype == F8MI_BF16 ? launch_whole<F8MI_BF16>(g, s, stream) : s.dtype == F8MI_FP16 ? launch_whole<F8MI_FP16>(g, s, stream) : launch_whole<F8MI_FP32>(g, s, stream);
    if (int rc = launch_shrink(g, s, stream)) return rc;
    return launch_expand(g, s, stream);
}
template <int DT, bool COLS_FIRST>
static void launch_outer16(const OuterArgs& g, const AdapterTile* chunks, int64_t n_chunks, hipStream_t stream) {
    const int blocks = (g.cols + OUTER_COLS - 1) / OUTER_COLS, rt = g.rp / 16;
    const dim3 grid((unsigned)(n_chunks * blocks), (unsigned)((g.rp + OUTER_RANK - 1) / OUTER_RANK));
    if (rt == 1) hipLaunchKernelGGL((adapter_outer16_kernel<DT, 1, COLS_FIRST>), grid, dim3(OUTER_THREADS), 0, stream, g, chunks, blocks);
    else if (rt == 2) hipLaunchKernelGGL((adapter_outer16_kernel<DT, 2, COLS_FIRST>), grid, dim3(OUTER_THREADS), 0, stream, g, chunks, blocks);
    else hipLaunchKernelGGL((adapter_outer16_kernel<DT, 4, COLS_FIRST>), grid, dim3(OUTER_THREADS), 0, stream, g, chunks, blocks);
}
template <int DT>
static void launch_outer2(const OuterArgs& g, const AdapterTile* chunks, int64_t n_chunks, hipStream_t stream) {
    if constexpr (DT != F8MI_FP32)
        if (g.cols >= OUTER_COLS) return g.cols_first ? launch_outer16<DT, true>(g, chunks, n_chunks, stream) : launch_outer16<DT, false>(g, chunks, n_chunks, stream);
    const dim3 grid((unsigned)n_chunks, (unsigned)((g.cols + OUTER_COLS - 1) / OUTER_COLS), (unsigned)((g.rp + OUTER_RANK - 1) / OUTER_RANK));
    hipLaunchKernelGGL(adapter_outer_kernel<DT>, grid, dim3(OUTER_THREADS), 0, stream, g, chunks);
}
static int launch_outer(const OuterArgs& g, int dtype, hipStream_t stream) {
    const AdapterTable table(g.m, g.count);
    const int64_t chunks = table.tiles(adapter_chunk_rows(g.m));
    const AdapterTile* list = (const AdapterTile*)(g.table + table.chunks());
    if (dtype == F8MI_BF16) launch_outer2<F8MI_BF16>(g, list, chunks, stream);
    else if (dtype == F8MI_FP16) launch_outer2<F8MI_FP16>(g, list, chunks, stream);
    else launch_outer2<F8MI_FP32>(g, list, chunks, stream);
    return check_hip(hipGetLastError(), "adapter gradient kernel launch");
}
static int launch_outer_finish(const AdapterShape& s, const OuterSums& da, const OuterSums& db, const int32_t* table, const float* scale, float factor, int out_dtype, hipStream_t stream) {
    const int64_t first = (da.size + 255) / 256, second = (db.size + 255) / 256;
    hipLaunchKernelGGL(adapter_outer_finish_kernel, dim3((unsigned)(first + second), (unsigned)s.count), dim3(256), 0, stream, da, db, (int)first, table + s.table().chunk_start(), scale, factor, out_dtype);
    return check_hip(hipGetLastError(), "adapter gradient sum kernel launch");
}

static int launch_zeros(void* da, int64_t da_size, void* db, int64_t db_size, int out_dtype, hipStream_t stream) {
    const dim3 grid((unsigned)std::min<int64_t>((da_size + db_size + 255) / 256, (int64_t)cu_count() * 8));
    if (out_dtype == F8MI_FP32) hipLaunchKernelGGL(adapter_zeros_kernel<uint32_t>, grid, dim3(256), 0, stream, (uint32_t*)da, da_size, (uint32_t*)db, db_size);
    else hipLaunchKernelGGL(adapter_zeros_kernel<uint16_t>, grid, dim3(256), 0, stream, (uint16_t*)da, da_size, (uint16_t*)db, db_size);
    return check_hip(hipGetLastError(), "adapter gradient zeros kernel launch");
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
    int64_t partial, dh, at, bt, sums_a, sums_b, bytes;
    AdapterBackwardSpace(const AdapterShape& s, bool need_dx, bool need_da, bool need_db) {
        const int64_t size = s.dtype == F8MI_FP32 ? 4 : 2, chunks = s.table().tiles(adapter_chunk_rows(s.m));
        const bool inner = need_dx || need_da;
        int64_t at_byte = 0;
        auto take = [&](int64_t n) { const int64_t o = at_byte; at_byte += up256(n); return o; };
        partial = take(inner ? s.partial_bytes(s.n, need_dx ? s.k : 0) : 0);
        dh = take(inner ? s.m * s.rp() * 4 : 0);
        bt = take(inner && !s.turns_b() ? s.count * s.n * s.r * size : 0);
        at = take(need_dx && !s.turns_a() ? s.count * s.k * s.r * size : 0);
        sums_a = take(need_da ? chunks * s.k * s.r * 4 : 0);
        sums_b = take(need_db ? chunks * s.n * s.r * 4 : 0);
        bytes = at_byte;
    }
};

}  // namespace f8mi

using namespace f8mi;

extern "C" int64_t f8mi_adapters_workspace_bytes(int64_t m, int64_t k, int64_t n, int64_t r, int64_t count, int dtype) {
    const AdapterShape s{m, k, n, r, count, dtype};
    return adapters_check("f8mi_adapters_workspace_bytes", s) || m == 0 ? 0 : s.partial_bytes(k, n);
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
    const int64_t need = s.partial_bytes(k, n);
    if ((need && !workspace) || workspace_bytes < need || (uintptr_t)workspace % 16 != 0 || (uintptr_t)table % 16 != 0 || (uintptr_t)h % 16 != 0) { set_error("f8mi_adapters: 16-byte aligned workspace of %lld bytes, table and h", (long long)need); return F8MI_ERR_INVALID_ARG; }
    const AdapterArgs g{(const uint8_t*)x, ldx, (const uint8_t*)a, (const int32_t*)table, (float*)workspace, m, (int)k, (int)r, (int)s.rp(), (int)count, (int)s.splits(k),
                        (const uint8_t*)b, scale, factor, (const uint8_t*)y, ldy, (uint8_t*)out, h, (int)n, 0, 0, false, false};
    return launch_products(g, s, stream);
}

extern "C" int f8mi_adapters_backward(const void* dout, int64_t ld_dout, const void* x, int64_t ldx, const void* a, const void* b, const float* scale, float factor, const void* table, const float* h, int64_t m,
                                      int64_t k, int64_t n, int64_t r, int64_t count, int dtype, void* dx, void* da, void* db, int p_dtype, void* workspace, int64_t workspace_bytes, void* stream_) {
    const AdapterShape s{m, k, n, r, count, dtype};
    hipStream_t stream = (hipStream_t)stream_;
    if (int rc = adapters_check("f8mi_adapters_backward", s)) return rc;
    if (!dx && !da && !db) return F8MI_OK;
    if (p_dtype < 0 || p_dtype > 2) { set_error("f8mi_adapters_backward: unknown dtype code %d", p_dtype); return F8MI_ERR_INVALID_ARG; }
    if (m == 0) return da || db ? launch_zeros(da, da ? count * r * k : 0, db, db ? count * n * r : 0, p_dtype, stream) : F8MI_OK;
    if (!dout || !table || bad_stride(ld_dout, n) || (da && (!x || bad_stride(ldx, k))) || (dx && !a) || ((dx || da) && !b) || (db && !h)) { set_error("f8mi_adapters_backward: null pointer or row stride"); return F8MI_ERR_INVALID_ARG; }
    const AdapterBackwardSpace space(s, dx, da, db);
    if (space.bytes && (!workspace || workspace_bytes < space.bytes || (uintptr_t)workspace % 256 != 0)) { set_error("f8mi_adapters_backward: 256-byte aligned workspace of %lld bytes needed", (long long)space.bytes); return F8MI_ERR_INVALID_ARG; }
    if ((uintptr_t)table % 16 != 0 || (uintptr_t)h % 16 != 0) { set_error("f8mi_adapters_backward: table and h are 16-byte aligned"); return F8MI_ERR_INVALID_ARG; }
    uint8_t* ws = (uint8_t*)workspace;
    float* dh = (float*)(ws + space.dh);
    if (dx || da) {
        if (!s.turns_b())
            if (int rc = launch_transpose(b, ws + space.bt, count, (int)n, (int)r, dtype, stream)) return rc;
        if (dx && !s.turns_a())
            if (int rc = launch_transpose(a, ws + space.at, count, (int)r, (int)k, dtype, stream)) return rc;
        const AdapterArgs g{(const uint8_t*)dout, ld_dout, s.turns_b() ? (const uint8_t*)b : ws + space.bt, (const int32_t*)table, (float*)(ws + space.partial), m, (int)n, (int)r, (int)s.rp(), (int)count, (int)s.splits(n),
                            !dx ? nullptr : s.turns_a() ? (const uint8_t*)a : ws + space.at, scale, factor, nullptr, 0, (uint8_t*)dx, dh, dx ? (int)k : 0, 0, 0, s.turns_b(), dx && s.turns_a()};
        if (int rc = launch_products(g, s, stream)) return rc;
    }
    float *sums_a = (float*)(ws + space.sums_a), *sums_b = (float*)(ws + space.sums_b);
    const OuterArgs o{nullptr, 0, nullptr, (const int32_t*)table, m, 0, (int)r, (int)s.rp(), (int)count, 0, nullptr};
    if (da) {
        OuterArgs q = o;
        q.big = (const uint8_t*)x; q.ld = ldx; q.small = dh; q.cols = (int)k; q.partial = sums_a;
        if (int rc = launch_outer(q, dtype, stream)) return rc;
    }
    if (db) {
        OuterArgs q = o;
        q.big = (const uint8_t*)dout; q.ld = ld_dout; q.small = h; q.cols = (int)n; q.cols_first = 1; q.partial = sums_b;
        if (int rc = launch_outer(q, dtype, stream)) return rc;
    }
    if (da || db) return launch_outer_finish(s, {sums_a, da ? k * r : 0, da}, {sums_b, db ? n * r : 0, db}, (const int32_t*)table, scale, factor, p_dtype, stream);
    return F8MI_OK;
}
