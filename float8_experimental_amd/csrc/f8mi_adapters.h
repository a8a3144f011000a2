// Low-rank adapters of many requests beside one projection: what the kernels share.
//
// Row i of the batch has the adapter e = ids[i] (or none, where ids[i] is no adapter's number): out_i = y_i + scale_e * B_e (A_e x_i), A_e [r][k], B_e [n][r].
// The products of an adapter are products of matrices once its rows are together: a table, made once for a batch and kept for all
// layers, lists the rows by adapter (those without one last) and cuts each adapter's rows into tiles of 16, of 64 and into chunks.
#pragma once
#include "f8mi_row.h"

namespace f8mi {

// Rows whose sums for the adapters' gradients one workgroup adds up: enough chunks to fill the chip, few enough that their partial gradients are small.
__host__ __device__ inline int64_t adapter_chunk_rows(int64_t m) {
    int64_t h = 64;
    while (h < 512 && h * 32 < m) h *= 2;
    return h;
}
struct AdapterTile {
    int32_t group, first, rows, none;  // rows first .. first + rows - 1 of the order; rows 0: nothing
};
// Where the parts of the table lie, in 32-bit words.  groups = adapters + 1 (the last: no adapter).
struct AdapterTable {
    int64_t m, groups;
    __host__ __device__ AdapterTable(int64_t m_, int64_t count) : m(m_), groups(count + 1) {}
    static __host__ __device__ int64_t up4(int64_t v) { return (v + 3) & ~(int64_t)3; }
    __host__ __device__ int64_t tiles(int64_t height) const { return m / height + (groups < m ? groups : m); }  // at most: one in each group is not full
    __host__ __device__ int64_t counts() const { return 0; }                        // [groups]
    __host__ __device__ int64_t chunk_start() const { return up4(groups); }         // [groups + 1]: of a group's chunks
    __host__ __device__ int64_t order() const { return chunk_start() + up4(groups + 1); }  // [m]
    __host__ __device__ int64_t tiles16() const { return order() + up4(m); }
    __host__ __device__ int64_t tiles64() const { return tiles16() + 4 * tiles(16); }
    __host__ __device__ int64_t chunks() const { return tiles64() + 4 * tiles(64); }
    __host__ __device__ int64_t words() const { return chunks() + 4 * tiles(adapter_chunk_rows(m)); }
};

}  // namespace f8mi
