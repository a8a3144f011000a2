// The table of a batch's rows by adapter (f8mi_adapters.h): a stable counting sort in two launches, a workgroup an adapter.  It runs once for a batch,
// whose layers all use the table; the ids come out of the L2 after the first workgroup.
#include <algorithm>

#include "f8mi_adapters.h"

namespace f8mi {

constexpr int ROWS_THREADS = 1024;  // (8192 rows, both launches: 17 us, where 256 threads take 19; 64 rows 9, all latency)

// the group of a row: any number that is no adapter's means none
template <typename ID>
__device__ __forceinline__ int group_of(const ID* ids, int64_t i, int count) {
    const int64_t e = ids[i];
    return e >= 0 && e < count ? (int)e : count;
}

template <typename ID>
__global__ __launch_bounds__(ROWS_THREADS) void adapter_count_kernel(const ID* __restrict__ ids, int64_t m, int count, int32_t* __restrict__ counts) {
    __shared__ int part[ROWS_THREADS / 64];
    int n = 0;
    for (int64_t i = threadIdx.x; i < m; i += ROWS_THREADS) n += group_of(ids, i, count) == (int)blockIdx.x;
    for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < ROWS_THREADS / 64; w++) n += part[w];
        counts[blockIdx.x] = n;
    }
}

__device__ __forceinline__ int block_sum(int v, int* part) {  // over the workgroup, in every lane
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < ROWS_THREADS / 64; w++) v += part[w];
    return v;
}

template <typename ID>
__global__ __launch_bounds__(ROWS_THREADS) void adapter_place_kernel(const ID* __restrict__ ids, int64_t m, int count, int32_t* __restrict__ words) {
    __shared__ int part[ROWS_THREADS / 64];
    const AdapterTable table(m, count);
    const int g = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int32_t* counts = words + table.counts();
    const int heights[3] = {16, 64, (int)adapter_chunk_rows(m)};
    const int64_t at[3] = {table.tiles16(), table.tiles64(), table.chunks()};
    int before = 0, tiles[3] = {0, 0, 0};
    for (int i = t; i < g; i += ROWS_THREADS) {
        const int c = counts[i];
        before += c;
        for (int h = 0; h < 3; h++) tiles[h] += (c + heights[h] - 1) / heights[h];
    }
    before = block_sum(before, part);
    for (int h = 0; h < 3; h++) tiles[h] = block_sum(tiles[h], part);
    const int mine = counts[g];
    for (int h = 0; h < 3; h++) {
        AdapterTile* list = (AdapterTile*)(words + at[h]);
        const int n = (mine + heights[h] - 1) / heights[h];
        for (int i = t; i < n; i += ROWS_THREADS) list[tiles[h] + i] = {g, before + i * heights[h], min(heights[h], mine - i * heights[h]), 0};
        if (g == count)
            for (int64_t i = tiles[h] + n + t; i < table.tiles(heights[h]); i += ROWS_THREADS) list[i] = {0, 0, 0, 0};
    }
    if (t == 0) {
        int32_t* start = words + table.chunk_start();
        start[g] = tiles[2];
        if (g == count) start[g + 1] = tiles[2] + (mine + heights[2] - 1) / heights[2];
    }
    // the rows of the group, in the order of the batch
    int32_t* order = words + table.order();
    for (int64_t i0 = 0; i0 < m; i0 += ROWS_THREADS) {
        const int64_t i = i0 + t;
        const bool in = i < m && group_of(ids, i, count) == g;
        const uint64_t votes = __ballot(in);
        __syncthreads();
        if (lane == 0) part[wave] = __popcll(votes);
        __syncthreads();
        int rank = before + __popcll(votes & ((1ull << lane) - 1));
        for (int w = 0; w < ROWS_THREADS / 64; w++) {
            if (w < wave) rank += part[w];
            before += part[w];
        }
        if (in) order[rank] = (int32_t)i;
    }
}

template <typename ID>
static int launch_adapter_rows(const void* ids, int64_t m, int count, int32_t* words, hipStream_t stream) {
    hipLaunchKernelGGL(adapter_count_kernel<ID>, dim3((unsigned)count + 1), dim3(ROWS_THREADS), 0, stream, (const ID*)ids, m, count, words + AdapterTable(m, count).counts());
    if (int rc = check_hip(hipGetLastError(), "adapter rows count kernel launch")) return rc;
    hipLaunchKernelGGL(adapter_place_kernel<ID>, dim3((unsigned)count + 1), dim3(ROWS_THREADS), 0, stream, (const ID*)ids, m, count, words);
    return check_hip(hipGetLastError(), "adapter rows place kernel launch");
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int64_t f8mi_adapter_rows_words(int64_t m, int64_t count) { return m < 0 || count < 1 ? 0 : AdapterTable(m, count).words(); }

extern "C" int f8mi_adapter_rows(const void* ids, int id_bytes, int64_t m, int64_t count, void* table, void* stream) {
    if (m < 0 || count < 1 || (id_bytes != 4 && id_bytes != 8)) { set_error("f8mi_adapter_rows: bad m=%lld, count=%lld or ids of %d bytes", (long long)m, (long long)count, id_bytes); return F8MI_ERR_INVALID_ARG; }
    if (m > F8MI_ADAPTER_MAX_ROWS || count > F8MI_ADAPTER_MAX_COUNT) { set_error("f8mi_adapter_rows: at most %d rows and %d adapters", F8MI_ADAPTER_MAX_ROWS, F8MI_ADAPTER_MAX_COUNT); return F8MI_ERR_UNSUPPORTED; }
    if (m == 0) return F8MI_OK;
    if (!ids || !table || (uintptr_t)ids % id_bytes != 0 || (uintptr_t)table % 16 != 0) { set_error("f8mi_adapter_rows: null or unaligned pointer"); return F8MI_ERR_INVALID_ARG; }
    if (id_bytes == 4) return launch_adapter_rows<int32_t>(ids, m, (int)count, (int32_t*)table, (hipStream_t)stream);
    return launch_adapter_rows<int64_t>(ids, m, (int)count, (int32_t*)table, (hipStream_t)stream);
}
