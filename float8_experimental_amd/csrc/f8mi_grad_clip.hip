// The norm of a list of gradients as if they were one vector, and the gradients scaled to at most a given norm.
//
// HBM-bound: one read for the norm, one read and one write where something is scaled.  A launch takes up to GRADS tensors in its arguments
// (no table to build in device memory); their pieces of 32 KB are dealt to the workgroups as contiguous runs, so that a workgroup
// looks its first tensor up once and then walks on.  Sums are kept in 64 bits: squares of fp32 gradients neither overflow nor
// vanish, and the sum does not depend on how many values there are.  Every workgroup writes its part; every workgroup of the scaling launch
// adds all of them, in the same order, instead of a launch for it.  Where nothing is to be clipped, gradients that are scaled in place
// are left as they are: a factor of 1 changes no bit.
//
// Measured: the norm of 1.3e9 bf16 values that need no clipping 386 us (6.8 TB/s), 4.4e8 of them clipped into fp32 copies 594 us (131 for the norm at 6.7 TB/s,
// 461 for the copies at 5.7), in place 520 us, into copies of the same type 441, 48 small tensors 14 - 16 us (two launches).
#include <algorithm>

#include "f8mi_gemm_util.h"

namespace f8mi {

constexpr int GRADS = 96;             // tensors a launch
constexpr int GRAD_THREADS = 256, GRAD_UNROLL = 8;
constexpr int GRAD_PIECE = GRAD_THREADS * GRAD_UNROLL * 16;  // bytes of input
constexpr int GRAD_PARTS = 1024;      // workgroups of all launches for the norm, or as many as there are launches if that is more
// Workgroups of a launch that scales: one for each piece where it copies (4.4e8 bf16 values to fp32, us with 4096 / 8192 / 65536 of them: 640 / 625 /
// 595).  In place few, which are over sooner where there is nothing to clip; other numbers were not measured there.
constexpr int64_t GRAD_COPY_WGS = 65536, GRAD_IN_PLACE_WGS = 4096;

struct GradTable {
    const uint8_t* x[GRADS];
    uint8_t* out[GRADS];
    int64_t n[GRADS];
    int64_t end[GRADS];  // pieces of the tensors up to and with this one
    uint8_t dtype[GRADS], out_dtype[GRADS];
    int count;
};
static_assert(sizeof(GradTable) < 3600, "launch arguments are limited to 4 KB");

__host__ __device__ constexpr int64_t grad_piece(int dtype) { return GRAD_PIECE / (dtype == F8MI_FP32 ? 4 : 2); }

template <int DT>
struct GradVec {
    static constexpr int SIZE = DT == F8MI_FP32 ? 4 : 2, V = 16 / SIZE;
};
template <int DT>
__device__ __forceinline__ void grad_values(uint4 q, float (&v)[GradVec<DT>::V]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == F8MI_FP32) v[i] = __uint_as_float(w[i]);
        else unpack2<DT>(w[i], v[2 * i], v[2 * i + 1]);
    }
}
template <int DT>
__device__ __forceinline__ float grad_value(const uint8_t* x, int64_t i) {
    if constexpr (DT == F8MI_FP32) return ((const float*)x)[i];
    else if constexpr (DT == F8MI_BF16) return bf16_bits_to_float(((const uint16_t*)x)[i]);
    else return fp16_bits_to_float(((const uint16_t*)x)[i]);
}

// What a norm adds up: squares, magnitudes, or the largest magnitude (the fp32 bits, under which a NaN is larger than everything)
template <int KIND>
struct Norm {
    double sum = 0.0;
    uint32_t most = 0u;
    __device__ __forceinline__ void add(float v) {
        if constexpr (KIND == F8MI_NORM_2) sum = __builtin_fma((double)v, (double)v, sum);
        else if constexpr (KIND == F8MI_NORM_1) sum += (double)__builtin_fabsf(v);
        else most = max(most, __float_as_uint(v) & 0x7fffffffu);
    }
    __device__ __forceinline__ void add(const Norm& o) {
        sum += o.sum;
        most = max(most, o.most);
    }
    __device__ __forceinline__ double part() const { return KIND == F8MI_NORM_INF ? (double)__uint_as_float(most) : sum; }
    __device__ __forceinline__ void add_part(double p) {
        if constexpr (KIND == F8MI_NORM_INF) most = max(most, __float_as_uint((float)p) & 0x7fffffffu);
        else sum += p;
    }
    // over the workgroup, in every lane of the first wave
    __device__ __forceinline__ void all_lanes(double* slots) {
        double p = part();
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            Norm a;
            a.add_part(p);
            a.add_part(__shfl_xor(p, off, 64));
            p = a.part();
        }
        if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = p;
        __syncthreads();
        sum = 0.0;
        most = 0u;
#pragma unroll
        for (int w = 0; w < GRAD_THREADS / 64; w++) add_part(slots[w]);
    }
};

template <int KIND, int DT>
__device__ __forceinline__ void grad_norm_piece(const uint8_t* x, int64_t first, int64_t n, Norm<KIND>& total) {
    constexpr int V = GradVec<DT>::V, SIZE = GradVec<DT>::SIZE;
    float v[V];
    if (first + grad_piece(DT) <= n) {
        uint4 q[GRAD_UNROLL];
        const uint8_t* p = x + first * SIZE + threadIdx.x * 16;
#pragma unroll
        for (int u = 0; u < GRAD_UNROLL; u++) q[u] = load_nt16_any(p + u * GRAD_THREADS * 16);
#pragma unroll
        for (int u = 0; u < GRAD_UNROLL; u++) {
            grad_values<DT>(q[u], v);
#pragma unroll
            for (int i = 0; i < V; i++) total.add(v[i]);
        }
        return;
    }
    for (int64_t at = first + threadIdx.x * V; at < n; at += GRAD_THREADS * V) {
        if (at + V <= n) {
            grad_values<DT>(load_nt16_any(x + at * SIZE), v);
#pragma unroll
            for (int i = 0; i < V; i++) total.add(v[i]);
        } else {
            for (int64_t i = at; i < n; i++) total.add(grad_value<DT>(x, i));
        }
    }
}

// f(tensor, first value) for the pieces of workgroup `wg` of `wgs`
template <typename F>
__device__ __forceinline__ void grad_walk(const GradTable& t, int wg, int wgs, F f) {
    const int64_t pieces = t.end[t.count - 1];
    int64_t piece = pieces * wg / wgs;
    const int64_t last = pieces * (wg + 1) / wgs;
    if (piece >= last) return;
    int lo = 0, hi = t.count - 1;  // the first tensor that ends past `piece`
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t.end[mid] > piece) hi = mid;
        else lo = mid + 1;
    }
    for (; piece < last; piece++) {
        while (t.end[lo] <= piece) lo++;
        f(lo, (piece - (lo ? t.end[lo - 1] : 0)) * grad_piece(t.dtype[lo]));
    }
}

template <int KIND>
__global__ __launch_bounds__(GRAD_THREADS) void grad_norm_kernel(const GradTable t, double* __restrict__ parts) {
    __shared__ double slots[GRAD_THREADS / 64];
    Norm<KIND> total;
    grad_walk(t, blockIdx.x, gridDim.x, [&](int i, int64_t first) {
        if (t.dtype[i] == F8MI_BF16) grad_norm_piece<KIND, F8MI_BF16>(t.x[i], first, t.n[i], total);
        else if (t.dtype[i] == F8MI_FP16) grad_norm_piece<KIND, F8MI_FP16>(t.x[i], first, t.n[i], total);
        else grad_norm_piece<KIND, F8MI_FP32>(t.x[i], first, t.n[i], total);
    });
    total.all_lanes(slots);
    if (threadIdx.x == 0) parts[blockIdx.x] = total.part();
}

// The norm, from all parts, in every lane
template <int KIND>
__device__ __forceinline__ float grad_norm_of(const double* parts, int n_parts, double* slots) {
    Norm<KIND> total;
    for (int i = threadIdx.x; i < n_parts; i += GRAD_THREADS) total.add_part(parts[i]);
    total.all_lanes(slots);
    return KIND == F8MI_NORM_2 ? (float)__builtin_sqrt(total.sum) : (float)total.part();
}

// v * factor rounded to fp32, which a conversion to fp16 behind it would otherwise be folded into (one rounding less, and no -0)
template <int OT>
__device__ __forceinline__ float scaled(float v, float factor) {
    float p = __fmul_rn(v, factor);
    if constexpr (OT == F8MI_FP16) asm volatile("" : "+v"(p));
    return p;
}

__device__ __forceinline__ void stream16(uint8_t* dst, float a, float b, float c, float d) {
    __builtin_nontemporal_store((u32x4){__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d)}, (u32x4_any*)dst);
}

template <int DT, int OT>
__device__ __forceinline__ void grad_scale_piece(const uint8_t* x, uint8_t* out, int64_t first, int64_t n, float factor) {
    constexpr int V = GradVec<DT>::V, SIZE = GradVec<DT>::SIZE, OSIZE = OT == F8MI_FP32 ? 4 : 2;
    auto store = [&](uint8_t* dst, const float (&v)[V]) __attribute__((always_inline)) {
        if constexpr (OT == F8MI_FP32) {
#pragma unroll
            for (int i = 0; i < V; i += 4) stream16(dst + i * 4, v[i] * factor, v[i + 1] * factor, v[i + 2] * factor, v[i + 3] * factor);
        } else {
            uint32_t w[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; i++) w[i] = pack2<OT>(scaled<OT>(v[2 * i], factor), scaled<OT>(v[2 * i + 1], factor));
            if constexpr (V == 8) __builtin_nontemporal_store((u32x4){w[0], w[1], w[2], w[3]}, (u32x4_any*)dst);
            else __builtin_nontemporal_store((u32x2){w[0], w[1]}, (u32x2_any*)dst);
        }
    };
    if (DT != F8MI_FP32 && OT == F8MI_FP32 && first + grad_piece(DT) <= n) {
        // four values a lane, 8 bytes in and 16 out: a lane's eight would leave as two stores of every other 16 bytes, which streamed
        // (not through the caches, which the gradients would push out of) took 1.5 times as long
        u32x2 q[2 * GRAD_UNROLL];
        const int64_t at = first + threadIdx.x * 4;
#pragma unroll
        for (int u = 0; u < 2 * GRAD_UNROLL; u++) q[u] = __builtin_nontemporal_load((const u32x2_any*)(x + (at + u * GRAD_THREADS * 4) * SIZE));
#pragma unroll
        for (int u = 0; u < 2 * GRAD_UNROLL; u++) {
            float v[4];
            unpack2<DT == F8MI_FP32 ? F8MI_BF16 : DT>(q[u].x, v[0], v[1]);
            unpack2<DT == F8MI_FP32 ? F8MI_BF16 : DT>(q[u].y, v[2], v[3]);
            stream16(out + (at + u * GRAD_THREADS * 4) * OSIZE, v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor);
        }
        return;
    }
    if (first + grad_piece(DT) <= n) {
        uint4 q[GRAD_UNROLL];
        const int64_t at = first + threadIdx.x * V;
#pragma unroll
        for (int u = 0; u < GRAD_UNROLL; u++) q[u] = load_nt16_any(x + (at + u * GRAD_THREADS * V) * SIZE);
#pragma unroll
        for (int u = 0; u < GRAD_UNROLL; u++) {
            float v[V];
            grad_values<DT>(q[u], v);
            store(out + (at + u * GRAD_THREADS * V) * OSIZE, v);
        }
        return;
    }
    for (int64_t at = first + threadIdx.x * V; at < n; at += GRAD_THREADS * V) {
        if (at + V <= n) {
            float v[V];
            grad_values<DT>(load_nt16_any(x + at * SIZE), v);
            store(out + at * OSIZE, v);
        } else {
            for (int64_t i = at; i < n; i++) {
                const float v = scaled<OT>(grad_value<DT>(x, i), factor);
                if constexpr (OT == F8MI_FP32) ((float*)out)[i] = v;
                else ((uint16_t*)out)[i] = (uint16_t)pack2<OT>(v, 0.f);
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ void grad_scale_any(const GradTable& t, int i, int64_t first, float factor) {
    if (t.out_dtype[i] == F8MI_FP32) grad_scale_piece<DT, F8MI_FP32>(t.x[i], t.out[i], first, t.n[i], factor);
    else if (t.out_dtype[i] == F8MI_BF16) grad_scale_piece<DT, F8MI_BF16>(t.x[i], t.out[i], first, t.n[i], factor);
    else grad_scale_piece<DT, F8MI_FP16>(t.x[i], t.out[i], first, t.n[i], factor);
}

// norm_out: written by the first workgroup (null in all launches but the first).  in_place: every tensor's `out` is its `x`.
template <int KIND>
__global__ __launch_bounds__(GRAD_THREADS) void grad_scale_kernel(const GradTable t, const double* __restrict__ parts, int n_parts, float max_norm, int in_place,
                                                                  float* __restrict__ norm_out) {
    __shared__ double slots[GRAD_THREADS / 64];
    const float norm = grad_norm_of<KIND>(parts, n_parts, slots);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float ratio = __fdiv_rn(max_norm, norm + 1e-6f);
    const float factor = ratio > 1.f ? 1.f : ratio;  // a NaN stays
    if (in_place && factor == 1.f) return;
    grad_walk(t, blockIdx.x, gridDim.x, [&](int i, int64_t first) {
        if (t.dtype[i] == F8MI_BF16) grad_scale_any<F8MI_BF16>(t, i, first, factor);
        else if (t.dtype[i] == F8MI_FP16) grad_scale_any<F8MI_FP16>(t, i, first, factor);
        else grad_scale_any<F8MI_FP32>(t, i, first, factor);
    });
}

template <int KIND>
__global__ __launch_bounds__(GRAD_THREADS) void grad_norm_finish_kernel(const double* __restrict__ parts, int n_parts, float* __restrict__ norm_out) {
    __shared__ double slots[GRAD_THREADS / 64];
    const float norm = grad_norm_of<KIND>(parts, n_parts, slots);
    if (threadIdx.x == 0) *norm_out = norm;
}

static int64_t grad_launches(int64_t count) { return std::max<int64_t>(1, (count + GRADS - 1) / GRADS); }
static int grad_parts_of_a_launch(int64_t count) { return (int)std::max<int64_t>(1, GRAD_PARTS / grad_launches(count)); }

template <int KIND>
static int launch_grads(const f8mi_grad* g, int64_t count, float max_norm, bool scale, float* norm_out, double* parts, hipStream_t stream) {
    GradTable t;
    const int most = grad_parts_of_a_launch(count);
    int n_parts = 0;
    const bool has_scale = scale;
    for (int pass = 0; pass < (has_scale ? 2 : 1); pass++) {
        int64_t at = 0;
        bool first_launch = true;
        while (at < count || (first_launch && pass == 1)) {
            t.count = 0;
            int64_t pieces = 0;
            int in_place = 1;
            for (; at < count && t.count < GRADS; at++) {
                if (g[at].n == 0) continue;
                const int c = t.count++;
                t.x[c] = (const uint8_t*)g[at].x;
                t.out[c] = (uint8_t*)g[at].out;
                t.n[c] = g[at].n;
                t.dtype[c] = (uint8_t)g[at].dtype;
                t.out_dtype[c] = (uint8_t)g[at].out_dtype;
                pieces += (g[at].n + grad_piece(g[at].dtype) - 1) / grad_piece(g[at].dtype);
                t.end[c] = pieces;
                in_place &= g[at].out == g[at].x;
            }
            if (t.count == 0) break;
            if (pass == 0) {
                const int wgs = (int)std::min<int64_t>(pieces, most);
                hipLaunchKernelGGL(grad_norm_kernel<KIND>, dim3((unsigned)wgs), dim3(GRAD_THREADS), 0, stream, t, parts + n_parts);
                n_parts += wgs;
            } else {
                const unsigned wgs = (unsigned)std::min<int64_t>(pieces, in_place ? GRAD_IN_PLACE_WGS : GRAD_COPY_WGS);
                hipLaunchKernelGGL(grad_scale_kernel<KIND>, dim3(wgs), dim3(GRAD_THREADS), 0, stream, t, parts, n_parts, max_norm, in_place, first_launch ? norm_out : nullptr);
            }
            first_launch = false;
        }
        if (pass == 1 && !first_launch) return check_hip(hipGetLastError(), "gradient clipping kernel launch");
    }
    hipLaunchKernelGGL(grad_norm_finish_kernel<KIND>, dim3(1), dim3(GRAD_THREADS), 0, stream, parts, n_parts, norm_out);
    return check_hip(hipGetLastError(), "gradient norm kernel launch");
}

}  // namespace f8mi

using namespace f8mi;

extern "C" int64_t f8mi_grad_clip_workspace_bytes(int64_t count) { return count < 0 ? 0 : grad_launches(count) * grad_parts_of_a_launch(count) * (int64_t)sizeof(double); }

extern "C" int f8mi_grad_clip(const f8mi_grad* grads, int64_t count, int norm_kind, float max_norm, int scale, float* norm_dev, void* workspace, int64_t workspace_bytes,
                              void* stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (count < 0 || (count > 0 && !grads)) { set_error("f8mi_grad_clip: no tensors at %p (count=%lld)", (const void*)grads, (long long)count); return F8MI_ERR_INVALID_ARG; }
    if (norm_kind != F8MI_NORM_2 && norm_kind != F8MI_NORM_1 && norm_kind != F8MI_NORM_INF) { set_error("f8mi_grad_clip: unknown norm %d", norm_kind); return F8MI_ERR_INVALID_ARG; }
    if (!norm_dev || !workspace || workspace_bytes < f8mi_grad_clip_workspace_bytes(count) || (uintptr_t)workspace % 8 != 0) { set_error("f8mi_grad_clip: no place for the norm, or a workspace of less than %lld bytes", (long long)f8mi_grad_clip_workspace_bytes(count)); return F8MI_ERR_INVALID_ARG; }
    for (int64_t i = 0; i < count; i++) {
        const f8mi_grad& g = grads[i];
        if (g.n < 0 || g.dtype < 0 || g.dtype > 2 || (g.n > 0 && !g.x)) { set_error("f8mi_grad_clip: tensor %lld: null pointer, size or dtype code", (long long)i); return F8MI_ERR_INVALID_ARG; }
        if (scale && g.n > 0 && (!g.out || g.out_dtype < 0 || g.out_dtype > 2 || (g.out == g.x && g.out_dtype != g.dtype))) { set_error("f8mi_grad_clip: tensor %lld: no place for the scaled values, or one of another type on top of them", (long long)i); return F8MI_ERR_INVALID_ARG; }
    }
    double* parts = (double*)workspace;
    if (norm_kind == F8MI_NORM_2) return launch_grads<F8MI_NORM_2>(grads, count, max_norm, scale != 0, norm_dev, parts, stream);
    if (norm_kind == F8MI_NORM_1) return launch_grads<F8MI_NORM_1>(grads, count, max_norm, scale != 0, norm_dev, parts, stream);
    return launch_grads<F8MI_NORM_INF>(grads, count, max_norm, scale != 0, norm_dev, parts, stream);
}
