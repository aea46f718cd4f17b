// Layer norm, its gradients, dropout, and the residual form of both, over rows of float32, float64, float16 or
// bfloat16.
//
//   forward   h = residual + dropout(x);  mean, var over the row;  y = (h - mean) * rstd * weight + bias
//   backward  xh = (h - mean) * rstd, g = dy * weight:
//             dh' = rstd * (g - mean(g) - xh * mean(g * xh)) + dh;  dx = dropout(dh');
//             dweight = sum over rows of dy * xh;  dbias = sum over rows of dy
//
// A row stays in the registers of its threads between its one read and its one write, so the variance is taken about
// the mean (two passes over registers, not over memory).  Sums, statistics and gradients are float32 (float64 for
// float64 rows); the rows' type is rounded to once, on the way out.  Sums run in a fixed order: results repeat bit for
// bit.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "norm.h"

namespace qb {

template <typename T> struct Accumulator { using type = float; };
template <> struct Accumulator<double> { using type = double; };

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T, typename A> __device__ __forceinline__ T narrow(A v) { return (T)v; }
template <> __device__ __forceinline__ __half narrow<__half, float>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16, float>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float reciprocal_root(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double reciprocal_root(double v) { return 1.0 / sqrt(v); }

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// Columns [c, c + V) of a row, those at or behind `end` left as zero.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* row, int c, int end) {
    Pack<T, V> p;
    if (c + V <= end) {
        p = *reinterpret_cast<const Pack<T, V>*>(row + c);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p.v[i] = c + i < end ? row[c + i] : narrow<T>((typename Accumulator<T>::type)0);
    }
    return p;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* row, int c, int end, const Pack<T, V>& p) {
    if (c + V <= end) {
        *reinterpret_cast<Pack<T, V>*>(row + c) = p;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < end) row[c + i] = p.v[i];
    }
}

template <typename T, typename A>
__device__ __forceinline__ A load_param(const void* params, bool f32, int c) {
    return f32 ? (A) static_cast<const float*>(params)[c] : (A)widen(static_cast<const T*>(params)[c]);
}

// Sums over the threads of a row, the same in every one of them: shuffles within a warp, shared memory across the
// warps of the row's group (a named barrier for each group, so groups do not wait for one another), distributed shared
// memory across the CTAs of a cluster.  Two buffers in turn, so each sum costs one barrier at each level.
template <typename A, int N> struct RowSum {
    struct Shared {
        A warps[2][NORM_MAX_THREADS / 32][N];
        A ranks[2][NORM_MAX_CLUSTER][N];
    };
    Shared& shared;
    const int threads_per_row;
    const int cluster;
    int turn = 0;
    __device__ RowSum(Shared& s, int t, int c) : shared(s), threads_per_row(t), cluster(c) {}

    __device__ __forceinline__ void operator()(A (&v)[N]) {
        const int span = threads_per_row < 32 ? threads_per_row : 32;
        for (int offset = span / 2; offset > 0; offset /= 2)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], offset);
        if (threads_per_row <= 32) return;
        const int warp = threadIdx.x / 32, warps = threads_per_row / 32, group = warp / warps, first = group * warps;
        if (threadIdx.x % 32 == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) shared.warps[turn][warp][n] = v[n];
        asm volatile("bar.sync %0, %1;" ::"r"(group), "r"(threads_per_row) : "memory");
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = shared.warps[turn][first][n];
        for (int w = 1; w < warps; ++w)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += shared.warps[turn][first + w][n];
        if (cluster > 1) {
            auto c = cooperative_groups::this_cluster();
            if ((int)threadIdx.x < cluster) {
                A* there = c.map_shared_rank(&shared.ranks[turn][c.block_rank()][0], threadIdx.x);
#pragma unroll
                for (int n = 0; n < N; ++n) there[n] = v[n];
            }
            c.sync();
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = shared.ranks[turn][0][n];
            for (int r = 1; r < cluster; ++r)
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] += shared.ranks[turn][r][n];
        }
        turn ^= 1;
    }
};

// Rows on their way in: every thread copies the packs that it will work on itself (cp.async into slots of its own), a
// few rows ahead of the one in work, so the copies need no barrier and their latency is hidden whatever the occupancy.
// Packs behind a row's end or the last row arrive as zeros.
template <typename T, int V, int ARRAYS, int STAGES> struct RowRing {
    static constexpr int E = norm_elements(sizeof(T)), K = E / V, BYTES = V * sizeof(T);
    Pack<T, V>* const slots;  // [STAGES][ARRAYS][K][blockDim.x]
    __device__ explicit RowRing(void* shared) : slots(static_cast<Pack<T, V>*>(shared) + threadIdx.x) {}
    __device__ __forceinline__ Pack<T, V>* at(int stage, int array, int k) const {
        return slots + ((stage * ARRAYS + array) * K + k) * blockDim.x;
    }
    // Columns [c, c + V) of `row`; `end` is the row's end, 0 for a row that is not there.
    __device__ __forceinline__ void fetch(int stage, int array, int k, const T* row, int c, int end) const {
        Pack<T, V>* slot = at(stage, array, k);
        const int bytes = c >= end ? 0 : c + V <= end ? BYTES : (end - c) * (int)sizeof(T);
        if constexpr (BYTES >= 4) {
            const unsigned to = (unsigned)__cvta_generic_to_shared(slot);
            const void* from = bytes > 0 ? static_cast<const void*>(row + c) : static_cast<const void*>(row);
            if constexpr (BYTES == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES < 4 ? 4 : BYTES), "r"(bytes) : "memory");
        } else {
            slot->v[0] = bytes > 0 ? row[c] : narrow<T>((typename Accumulator<T>::type)0);
        }
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // All but the youngest STAGES - 1 batches of copies have landed.
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
};

// RESIDUAL: x passes through dropout and may be added to a residual; otherwise h = x.
template <typename T, int V, bool RESIDUAL>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
norm_forward_kernel(const __grid_constant__ NormForwardArgs p, const RowShape shape) {
    using A = typename Accumulator<T>::type;
    using Ring = RowRing<T, V, RESIDUAL ? 2 : 1, norm_stages(sizeof(T), RESIDUAL ? 2 : 1)>;
    constexpr int E = Ring::E, K = Ring::K, STAGES = norm_stages(sizeof(T), RESIDUAL ? 2 : 1);
    __shared__ typename RowSum<A, 1>::Shared shared;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const Ring ring(dynamic);
    RowSum<A, 1> row_sum(shared, shape.threads_per_row, shape.cluster);
    const int t = threadIdx.x % shape.threads_per_row, group = threadIdx.x / shape.threads_per_row;
    const int rank = blockIdx.x % shape.cluster;
    const int begin = rank * shape.slice;
    const int end = begin + shape.slice < p.cols ? begin + shape.slice : p.cols;
    const int at = begin + t * V, hop = shape.threads_per_row * V;  // pack k: columns from at + k * hop on
    const long long step = (long long)(gridDim.x / shape.cluster) * shape.groups;
    long long row = (long long)(blockIdx.x / shape.cluster) * shape.groups + group, ahead = row;
    const T* const x = static_cast<const T*>(p.x.data);
    const T* const residual = static_cast<const T*>(p.residual.data);

    auto fetch = [&](int stage) {
        const bool there = ahead < p.rows;
        const T* from = there ? x + ahead * p.x.stride : x;
#pragma unroll
        for (int k = 0; k < K; ++k) ring.fetch(stage, 0, k, from, at + k * hop, there ? end : 0);
        if (RESIDUAL && residual != nullptr) {
            from = there ? residual + ahead * p.residual.stride : residual;
#pragma unroll
            for (int k = 0; k < K; ++k) ring.fetch(stage, RESIDUAL, k, from, at + k * hop, there ? end : 0);
        }
        ring.commit();
        ahead += step;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(s);

    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale;
    A weight[E], bias[E];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = at + k * hop + i;
            weight[k * V + i] = p.weight != nullptr && c < end ? load_param<T, A>(p.weight, p.params_f32, c) : (A)1;
            bias[k * V + i] = p.bias != nullptr && c < end ? load_param<T, A>(p.bias, p.params_f32, c) : (A)0;
        }

    // The groups of a CTA and the CTAs of a cluster make the same number of turns: `first` is that of group 0.
    int stage = 0;
    for (long long first = row - group; first < p.rows; first += step, row += step) {
        fetch(stage == 0 ? STAGES - 1 : stage - 1);  // into the slots that were read in the last turn
        ring.wait();
        const int limit = row < p.rows ? end : 0;
        A h[E];
        A sum[1] = {(A)0};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = at + k * hop;
            const Pack<T, V> raw = *ring.at(stage, 0, k);
#pragma unroll
            for (int i = 0; i < V; ++i) h[k * V + i] = widen(raw.v[i]);
            if (RESIDUAL) {
                if (p.draw.threshold != 0) {
                    bool keep[V];
                    draws.keep((unsigned long long)row * p.cols + c, keep);
#pragma unroll
                    for (int i = 0; i < V; ++i) h[k * V + i] = keep[i] ? h[k * V + i] * scale : (A)0;
                }
                if (residual != nullptr) {
                    const Pack<T, V> res = *ring.at(stage, RESIDUAL, k);
#pragma unroll
                    for (int i = 0; i < V; ++i) h[k * V + i] += widen(res.v[i]);
                }
                if (p.h.data != nullptr) {
                    Pack<T, V> out;
#pragma unroll
                    for (int i = 0; i < V; ++i) out.v[i] = narrow<T>(h[k * V + i]);
                    store_pack<T, V>(static_cast<T*>(p.h.data) + row * p.h.stride, c, limit, out);
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0] += h[k * V + i];
        }
        row_sum(sum);
        const A mean = sum[0] / (A)p.cols;
        A squares[1] = {(A)0};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A d = h[k * V + i] - mean;
                if (at + k * hop + i < end) squares[0] += d * d;
            }
        row_sum(squares);
        const A rstd = reciprocal_root(squares[0] / (A)p.cols + (A)p.epsilon);
        T* y = static_cast<T*>(p.y.data) + row * p.y.stride;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Pack<T, V> out;
#pragma unroll
            for (int i = 0; i < V; ++i)
                out.v[i] = narrow<T>((h[k * V + i] - mean) * rstd * weight[k * V + i] + bias[k * V + i]);
            store_pack<T, V>(y, at + k * hop, limit, out);
        }
        if (limit > 0 && t == 0 && rank == 0) {
            if (p.mean != nullptr) static_cast<A*>(p.mean)[row] = mean;
            if (p.rstd != nullptr) static_cast<A*>(p.rstd)[row] = rstd;
        }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
}

// A parameter's gradient in the parameters' type.
template <typename T, typename A>
__device__ __forceinline__ void store_gradient(void* out, bool f32, int c, A v) {
    if (f32) static_cast<float*>(out)[c] = (float)v;
    else static_cast<T*>(out)[c] = narrow<T>(v);
}

// RESIDUAL: dh is added to the row's gradient, which goes to dresidual, and through dropout's mask to dx.
// Threads keep their columns' share of dweight and dbias in registers over all rows of the CTA; at the end the CTA's
// groups are added up through shared memory, in order, and the CTA writes one row of partial sums (the gradients
// themselves where there is only one).
template <typename T, int V, bool RESIDUAL>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
norm_backward_kernel(const __grid_constant__ NormBackwardArgs p, const RowShape shape) {
    using A = typename Accumulator<T>::type;
    using Ring = RowRing<T, V, RESIDUAL ? 3 : 2, norm_stages(sizeof(T), RESIDUAL ? 3 : 2)>;
    constexpr int E = Ring::E, K = Ring::K, STAGES = norm_stages(sizeof(T), RESIDUAL ? 3 : 2);
    __shared__ typename RowSum<A, 2>::Shared shared;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const Ring ring(dynamic);
    RowSum<A, 2> row_sum(shared, shape.threads_per_row, shape.cluster);
    const int t = threadIdx.x % shape.threads_per_row, group = threadIdx.x / shape.threads_per_row;
    const int rank = blockIdx.x % shape.cluster;
    const int begin = rank * shape.slice;
    const int end = begin + shape.slice < p.cols ? begin + shape.slice : p.cols;
    const int at = begin + t * V, hop = shape.threads_per_row * V;
    const long long step = (long long)(gridDim.x / shape.cluster) * shape.groups;
    long long row = (long long)(blockIdx.x / shape.cluster) * shape.groups + group, ahead = row;
    const T* const dy = static_cast<const T*>(p.dy.data);
    const T* const h = static_cast<const T*>(p.h.data);
    const T* const dh = static_cast<const T*>(p.dh.data);

    auto fetch = [&](int stage) {
        const bool there = ahead < p.rows;
        const int limit = there ? end : 0;
        const long long r = there ? ahead : 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            ring.fetch(stage, 0, k, dy + r * p.dy.stride, at + k * hop, limit);
            ring.fetch(stage, 1, k, h + r * p.h.stride, at + k * hop, limit);
            if (RESIDUAL && dh != nullptr) ring.fetch(stage, 1 + RESIDUAL, k, dh + r * p.dh.stride, at + k * hop, limit);
        }
        ring.commit();
        ahead += step;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(s);

    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale;
    A weight[E], dweight[E], dbias[E];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = at + k * hop + i;
            weight[k * V + i] = p.weight != nullptr && c < end ? load_param<T, A>(p.weight, p.params_f32, c) : (A)1;
            dweight[k * V + i] = dbias[k * V + i] = (A)0;
        }

    A next_mean = row < p.rows ? static_cast<const A*>(p.mean)[row] : (A)0;
    A next_rstd = row < p.rows ? static_cast<const A*>(p.rstd)[row] : (A)0;
    int stage = 0;
    for (long long first = row - group; first < p.rows; first += step, row += step) {
        fetch(stage == 0 ? STAGES - 1 : stage - 1);
        const A mean = next_mean, rstd = next_rstd;
        if (row + step < p.rows) {
            next_mean = static_cast<const A*>(p.mean)[row + step];
            next_rstd = static_cast<const A*>(p.rstd)[row + step];
        }
        ring.wait();
        const int limit = row < p.rows ? end : 0;
        A sums[2] = {(A)0, (A)0};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Pack<T, V> dy_raw = *ring.at(stage, 0, k), h_raw = *ring.at(stage, 1, k);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A d = widen(dy_raw.v[i]), normal = (widen(h_raw.v[i]) - mean) * rstd;
                const A g = d * weight[k * V + i];
                dweight[k * V + i] += d * normal;
                dbias[k * V + i] += d;
                sums[0] += g;
                sums[1] += g * normal;
            }
        }
        row_sum(sums);
        const A along_one = sums[0] / (A)p.cols, along_normal = sums[1] / (A)p.cols;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = at + k * hop;
            const Pack<T, V> dy_raw = *ring.at(stage, 0, k), h_raw = *ring.at(stage, 1, k);
            A d[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A normal = (widen(h_raw.v[i]) - mean) * rstd;
                d[i] = rstd * (widen(dy_raw.v[i]) * weight[k * V + i] - along_one - normal * along_normal);
            }
            Pack<T, V> out;
            if (RESIDUAL) {
                if (dh != nullptr) {
                    const Pack<T, V> more = *ring.at(stage, 1 + RESIDUAL, k);
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] += widen(more.v[i]);
                }
                if (p.dresidual.data != nullptr) {
#pragma unroll
                    for (int i = 0; i < V; ++i) out.v[i] = narrow<T>(d[i]);
                    store_pack<T, V>(static_cast<T*>(p.dresidual.data) + row * p.dresidual.stride, c, limit, out);
                }
                if (p.draw.threshold != 0) {
                    bool keep[V];
                    draws.keep((unsigned long long)row * p.cols + c, keep);
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] = keep[i] ? d[i] * scale : (A)0;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) out.v[i] = narrow<T>(d[i]);
            store_pack<T, V>(static_cast<T*>(p.dx.data) + row * p.dx.stride, c, limit, out);
        }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }

    if (p.dweight == nullptr && p.dbias == nullptr) return;
    const bool whole = gridDim.x == (unsigned)shape.cluster;  // no other CTA has these columns
    A* const partial = static_cast<A*>(p.partial) + (long long)(blockIdx.x / shape.cluster) * 2 * p.cols;
    // Groups within a warp by shuffles, those of different warps (or warp groups) through shared memory, [team][2][width].
    for (int offset = 16; offset >= shape.threads_per_row; offset /= 2)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dweight[e] += __shfl_xor_sync(0xffffffffu, dweight[e], offset);
            dbias[e] += __shfl_xor_sync(0xffffffffu, dbias[e], offset);
        }
    const int width = shape.threads_per_row * E;
    const int teams = shape.threads_per_row < 32 ? (int)blockDim.x / 32 : shape.groups;
    const int team = shape.threads_per_row < 32 ? (int)threadIdx.x / 32 : group;
    A* const tile = reinterpret_cast<A*>(dynamic);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring is no longer read or written
    if (shape.threads_per_row >= 32 || (int)(threadIdx.x % 32) < shape.threads_per_row)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = (e / V) * hop + t * V + e % V;
            tile[team * 2 * width + c] = dweight[e];
            tile[team * 2 * width + width + c] = dbias[e];
        }
    __syncthreads();
    for (int c = threadIdx.x; c < end - begin; c += blockDim.x) {
        A w = tile[c], b = tile[width + c];
        for (int i = 1; i < teams; ++i) {
            w += tile[i * 2 * width + c];
            b += tile[i * 2 * width + width + c];
        }
        if (whole) {
            if (p.dweight != nullptr) store_gradient<T>(p.dweight, p.params_f32, begin + c, w);
            if (p.dbias != nullptr) store_gradient<T>(p.dbias, p.params_f32, begin + c, b);
        } else {
            partial[begin + c] = w;
            partial[p.cols + begin + c] = b;
        }
    }
}

// dweight and dbias from the partial rows: 32 columns of one of the two for each CTA, eight threads along the rows of
// each column, added in double in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) norm_join_kernel(const __grid_constant__ NormBackwardArgs p, int partials) {
    using A = typename Accumulator<T>::type;
    __shared__ double sums[8][33];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
    void* out = blockIdx.y == 0 ? p.dweight : p.dbias;
    if (out == nullptr) return;
    const A* partial = static_cast<const A*>(p.partial) + (long long)blockIdx.y * p.cols;
    double sum = 0.0;
    if (c < p.cols)
        for (int r = lane; r < partials; r += 8) sum += (double)partial[(long long)r * 2 * p.cols + c];
    sums[lane][threadIdx.x % 32] = sum;
    __syncthreads();
    if (lane != 0 || c >= p.cols) return;
#pragma unroll
    for (int r = 1; r < 8; ++r) sum += sums[r][threadIdx.x];
    store_gradient<T>(out, p.params_f32, c, (A)sum);
}

template <typename T, int V>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutArgs p, int threads_per_row) {
    using A = typename Accumulator<T>::type;
    const int t = threadIdx.x % threads_per_row, group = threadIdx.x / threads_per_row, groups = blockDim.x / threads_per_row;
    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale;
    for (long long row = (long long)blockIdx.y * groups + group; row < p.rows; row += (long long)gridDim.y * groups) {
        const T* x = static_cast<const T*>(p.x.data) + row * p.x.stride;
        T* y = static_cast<T*>(p.y.data) + row * p.y.stride;
        for (long long c = ((long long)blockIdx.x * threads_per_row + t) * V; c < p.cols; c += (long long)gridDim.x * threads_per_row * V) {
            const int end = p.cols - c < V ? (int)(p.cols - c) : V;
            Pack<T, V> v = load_pack<T, V>(x + c, 0, end);
            if (p.draw.threshold != 0) {
                bool keep[V];
                draws.keep((unsigned long long)row * p.cols + c, keep);
#pragma unroll
                for (int i = 0; i < V; ++i) v.v[i] = narrow<T>(keep[i] ? widen(v.v[i]) * scale : (A)0);
            }
            store_pack<T, V>(y + c, 0, end, v);
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------

// Whether rows start on 16-byte boundaries, so that a thread can take 16 bytes at a time.
inline bool rows_aligned(const RowArray& a, long long rows, size_t element) {
    return reinterpret_cast<uintptr_t>(a.data) % 16 == 0 && (rows <= 1 || a.stride * element % 16 == 0);
}

template <typename... P, typename... Q>
cudaError_t launch_rows(void (*kernel)(P...), unsigned grid, unsigned threads, size_t shared, int cluster, cudaStream_t stream, const Q&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

template <typename T>
cudaError_t norm_forward_launch(const NormForwardArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const RowShape s = row_shape(a.cols, norm_elements(sizeof(T)));
    const int threads = s.threads_per_row * s.groups;
    const long long batches = (a.rows + s.groups - 1) / s.groups;
    const long long resident = NORM_SMS * std::max(1, NORM_MAX_THREADS / threads) / s.cluster;
    const unsigned grid = (unsigned)((batches < resident ? batches : resident) * s.cluster);
    const bool wide = rows_aligned(a.x, a.rows, sizeof(T)) && rows_aligned(a.residual, a.rows, sizeof(T)) &&
                      rows_aligned(a.h, a.rows, sizeof(T)) && rows_aligned(a.y, a.rows, sizeof(T));
    const bool residual = a.residual.data != nullptr || a.h.data != nullptr || a.draw.threshold != 0;
    auto kernel = wide ? (residual ? norm_forward_kernel<T, V, true> : norm_forward_kernel<T, V, false>)
                       : (residual ? norm_forward_kernel<T, 1, true> : norm_forward_kernel<T, 1, false>);
    const size_t ring = norm_ring_bytes(sizeof(T), residual ? 2 : 1);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(ring * NORM_MAX_THREADS));
    return e != cudaSuccess ? e : launch_rows(kernel, grid, threads, ring * threads, s.cluster, stream, a, s);
}

template <typename T>
cudaError_t norm_backward_launch(const NormBackwardArgs& a, cudaStream_t stream) {
    using A = typename Accumulator<T>::type;
    constexpr int V = 16 / sizeof(T);
    const RowShape s = row_shape(a.cols, norm_elements(sizeof(T)));
    const int threads = s.threads_per_row * s.groups;
    const int partials = norm_partials(a.rows, s);
    const unsigned grid = (unsigned)partials * s.cluster;
    const bool wide = rows_aligned(a.dy, a.rows, sizeof(T)) && rows_aligned(a.dh, a.rows, sizeof(T)) &&
                      rows_aligned(a.h, a.rows, sizeof(T)) && rows_aligned(a.dx, a.rows, sizeof(T)) &&
                      rows_aligned(a.dresidual, a.rows, sizeof(T));
    const bool residual = a.dh.data != nullptr || a.dresidual.data != nullptr || a.draw.threshold != 0;
    auto kernel = wide ? (residual ? norm_backward_kernel<T, V, true> : norm_backward_kernel<T, V, false>)
                       : (residual ? norm_backward_kernel<T, 1, true> : norm_backward_kernel<T, 1, false>);
    // The ring's space later holds the groups' shares of the parameters' gradients: two values for each element.
    const size_t each = std::max(norm_ring_bytes(sizeof(T), residual ? 3 : 2), 2 * norm_elements(sizeof(T)) * sizeof(A));
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(each * NORM_MAX_THREADS));
    if (e == cudaSuccess) e = launch_rows(kernel, grid, threads, each * threads, s.cluster, stream, a, s);
    if (e != cudaSuccess || partials == 1 || (a.dweight == nullptr && a.dbias == nullptr)) return e;
    norm_join_kernel<T><<<dim3((a.cols + 31) / 32, 2), 256, 0, stream>>>(a, partials);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dropout_launch(const DropoutArgs& given, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    DropoutArgs a = given;
    if (a.x.stride == a.cols && a.y.stride == a.cols) {  // rows that follow on each other are one long row
        a.cols *= a.rows;
        a.rows = 1;
    }
    const bool wide = rows_aligned(a.x, a.rows, sizeof(T)) && rows_aligned(a.y, a.rows, sizeof(T));
    const long long packs = wide ? (a.cols + V - 1) / V : a.cols;
    int threads_per_row = 1;
    while (threads_per_row < packs && threads_per_row < 256) threads_per_row *= 2;
    const int groups = 256 / threads_per_row;
    const long long resident = NORM_SMS * 8;
    const long long across = (packs + threads_per_row - 1) / threads_per_row, down = (a.rows + groups - 1) / groups;
    const long long gx = across < resident ? across : resident;
    const long long most = (resident + gx - 1) / gx, gy = down < most ? down : most;
    const dim3 grid((unsigned)gx, (unsigned)gy);
    if (wide) dropout_kernel<T, V><<<grid, 256, 0, stream>>>(a, threads_per_row);
    else dropout_kernel<T, 1><<<grid, 256, 0, stream>>>(a, threads_per_row);
    return cudaGetLastError();
}

#define QB_INSTANTIATE_NORM(T)                                                              \
    template cudaError_t norm_forward_launch<T>(const NormForwardArgs&, cudaStream_t);      \
    template cudaError_t norm_backward_launch<T>(const NormBackwardArgs&, cudaStream_t);    \
    template cudaError_t dropout_launch<T>(const DropoutArgs&, cudaStream_t);

}  // namespace qb
