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
#include <type_traits>

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
// Within 2 units in the last place (float32), 1 (float64); 0 for an infinite variance.
__device__ __forceinline__ float reciprocal_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double reciprocal_root(double v) { return 1.0 / sqrt(v); }

// Elements are worked on two at a time: float32 pairs are one instruction on this architecture, and the kernels would
// otherwise be bound by instruction issue while 16-bit rows stream by.
template <typename A> struct Two;
template <> struct Two<float> {
    float2 v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) : v(make_float2(a, b)) {}
    __device__ __forceinline__ explicit Two(float a) : v(make_float2(a, a)) {}
    __device__ __forceinline__ float sum() const { return v.x + v.y; }
};
template <> struct Two<double> {
    double2 v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(double a, double b) : v(make_double2(a, b)) {}
    __device__ __forceinline__ explicit Two(double a) : v(make_double2(a, a)) {}
    __device__ __forceinline__ double sum() const { return v.x + v.y; }
};
__device__ __forceinline__ Two<float> operator+(Two<float> a, Two<float> b) { a.v = __fadd2_rn(a.v, b.v); return a; }
__device__ __forceinline__ Two<float> operator*(Two<float> a, Two<float> b) { a.v = __fmul2_rn(a.v, b.v); return a; }
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) { a.v = __ffma2_rn(a.v, b.v, c.v); return a; }
__device__ __forceinline__ Two<double> operator+(Two<double> a, Two<double> b) { return {a.v.x + b.v.x, a.v.y + b.v.y}; }
__device__ __forceinline__ Two<double> operator*(Two<double> a, Two<double> b) { return {a.v.x * b.v.x, a.v.y * b.v.y}; }
__device__ __forceinline__ Two<double> fma(Two<double> a, Two<double> b, Two<double> c) { return {::fma(a.v.x, b.v.x, c.v.x), ::fma(a.v.y, b.v.y, c.v.y)}; }

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// A thread's packs of a row as pairs of accumulation-type values: pair q holds elements 2 q and 2 q + 1 of the packs
// put one behind the other (of the same pack, or of two packs of one element).
template <typename T, typename A>
__device__ __forceinline__ T narrow_of(const Two<A>& p, int i) { return narrow<T>(i == 0 ? p.v.x : p.v.y); }

template <typename T, int V, typename A>
__device__ __forceinline__ void widen_pack(const Pack<T, V>& raw, Two<A>* pairs, int k) {
    if constexpr (V == 1) {
        (k % 2 == 0 ? pairs[k / 2].v.x : pairs[k / 2].v.y) = widen(raw.v[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            Two<A>& p = pairs[(k * V + i) / 2];
            if constexpr (std::is_same<T, __half>::value) {
                p.v = __half22float2(*reinterpret_cast<const __half2*>(&raw.v[i]));
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // a bfloat16 is the upper half of a float32
                const unsigned both = *reinterpret_cast<const unsigned*>(&raw.v[i]);
                p.v.x = __uint_as_float(both << 16);
                p.v.y = __uint_as_float(both & 0xffff0000u);
            } else {
                p.v.x = raw.v[i];
                p.v.y = raw.v[i + 1];
            }
        }
    }
}

template <typename T, int V, typename A>
__device__ __forceinline__ Pack<T, V> narrow_pack(const Two<A>* pairs, int k) {
    Pack<T, V> out;
    if constexpr (V == 1) {
        out.v[0] = narrow_of<T>(pairs[k / 2], k % 2);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const Two<A>& p = pairs[(k * V + i) / 2];
            if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(&out.v[i]) = __float22half2_rn(p.v);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(&out.v[i]) = __float22bfloat162_rn(p.v);
            else out.v[i] = narrow<T>(p.v.x), out.v[i + 1] = narrow<T>(p.v.y);
        }
    }
    return out;
}

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
        A warps[2][2][NORM_MAX_THREADS / 32];
        A ranks[2][NORM_MAX_CLUSTER][N];
    };
    Shared& shared;
    const int threads_per_row;
    const int cluster;
    int turn = 0;
    __device__ RowSum(Shared& s, int t, int c) : shared(s), threads_per_row(t), cluster(c) {}

    // Over the lanes of one row in a warp; every lane has the sums.
    __device__ __forceinline__ void across(A (&v)[N]) const {
        for (int offset = threads_per_row / 2; offset > 0; offset /= 2)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], offset);
    }

    __device__ __forceinline__ void operator()(A (&v)[N]) {
        if (threads_per_row < 32) return across(v);
        // Over the warp.  Of two sums, one half of the lanes goes on with the first and the other with the second.
        const int lane = threadIdx.x % 32;
        A part = v[0];
        if (N == 2) {
            const A send = lane < 16 ? v[N - 1] : v[0];
            part = (lane < 16 ? v[0] : v[N - 1]) + __shfl_xor_sync(0xffffffffu, send, 16);
        } else {
            part += __shfl_xor_sync(0xffffffffu, part, 16);
        }
#pragma unroll
        for (int offset = 8; offset > 0; offset /= 2) part += __shfl_xor_sync(0xffffffffu, part, offset);
        if (threads_per_row > 32) {
            // Over the (at most 16) warps of the row: lane l adds up from warp l % 16 on.
            const int warp = threadIdx.x / 32, warps = threads_per_row / 32, group = warp / warps, first = group * warps;
            if (lane % 16 == 0) shared.warps[turn][lane / 16][warp] = part;
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads_per_row) : "memory");  // 0 is the whole CTA's
            part = lane % 16 < warps ? shared.warps[turn][lane / 16][first + lane % 16] : (A)0;
#pragma unroll
            for (int offset = 8; offset > 0; offset /= 2) part += __shfl_xor_sync(0xffffffffu, part, offset);
        }
        v[0] = N == 2 ? __shfl_sync(0xffffffffu, part, 0) : part;
        if (N == 2) v[N - 1] = __shfl_sync(0xffffffffu, part, 16);
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
// Slot s of neighbouring threads lie next to each other: one warp's copy is one run of shared memory (with a thread's
// slots together instead, the same kernels took 10 to 35 % longer).
template <typename T, int V, int ARRAYS, int STAGES> struct RowRing {
    static constexpr int E = norm_elements(sizeof(T)), K = E / V, BYTES = V * sizeof(T);
    char* const slots;   // [STAGES][ARRAYS][K][threads]
    const int pitch;     // bytes from one slot of a thread to its next
    __device__ explicit RowRing(void* shared)
        : slots(static_cast<char*>(shared) + threadIdx.x * BYTES), pitch((int)blockDim.x * BYTES) {}
    __device__ __forceinline__ Pack<T, V>* at(int stage, int array, int k) const {
        return reinterpret_cast<Pack<T, V>*>(slots + (stage * (ARRAYS * K) + array * K + k) * pitch);
    }
    // `count` elements at `from`: a whole pack, less at a row's end, none for a row that is not there.
    __device__ __forceinline__ void fetch(int stage, int array, int k, const T* from, int count) const {
        Pack<T, V>* slot = at(stage, array, k);
        if constexpr (BYTES >= 4) {
            const unsigned to = (unsigned)__cvta_generic_to_shared(slot);
            const int bytes = count * (int)sizeof(T);
            if constexpr (BYTES == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES < 4 ? 4 : BYTES), "r"(bytes) : "memory");
        } else {
            slot->v[0] = count > 0 ? *from : narrow<T>((typename Accumulator<T>::type)0);
        }
    }
    // A thread's packs of a row as pairs.
    template <typename A> __device__ __forceinline__ void read(int stage, int array, Two<A> (&pairs)[E / 2]) const {
#pragma unroll
        for (int k = 0; k < K; ++k) widen_pack<T, V>(*at(stage, array, k), pairs, k);
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // All but the youngest STAGES - 1 batches of copies have landed.
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
};

// A kernel's place in the rows: which columns a thread holds, and which row its group is at.
template <typename T, int V> struct Place {
    static constexpr int E = norm_elements(sizeof(T)), K = E / V;
    int t, group, rank, begin, end, at, hop;
    long long step, row;
    __device__ __forceinline__ Place(const RowShape& shape, int cols) {
        t = threadIdx.x % shape.threads_per_row;
        group = threadIdx.x / shape.threads_per_row;
        rank = blockIdx.x % shape.cluster;
        begin = rank * shape.slice;
        end = begin + shape.slice < cols ? begin + shape.slice : cols;
        at = begin + t * V;  // pack k: columns from at + k * hop on
        hop = shape.threads_per_row * V;
        step = (long long)(gridDim.x / shape.cluster) * shape.groups;
        row = (long long)(blockIdx.x / shape.cluster) * shape.groups + group;
    }
    // Elements of pack k that are in the row.
    __device__ __forceinline__ int count(int k) const {
        const int left = end - at - k * hop;
        return left >= V ? V : left > 0 ? left : 0;
    }
    __device__ __forceinline__ bool whole() const { return at + (K - 1) * hop + V <= end; }
    __device__ __forceinline__ void store(T* row_at, int k, const Pack<T, V>& pack, bool all) const {
        if (all) *reinterpret_cast<Pack<T, V>*>(row_at + k * hop) = pack;
        else store_pack<T, V>(row_at + k * hop, 0, count(k), pack);
    }
};

// Adds scale or 0 by the elements' draws: pairs of pack k, whose first element has row-major number `index`.
template <int V, typename A>
__device__ __forceinline__ void drop(const DrawStream& draws, unsigned long long index, A scale, Two<A>* pairs, int k) {
    bool keep[V];
    draws.keep(index, keep);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        A& v = (k * V + i) % 2 == 0 ? pairs[(k * V + i) / 2].v.x : pairs[(k * V + i) / 2].v.y;
        v = keep[i] ? v * scale : (A)0;
    }
}

// RESIDUAL: x passes through dropout and may be added to a residual; otherwise h = x.
template <typename T, int V, bool RESIDUAL>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
norm_forward_kernel(const __grid_constant__ NormForwardArgs p, const RowShape shape) {
    using A = typename Accumulator<T>::type;
    constexpr int ARRAYS = RESIDUAL ? 2 : 1, STAGES = norm_stages(sizeof(T), ARRAYS);
    using Ring = RowRing<T, V, ARRAYS, STAGES>;
    constexpr int E = Ring::E, K = Ring::K;
    __shared__ typename RowSum<A, 1>::Shared shared;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const Ring ring(dynamic);
    RowSum<A, 1> row_sum(shared, shape.threads_per_row, shape.cluster);
    const Place<T, V> place(shape, p.cols);
    const bool whole = place.whole();
    long long row = place.row, ahead = place.row;
    const bool added = RESIDUAL && p.residual.data != nullptr;
    const T* x = static_cast<const T*>(p.x.data) + row * p.x.stride + place.at;
    const T* residual = static_cast<const T*>(p.residual.data) + row * p.residual.stride + place.at;
    T* h_out = static_cast<T*>(p.h.data) + row * p.h.stride + place.at;
    T* y = static_cast<T*>(p.y.data) + row * p.y.stride + place.at;

    auto fetch = [&](int stage) {
        const bool there = ahead < p.rows;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int count = there ? (whole ? V : place.count(k)) : 0;
            ring.fetch(stage, 0, k, x + k * place.hop, count);
            if (added) ring.fetch(stage, ARRAYS - 1, k, residual + k * place.hop, count);
        }
        ring.commit();
        ahead += place.step;
        x += p.x.advance;
        residual += p.residual.advance;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(s);

    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale, inverse = (A)1 / (A)p.cols;
    Two<A> weight[E / 2], bias[E / 2];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = place.at + e / V * place.hop + e % V;
        const A w = p.weight != nullptr && c < place.end ? load_param<T, A>(p.weight, p.params_f32, c) : (A)1;
        const A b = p.bias != nullptr && c < place.end ? load_param<T, A>(p.bias, p.params_f32, c) : (A)0;
        (e % 2 == 0 ? weight[e / 2].v.x : weight[e / 2].v.y) = w;
        (e % 2 == 0 ? bias[e / 2].v.x : bias[e / 2].v.y) = b;
    }

    // The groups of a CTA and the CTAs of a cluster make the same number of turns: `first` is that of group 0.
    int stage = 0;
    for (long long first = row - place.group; first < p.rows; first += place.step) {
        fetch(stage == 0 ? STAGES - 1 : stage - 1);  // into the slots that were read in the last turn
        ring.wait();
        const bool live = row < p.rows;
        Two<A> h[E / 2];
        ring.read(stage, 0, h);
        if (RESIDUAL) {
            if (p.draw.threshold != 0)
#pragma unroll
                for (int k = 0; k < K; ++k)
                    drop<V>(draws, (unsigned long long)row * p.cols + place.at + k * place.hop, scale, h, k);
            if (added) {
                Two<A> more[E / 2];
                ring.read(stage, ARRAYS - 1, more);
#pragma unroll
                for (int q = 0; q < E / 2; ++q) h[q] = h[q] + more[q];
            }
            if (p.h.data != nullptr && live)
#pragma unroll
                for (int k = 0; k < K; ++k) place.store(h_out, k, narrow_pack<T, V>(h, k), whole);
        }
        Two<A> total = h[0];
#pragma unroll
        for (int q = 1; q < E / 2; ++q) total = total + h[q];
        A sum[1] = {total.sum()};
        row_sum(sum);
        const A mean = sum[0] * inverse;
        Two<A> spread((A)0);
#pragma unroll
        for (int q = 0; q < E / 2; ++q) h[q] = h[q] + Two<A>(-mean);
        if (whole) {
#pragma unroll
            for (int q = 0; q < E / 2; ++q) spread = fma(h[q], h[q], spread);
        } else {  // what lies behind the row's end does not count
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const Two<A>& d = h[(k * V + i) / 2];
                    const A v = (k * V + i) % 2 == 0 ? d.v.x : d.v.y;
                    if (i < place.count(k)) spread.v.x += v * v;
                }
        }
        A squares[1] = {spread.sum()};
        row_sum(squares);
        const A rstd = reciprocal_root(squares[0] * inverse + (A)p.epsilon);
#pragma unroll
        for (int q = 0; q < E / 2; ++q) h[q] = fma(h[q] * Two<A>(rstd), weight[q], bias[q]);
        if (live) {
#pragma unroll
            for (int k = 0; k < K; ++k) place.store(y, k, narrow_pack<T, V>(h, k), whole);
            if (place.t == 0 && place.rank == 0) {
                if (p.mean != nullptr) static_cast<A*>(p.mean)[row] = mean;
                if (p.rstd != nullptr) static_cast<A*>(p.rstd)[row] = rstd;
            }
        }
        row += place.step;
        h_out += p.h.advance;
        y += p.y.advance;
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
    constexpr int ARRAYS = RESIDUAL ? 3 : 2, STAGES = norm_stages(sizeof(T), ARRAYS);
    using Ring = RowRing<T, V, ARRAYS, STAGES>;
    constexpr int E = Ring::E, K = Ring::K;
    __shared__ typename RowSum<A, 2>::Shared shared;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const Ring ring(dynamic);
    RowSum<A, 2> row_sum(shared, shape.threads_per_row, shape.cluster);
    const Place<T, V> place(shape, p.cols);
    const bool whole = place.whole();
    long long row = place.row, ahead = place.row;
    const bool added = RESIDUAL && p.dh.data != nullptr;
    const T* dy = static_cast<const T*>(p.dy.data) + row * p.dy.stride + place.at;
    const T* h = static_cast<const T*>(p.h.data) + row * p.h.stride + place.at;
    const T* dh = static_cast<const T*>(p.dh.data) + row * p.dh.stride + place.at;
    T* dx = static_cast<T*>(p.dx.data) + row * p.dx.stride + place.at;
    T* dresidual = static_cast<T*>(p.dresidual.data) + row * p.dresidual.stride + place.at;

    auto fetch = [&](int stage) {
        const bool there = ahead < p.rows;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int count = there ? (whole ? V : place.count(k)) : 0;
            ring.fetch(stage, 0, k, dy + k * place.hop, count);
            ring.fetch(stage, 1, k, h + k * place.hop, count);
            if (added) ring.fetch(stage, ARRAYS - 1, k, dh + k * place.hop, count);
        }
        ring.commit();
        ahead += place.step;
        dy += p.dy.advance;
        h += p.h.advance;
        dh += p.dh.advance;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(s);

    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale, inverse = (A)1 / (A)p.cols;
    Two<A> weight[E / 2], dweight[E / 2], dbias[E / 2];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = place.at + e / V * place.hop + e % V;
        (e % 2 == 0 ? weight[e / 2].v.x : weight[e / 2].v.y) =
            p.weight != nullptr && c < place.end ? load_param<T, A>(p.weight, p.params_f32, c) : (A)1;
        dweight[e / 2] = dbias[e / 2] = Two<A>((A)0);
    }

    const A* means = static_cast<const A*>(p.mean);
    const A* rstds = static_cast<const A*>(p.rstd);
    A next_mean = row < p.rows ? means[row] : (A)0, next_rstd = row < p.rows ? rstds[row] : (A)0;
    int stage = 0;
    for (long long first = row - place.group; first < p.rows; first += place.step) {
        fetch(stage == 0 ? STAGES - 1 : stage - 1);
        const Two<A> away(-next_mean), rstd(next_rstd);
        if (row + place.step < p.rows) {
            next_mean = means[row + place.step];
            next_rstd = rstds[row + place.step];
        }
        ring.wait();
        Two<A> one((A)0), along((A)0);
        {
            Two<A> d[E / 2], normal[E / 2];
            ring.read(stage, 0, d);
            ring.read(stage, 1, normal);
#pragma unroll
            for (int q = 0; q < E / 2; ++q) {
                normal[q] = (normal[q] + away) * rstd;
                const Two<A> g = d[q] * weight[q];
                dweight[q] = fma(d[q], normal[q], dweight[q]);
                dbias[q] = dbias[q] + d[q];
                one = one + g;
                along = fma(g, normal[q], along);
            }
        }
        A sums[2] = {one.sum(), along.sum()};
        row_sum(sums);
        const Two<A> along_one(-sums[0] * inverse), along_normal(-sums[1] * inverse);
        // The row is read from its slots once more: the registers hold the parameters' gradients.
        Two<A> d[E / 2], normal[E / 2];
        ring.read(stage, 0, d);
        ring.read(stage, 1, normal);
#pragma unroll
        for (int q = 0; q < E / 2; ++q) {
            normal[q] = (normal[q] + away) * rstd;
            d[q] = rstd * (fma(d[q], weight[q], along_one) + normal[q] * along_normal);
        }
        const bool live = row < p.rows;
        if (RESIDUAL) {
            if (added) {
                ring.read(stage, ARRAYS - 1, normal);
#pragma unroll
                for (int q = 0; q < E / 2; ++q) d[q] = d[q] + normal[q];
            }
            if (p.dresidual.data != nullptr && live)
#pragma unroll
                for (int k = 0; k < K; ++k) place.store(dresidual, k, narrow_pack<T, V>(d, k), whole);
            if (p.draw.threshold != 0)
#pragma unroll
                for (int k = 0; k < K; ++k)
                    drop<V>(draws, (unsigned long long)row * p.cols + place.at + k * place.hop, scale, d, k);
        }
        if (live)
#pragma unroll
            for (int k = 0; k < K; ++k) place.store(dx, k, narrow_pack<T, V>(d, k), whole);
        row += place.step;
        dx += p.dx.advance;
        dresidual += p.dresidual.advance;
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }

    if (p.dweight == nullptr && p.dbias == nullptr) return;
    const bool final = gridDim.x == (unsigned)shape.cluster;  // no other CTA has these columns
    A* const partial = static_cast<A*>(p.partial) + (long long)(blockIdx.x / shape.cluster) * 2 * p.cols;
    // Groups within a warp by shuffles, those of different warps (or warp groups) through shared memory, [team][2][width].
    const int threads = shape.threads_per_row, width = threads * E;
    for (int offset = 16; offset >= threads; offset /= 2)
#pragma unroll
        for (int q = 0; q < E / 2; ++q) {
            dweight[q].v.x += __shfl_xor_sync(0xffffffffu, dweight[q].v.x, offset);
            dweight[q].v.y += __shfl_xor_sync(0xffffffffu, dweight[q].v.y, offset);
            dbias[q].v.x += __shfl_xor_sync(0xffffffffu, dbias[q].v.x, offset);
            dbias[q].v.y += __shfl_xor_sync(0xffffffffu, dbias[q].v.y, offset);
        }
    const int teams = threads < 32 ? (int)blockDim.x / 32 : shape.groups;
    const int team = threads < 32 ? (int)threadIdx.x / 32 : place.group;
    A* const tile = reinterpret_cast<A*>(dynamic);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring is no longer read or written
    if (threads >= 32 || (int)(threadIdx.x % 32) < threads)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = (e / V) * place.hop + place.t * V + e % V;
            tile[team * 2 * width + c] = e % 2 == 0 ? dweight[e / 2].v.x : dweight[e / 2].v.y;
            tile[team * 2 * width + width + c] = e % 2 == 0 ? dbias[e / 2].v.x : dbias[e / 2].v.y;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < place.end - place.begin; c += blockDim.x) {
        A w = tile[c], b = tile[width + c];
        for (int i = 1; i < teams; ++i) {
            w += tile[i * 2 * width + c];
            b += tile[i * 2 * width + width + c];
        }
        if (final) {
            if (p.dweight != nullptr) store_gradient<T>(p.dweight, p.params_f32, place.begin + c, w);
            if (p.dbias != nullptr) store_gradient<T>(p.dbias, p.params_f32, place.begin + c, b);
        } else {
            partial[place.begin + c] = w;
            partial[p.cols + place.begin + c] = b;
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
cudaError_t norm_forward_launch(const NormForwardArgs& given, cudaStream_t stream) {
    NormForwardArgs a = given;
    constexpr int V = 16 / sizeof(T);
    const RowShape s = row_shape(a.cols, norm_elements(sizeof(T)));
    const int threads = s.threads_per_row * s.groups;
    const long long batches = (a.rows + s.groups - 1) / s.groups;
    const long long resident = NORM_SMS * std::max(1, NORM_MAX_THREADS / threads) / s.cluster;
    const unsigned grid = (unsigned)((batches < resident ? batches : resident) * s.cluster);
    for (RowArray* r : {&a.x, &a.residual, &a.h, &a.y}) r->advance = (long long)(grid / s.cluster) * s.groups * r->stride;
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
cudaError_t norm_backward_launch(const NormBackwardArgs& given, cudaStream_t stream) {
    NormBackwardArgs a = given;
    using A = typename Accumulator<T>::type;
    constexpr int V = 16 / sizeof(T);
    const RowShape s = row_shape(a.cols, norm_elements(sizeof(T)));
    const int threads = s.threads_per_row * s.groups;
    const int partials = norm_partials(a.rows, s);
    const unsigned grid = (unsigned)partials * s.cluster;
    for (RowArray* r : {&a.dy, &a.dh, &a.h, &a.dx, &a.dresidual}) r->advance = (long long)partials * s.groups * r->stride;
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
