// Layer norm, its gradients, dropout, and the residual form of both, over rows of float32, float64, float16 or
// bfloat16.
//
//   forward   h = residual + dropout(x);  mean, var over the row;  y = (h - mean) * rstd * weight + bias
//   backward  xh = (h - mean) * rstd, g = dy * weight:
//             dh' = rstd * (g - mean(g) - xh * mean(g * xh)) + dh;  dx = dropout(dh');
//             dweight = sum over rows of dy * xh;  dbias = sum over rows of dy
//
// A row stays on the SM between its one read and its one write, so the variance is taken about the mean (two passes over
// registers, not over memory).  Sums, statistics and gradients are float32 (float64 for float64 rows); the rows' type is
// rounded to once, on the way out.  Sums run in a fixed order: results repeat bit for bit.
//
// All of it is bound by memory in principle (4 to 10 bytes of traffic for a 16-bit element against 12 to 36 instructions);
// what kept the first versions from it was instruction issue and the latency of the rows' sums, so the layout below is about
// few instructions for an element and rows that are fetched ahead.  Rates are given as a share of the measured copy rate of
// 6542 GB/s, times are of one B200 with inputs that change from call to call.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <initializer_list>
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
    unsigned long long v;  // the pair as the instructions take it
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
    __device__ __forceinline__ float2 both() const {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
    __device__ __forceinline__ float sum() const { const float2 f = both(); return f.x + f.y; }
};
template <> struct Two<double> {
    double2 v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(double a, double b) : v(make_double2(a, b)) {}
    __device__ __forceinline__ explicit Two(double a) : v(make_double2(a, a)) {}
    __device__ __forceinline__ double2 both() const { return v; }
    __device__ __forceinline__ double sum() const { return v.x + v.y; }
};
__device__ __forceinline__ Two<float> operator+(Two<float> a, Two<float> b) {
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
    return a;
}
__device__ __forceinline__ Two<float> operator*(Two<float> a, Two<float> b) {
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
    return a;
}
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Two<double> operator+(Two<double> a, Two<double> b) { return {a.v.x + b.v.x, a.v.y + b.v.y}; }
__device__ __forceinline__ Two<double> operator*(Two<double> a, Two<double> b) { return {a.v.x * b.v.x, a.v.y * b.v.y}; }
__device__ __forceinline__ Two<double> fma(Two<double> a, Two<double> b, Two<double> c) {
    return {::fma(a.v.x, b.v.x, c.v.x), ::fma(a.v.y, b.v.y, c.v.y)};
}

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// A thread's packs of a row as pairs of accumulation-type values: pair q holds elements 2 q and 2 q + 1 of the packs
// put one behind the other (of the same pack, or of two packs of one element).
template <typename T, int V, int K, typename A>
__device__ __forceinline__ void widen_packs(const Pack<T, V> (&raw)[K], Two<A> (&pairs)[K * V / 2]) {
#pragma unroll
    for (int q = 0; q < K * V / 2; ++q) {
        if constexpr (V == 1) {
            pairs[q] = Two<A>(widen(raw[2 * q].v[0]), widen(raw[2 * q + 1].v[0]));
        } else {
            const T* two = &raw[2 * q / V].v[2 * q % V];
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(two));
                pairs[q] = Two<A>(f.x, f.y);
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // a bfloat16 is the upper half of a float32
                const unsigned u = *reinterpret_cast<const unsigned*>(two);
                pairs[q] = Two<A>(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
            } else {
                pairs[q] = Two<A>(two[0], two[1]);
            }
        }
    }
}

template <typename T, int V, typename A, int H>
__device__ __forceinline__ Pack<T, V> narrow_pack(const Two<A> (&pairs)[H], int k) {
    Pack<T, V> out;
    if constexpr (V == 1) {
        const auto f = pairs[k / 2].both();
        out.v[0] = narrow<T>(k % 2 == 0 ? f.x : f.y);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const auto f = pairs[(k * V + i) / 2].both();
            if constexpr (std::is_same<T, __half>::value)
                *reinterpret_cast<__half2*>(&out.v[i]) = __float22half2_rn(f);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value)
                *reinterpret_cast<__nv_bfloat162*>(&out.v[i]) = __float22bfloat162_rn(f);
            else
                out.v[i] = narrow<T>(f.x), out.v[i + 1] = narrow<T>(f.y);
        }
    }
    return out;
}

// The first `count` elements of a pack.
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* to, int count, const Pack<T, V>& p) {
    if (count >= V) {
        *reinterpret_cast<Pack<T, V>*>(to) = p;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < count) to[i] = p.v[i];
    }
}

template <typename T, typename A>
__device__ __forceinline__ A load_param(const void* params, bool f32, int c) {
    return f32 ? (A) static_cast<const float*>(params)[c] : (A)widen(static_cast<const T*>(params)[c]);
}

// How a thread finds its place.  SPAN is 32 where a row has one or more whole warps, each with 32 * E columns of its own
// one behind the other; 0 where several rows share a warp (threads_per_row is then a power of two below 32).  Pack k of a
// thread starts at column `at` + k * hop.  With whole warps every distance within a thread's packs and slots is a
// constant of the instruction: with distances from the launch instead the kernels issued half as many instructions again
// (8192 x 4096 bfloat16 forward: 22 against 13 million warp instructions, 40 against 30 us at that step).
template <typename T, int V, int SPAN, int ROWS> struct Place {
    static constexpr int E = norm_elements(sizeof(T)), K = E / V;
    int t, group, rank, begin, end, at;
    int run_hop;
    int solid;           // packs that lie within the row in every thread of a warp
    int there[ROWS];     // turns in which row r of the group exists
    int step;            // rows from one turn to the next
    long long row;       // the group works on rows [row, row + ROWS) at once
    __device__ __forceinline__ Place(const RowShape& shape, int cols, long long rows) {
        const int span = SPAN == 32 ? 32 : shape.threads_per_row;
        t = threadIdx.x % shape.threads_per_row;
        group = threadIdx.x / shape.threads_per_row;
        rank = blockIdx.x % shape.cluster;
        begin = rank * shape.slice;
        end = begin + shape.slice < cols ? begin + shape.slice : cols;
        at = begin + t / span * span * E + t % span * V;
        run_hop = span * V;
        const int run = end - (begin + t / span * span * E);  // columns from the warp's first one on
        solid = run >= E * span ? K : run > 0 ? run / (span * V) : 0;
        step = (int)(gridDim.x / shape.cluster) * shape.groups * ROWS;
        row = ((long long)(blockIdx.x / shape.cluster) * shape.groups + group) * ROWS;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) there[r] = row + r < rows ? (int)((rows - row - r + step - 1) / step) : 0;
    }
    // Turns of the whole CTA and cluster: those of group 0's first row, whose barriers all take part in.
    __device__ __forceinline__ int turns(long long rows) const {
        const long long first = row - group * ROWS;
        return first < rows ? (int)((rows - first + step - 1) / step) : 0;
    }
    __device__ __forceinline__ int hop() const { return SPAN == 32 ? 32 * V : run_hop; }
    // Elements of pack k that are in the row.
    __device__ __forceinline__ int count(int k) const {
        const int left = end - at - k * hop();
        return left >= V ? V : left > 0 ? left : 0;
    }
    __device__ __forceinline__ bool whole() const { return solid == K; }
    template <typename A>
    __device__ __forceinline__ void store(T* row_at, const Two<A> (&pairs)[E / 2], bool all) const {
        if (all) {
#pragma unroll
            for (int k = 0; k < K; ++k) *reinterpret_cast<Pack<T, V>*>(row_at + k * hop()) = narrow_pack<T, V>(pairs, k);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) store_pack<T, V>(row_at + k * hop(), k < solid ? V : count(k), narrow_pack<T, V>(pairs, k));
        }
    }
};

// N sums over the threads of a row, the same in every one of them: shuffles within a warp, shared memory across the
// warps of the row's group (a named barrier for each group, so groups do not wait for one another), distributed shared
// memory across the CTAs of a cluster.  Two buffers in turn, so each call costs one barrier at each level.
template <typename A, int N, int SPAN> struct RowSum {
    static constexpr int LANES = 32 / N;  // that carry one of the sums on
    struct Shared {
        A warps[2][N][NORM_MAX_THREADS / 32];
        A ranks[2][NORM_MAX_CLUSTER][N];
    };
    Shared& shared;
    const int threads_per_row, cluster, lane, warp, warps, group;
    int turn = 0;
    __device__ __forceinline__ RowSum(Shared& s, const RowShape& shape)
        : shared(s), threads_per_row(shape.threads_per_row), cluster(shape.cluster), lane(threadIdx.x % 32), warp(threadIdx.x / 32),
          warps(shape.threads_per_row / 32), group(threadIdx.x / shape.threads_per_row) {
        if (SPAN == 32 && cluster > 1) cooperative_groups::this_cluster().barrier_arrive();
    }
    // Before the first sum: the shared memory of a cluster's other CTAs may be written only once they run.  Every thread
    // has arrived when it entered the kernel, so the wait lies under the first rows' copies.
    __device__ __forceinline__ void meet() const {
        if (SPAN == 32 && cluster > 1) cooperative_groups::this_cluster().barrier_wait();
    }

    __device__ __forceinline__ void operator()(A (&v)[N]) {
        if constexpr (SPAN == 32) {
            whole_warps(v);
        } else {
            for (int offset = threads_per_row / 2; offset > 0; offset /= 2)
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], offset);
        }
    }

private:
    __device__ __forceinline__ void whole_warps(A (&v)[N]) {
        // Over the warp.  While there are several sums, half of the lanes goes on with half of them: lanes
        // [n * LANES, (n + 1) * LANES) end up with sum n.
        A part[N];
#pragma unroll
        for (int n = 0; n < N; ++n) part[n] = v[n];
#pragma unroll
        for (int offset = 16, left = N; offset > 0; offset /= 2) {
            if (left > 1) {
                left /= 2;
#pragma unroll
                for (int n = 0; n < left; ++n) {
                    const A send = lane & offset ? part[n] : part[n + left];
                    part[n] = (lane & offset ? part[n + left] : part[n]) + __shfl_xor_sync(0xffffffffu, send, offset);
                }
            } else {
                part[0] += __shfl_xor_sync(0xffffffffu, part[0], offset);
            }
        }
        if (warps > 1) {  // over the (at most 16) warps of the row
            A* const here = shared.warps[turn][lane / LANES];
            if (lane % LANES == 0) here[warp] = part[0];
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads_per_row) : "memory");  // 0 is the whole CTA's
            constexpr int PART = LANES < 16 ? LANES : 16;
            const A* const there = here + group * warps;
            part[0] = lane % PART < warps ? there[lane % PART] : (A)0;
            if (PART < 16 && lane % PART + PART < warps) part[0] += there[lane % PART + PART];
#pragma unroll
            for (int offset = PART / 2; offset > 0; offset /= 2) part[0] += __shfl_xor_sync(0xffffffffu, part[0], offset);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = N == 1 ? part[0] : __shfl_sync(0xffffffffu, part[0], n * LANES);
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
// few turns ahead of the one in work, so the copies need no barrier and their latency is hidden whatever the occupancy.
// Packs behind a row's end or the last row arrive as zeros.  The same slot of a warp's lanes is one run of shared memory
// (with a thread's slots together instead, the kernels took 10 to 35 % longer).
template <typename T, int V, int ARRAYS, int ROWS, int STAGES> struct RowRing {
    static constexpr int E = norm_elements(sizeof(T)), K = E / V, BYTES = V * sizeof(T);
    static constexpr int STAGE_BYTES = ROWS * ARRAYS * K * 32 * BYTES;  // of a warp
    static constexpr int THREAD_BYTES = STAGES * ROWS * ARRAYS * E * sizeof(T);
    char* const slots;  // [warps][STAGES][ROWS][ARRAYS][K][32]
    __device__ __forceinline__ explicit RowRing(void* shared)
        : slots(static_cast<char*>(shared) + threadIdx.x / 32 * (STAGES * STAGE_BYTES) + threadIdx.x % 32 * BYTES) {}
    __device__ __forceinline__ char* stage(int s) const { return slots + s * STAGE_BYTES; }
    static __device__ __forceinline__ Pack<T, V>* at(char* stage, int r, int array, int k) {
        return reinterpret_cast<Pack<T, V>*>(stage + ((r * ARRAYS + array) * K + k) * 32 * BYTES);
    }
    // Pack k of an array: all of it, or its first `count` elements (none for a row that is not there).
    static __device__ __forceinline__ void fetch(char* stage, int r, int array, int k, const T* from) {
        const unsigned to = (unsigned)__cvta_generic_to_shared(at(stage, r, array, k));
        if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
    }
    static __device__ __forceinline__ void fetch(char* stage, int r, int array, int k, const T* from, int count) {
        const unsigned to = (unsigned)__cvta_generic_to_shared(at(stage, r, array, k));
        const int bytes = count * (int)sizeof(T);
        if constexpr (BYTES == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(bytes) : "memory");
    }
    // Row r of a turn: a thread's packs of all arrays, the last one of which may be absent.  No asynchronous copy is as small
    // as one 16-bit element: all loads go before the stores to the slots, and of a single array they wait in registers until
    // `settle` stores them at the turn's end (8192 x 4095 bfloat16 49 us, otherwise 62; of more arrays the registers spill).
    static constexpr bool LATE = BYTES < 4 && ARRAYS == 1;
    struct Pending { T v[BYTES < 4 ? ARRAYS : 1][BYTES < 4 ? K : 1]; };
    static __device__ __forceinline__ void put(char* stage, int r, const Pending& pending) {
#pragma unroll
        for (int a = 0; a < ARRAYS; ++a)
#pragma unroll
            for (int k = 0; k < K; ++k) at(stage, r, a, k)->v[0] = pending.v[a][k];
    }
    static __device__ __forceinline__ void settle(char* stage, const Pending (&pending)[ROWS]) {
        if constexpr (LATE)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) put(stage, r, pending[r]);
    }
    template <typename P>
    static __device__ __forceinline__ void fetch_row(char* stage, int r, const T* const (&from)[ARRAYS], bool last, const P& place,
                                                     bool there, Pending& pending) {
        if constexpr (BYTES < 4) {
#pragma unroll
            for (int a = 0; a < ARRAYS; ++a)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const bool present = there && place.count(k) > 0 && (last || a < ARRAYS - 1);
                    pending.v[a][k] = present ? from[a][k * place.hop()] : narrow<T>((typename Accumulator<T>::type)0);
                }
            if constexpr (!LATE) put(stage, r, pending);
        } else if (there && place.whole()) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int a = 0; a < ARRAYS; ++a)
                    if (last || a < ARRAYS - 1) fetch(stage, r, a, k, from[a] + k * place.hop());
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int count = there ? place.count(k) : 0;
#pragma unroll
                for (int a = 0; a < ARRAYS; ++a)
                    if (last || a < ARRAYS - 1) fetch(stage, r, a, k, from[a] + k * place.hop(), count);
            }
        }
    }
    // A thread's packs of a row as pairs.
    template <typename A> static __device__ __forceinline__ void read(char* stage, int r, int array, Two<A> (&pairs)[E / 2]) {
        Pack<T, V> raw[K];
#pragma unroll
        for (int k = 0; k < K; ++k) raw[k] = *at(stage, r, array, k);
        widen_packs<T, V>(raw, pairs);
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // All but the youngest STAGES - 1 turns' copies have landed.
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
};

// A thread's columns of a parameter, 1 or 0 where there is none.
template <typename T, int V, typename P, typename A, int H>
__device__ __forceinline__ void load_columns(const P& place, const void* params, bool f32, A absent, Two<A> (&pairs)[H]) {
#pragma unroll
    for (int q = 0; q < H; ++q) {
        A v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = place.at + (2 * q + i) / V * place.hop() + (2 * q + i) % V;
            v[i] = params != nullptr && c < place.end ? load_param<T, A>(params, f32, c) : absent;
        }
        pairs[q] = Two<A>(v[0], v[1]);
    }
}

// How a kernel draws: not at all; PLAIN where every pack starts with the low half of a word (even columns and counter) and
// no half is flipped; ANY otherwise.  The plain draws are straight code, which the compiler spreads over the waits of what is
// around them (5 of 104 us of the residual form's gradient at 8192 x 5120 bfloat16).
enum class Draws { NONE, PLAIN, ANY };
template <Draws D> using DrawsTag = std::integral_constant<Draws, D>;
template <int V>
__device__ __forceinline__ Draws draws_of(const DrawStream& draws, int cols) {
    if (!draws.active) return Draws::NONE;
    return V > 1 && draws.odd == 0 && cols % 2 == 0 && !draws.flips() ? Draws::PLAIN : Draws::ANY;
}

// Dropout of PACKS packs of V elements, `hop` columns from one to the next; `index` is the row-major number of the first.
// Both halves of a word are used; where the elements start with a high half, a pack takes one word more.  (The branches on
// that hold the whole work: decisions that leave them would have to pass through registers.)
template <int V, int PACKS, bool FLIP, typename A>
__device__ __forceinline__ void drop_from_low(const DrawStream& draws, long long index, int hop, A scale, Two<A>* pairs) {
    const unsigned long long first = draws.at(index);
#pragma unroll
    for (int k = 0; k < PACKS; ++k)
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const unsigned long long z = DrawStream::mix(first + ((unsigned long long)(k * hop / 2) + j) * DrawStream::GAMMA);
            const auto f = (pairs[k * V / 2 + j] * Two<A>(scale)).both();
            pairs[k * V / 2 + j] = Two<A>(draws.low_kept(z) ? f.x : (A)0, draws.high_kept<FLIP>(z) ? f.y : (A)0);
        }
}

template <int V, int PACKS, bool FLIP, typename A>
__device__ __forceinline__ void drop_from_high(const DrawStream& draws, long long index, int hop, A scale, Two<A>* pairs) {
    const unsigned long long first = draws.at(index);
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
        const unsigned long long at = first + (unsigned long long)(k * hop / 2) * DrawStream::GAMMA;
        unsigned long long last = DrawStream::mix(at);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const unsigned long long z = DrawStream::mix(at + (j + 1) * DrawStream::GAMMA);
            const auto f = (pairs[k * V / 2 + j] * Two<A>(scale)).both();
            pairs[k * V / 2 + j] = Two<A>(draws.high_kept<FLIP>(last) ? f.x : (A)0, draws.low_kept(z) ? f.y : (A)0);
            last = z;
        }
    }
}

template <int V, int PACKS, Draws D = Draws::ANY, typename A>
__device__ __forceinline__ void drop(const DrawStream& draws, long long index, int hop, A scale, Two<A>* pairs) {
    if constexpr (D == Draws::NONE) {
        return;
    } else if constexpr (V == 1) {
        // An even number of columns apart, a thread's elements are the same halves of words a constant apart.
        const unsigned long long first = draws.at(index);
        const bool even = hop % 2 == 0, high = draws.half(index) != 0;
        auto kept = [&](int k) {
            return even ? draws.kept_half(first + (unsigned long long)(k * (hop / 2)) * DrawStream::GAMMA, high)
                        : draws.kept(index + k * hop);
        };
#pragma unroll
        for (int k = 0; k < PACKS; k += 2) {
            const auto f = (pairs[k / 2] * Two<A>(scale)).both();
            pairs[k / 2] = Two<A>(kept(k) ? f.x : (A)0, kept(k + 1) ? f.y : (A)0);
        }
    } else if constexpr (D == Draws::PLAIN) {
        drop_from_low<V, PACKS, false>(draws, index, hop, scale, pairs);
    } else if (draws.flips()) {
        if (draws.half(index) == 0) drop_from_low<V, PACKS, true>(draws, index, hop, scale, pairs);
        else drop_from_high<V, PACKS, true>(draws, index, hop, scale, pairs);
    } else {
        if (draws.half(index) == 0) drop_from_low<V, PACKS, false>(draws, index, hop, scale, pairs);
        else drop_from_high<V, PACKS, false>(draws, index, hop, scale, pairs);
    }
}

// A residual kernel's rows by the way it draws.
template <int V, bool RESIDUAL, typename F>
__device__ __forceinline__ void by_draws(const DrawStream& draws, int cols, F&& rows) {
    if constexpr (RESIDUAL) {
        const Draws d = draws_of<V>(draws, cols);
        if (d == Draws::NONE) rows(DrawsTag<Draws::NONE>());
        else if (V > 1 && d == Draws::PLAIN) rows(DrawsTag<V == 1 ? Draws::ANY : Draws::PLAIN>());
        else rows(DrawsTag<Draws::ANY>());
    } else {
        rows(DrawsTag<Draws::NONE>());
    }
}

// RESIDUAL: x passes through dropout and may be added to a residual; otherwise h = x.
// 8192 x 4096 bfloat16: 26.7 us, 77 % (32768 rows: 88 us, 92 %: launch and first rows are 4 us); float32 45 us, 91 %.  The
// residual form of 4096 x 4096 bfloat16 32 us, 64 %, 28.5 without dropout: the draws are 10 integer instructions an element
// and 16 warps an SM do not hide all of them.  More warps with fewer registers, parameters in shared memory, and draws for
// the next turn during this one's sums all measured slower or the same.
template <typename T, int V, int SPAN, bool RESIDUAL>
__global__ void __maxnreg__(128)
norm_forward_kernel(const __grid_constant__ NormForwardArgs p, const RowShape shape) {
    using A = typename Accumulator<T>::type;
    constexpr bool WIDE = V * sizeof(T) == 16;
    constexpr int ARRAYS = RESIDUAL ? 2 : 1, R = norm_forward_rows(sizeof(T), WIDE);
    constexpr int STAGES = norm_forward_stages(sizeof(T), WIDE, RESIDUAL);
    using Ring = RowRing<T, V, ARRAYS, R, STAGES>;
    constexpr int E = Ring::E, K = Ring::K;
    __shared__ typename RowSum<A, R, SPAN>::Shared shared;
    extern __shared__ __align__(16) char dynamic[];
    const Ring ring(dynamic);
    RowSum<A, R, SPAN> row_sum(shared, shape);
    const Place<T, V, SPAN, R> place(shape, p.cols, p.rows);
    const bool whole = place.whole(), added = RESIDUAL && p.residual.data != nullptr;
    long long row = place.row;
    const T* x = static_cast<const T*>(p.x.data) + row * p.x.stride + place.at;
    const T* residual = static_cast<const T*>(p.residual.data) + row * p.residual.stride + place.at;
    T* h_out = static_cast<T*>(p.h.data) + row * p.h.stride + place.at;
    T* y = static_cast<T*>(p.y.data) + row * p.y.stride + place.at;

    typename Ring::Pending pending[R];
    auto fetch = [&](char* stage, int turn) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const T* from[ARRAYS];
            if (RESIDUAL) from[ARRAYS - 1] = residual + r * p.residual.stride;
            from[0] = x + r * p.x.stride;
            ring.fetch_row(stage, r, from, !RESIDUAL || added, place, turn < place.there[r], pending[r]);
        }
        ring.commit();
        x += p.x.advance;
        if (RESIDUAL) residual += p.residual.advance;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        fetch(ring.stage(s), s);
        ring.settle(ring.stage(s), pending);
    }

    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale, inverse = (A)1 / (A)p.cols;
    Two<A> weight[E / 2], bias[E / 2];
    load_columns<T, V>(place, p.weight, p.params_f32, (A)1, weight);
    load_columns<T, V>(place, p.bias, p.params_f32, (A)0, bias);

    row_sum.meet();
    by_draws<V, RESIDUAL>(draws, p.cols, [&](auto how) {
        const int turns = place.turns(p.rows);
        char *now = ring.stage(0), *free = ring.stage(STAGES - 1);  // the slots in work; those read in the last turn
        for (int turn = 0; turn < turns; ++turn) {
            char* const next = free;
            fetch(next, turn + STAGES - 1);
            ring.wait();
            Two<A> h[R][E / 2];
            A sum[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                ring.read(now, r, 0, h[r]);
                if (RESIDUAL) {
                    drop<V, K, decltype(how)::value>(draws, (row + r) * p.cols + place.at, place.hop(), scale, h[r]);
                    if (added) {
                        Two<A> more[E / 2];
                        ring.read(now, r, ARRAYS - 1, more);
#pragma unroll
                        for (int q = 0; q < E / 2; ++q) h[r][q] = h[r][q] + more[q];
                    }
                    if (p.h.data != nullptr && turn < place.there[r]) place.store(h_out + r * p.h.stride, h[r], whole);
                }
                Two<A> even = h[r][0], odd = h[r][1];
#pragma unroll
                for (int q = 2; q < E / 2; q += 2) even = even + h[r][q], odd = odd + h[r][q + 1];
                sum[r] = (even + odd).sum();
            }
            free = now;
            now = now == ring.stage(STAGES - 1) ? ring.stage(0) : now + Ring::STAGE_BYTES;
            row_sum(sum);
            A squares[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                sum[r] *= inverse;
                const Two<A> away(-sum[r]);
#pragma unroll
                for (int q = 0; q < E / 2; ++q) h[r][q] = h[r][q] + away;
                if (whole) {
                    Two<A> even = h[r][0] * h[r][0], odd = h[r][1] * h[r][1];
#pragma unroll
                    for (int q = 2; q < E / 2; q += 2) even = fma(h[r][q], h[r][q], even), odd = fma(h[r][q + 1], h[r][q + 1], odd);
                    squares[r] = (even + odd).sum();
                } else {  // what lies behind the row's end does not count
                    squares[r] = (A)0;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const int count = k < place.solid ? V : place.count(k);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const auto d = h[r][(k * V + i) / 2].both();
                            const A v = (k * V + i) % 2 == 0 ? d.x : d.y;
                            if (i < count) squares[r] += v * v;
                        }
                    }
                }
            }
            row_sum(squares);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const A rstd = reciprocal_root(squares[r] * inverse + (A)p.epsilon);
                const Two<A> factor(rstd);
#pragma unroll
                for (int q = 0; q < E / 2; ++q) h[r][q] = fma(h[r][q] * factor, weight[q], bias[q]);
                if (turn < place.there[r]) {
                    place.store(y + r * p.y.stride, h[r], whole);
                    if (place.t == 0 && place.rank == 0) {
                        if (p.mean != nullptr) static_cast<A*>(p.mean)[row + r] = sum[r];
                        if (p.rstd != nullptr) static_cast<A*>(p.rstd)[row + r] = rstd;
                    }
                }
            }
            ring.settle(next, pending);
            row += place.step;
            y += p.y.advance;
            if (RESIDUAL) h_out += p.h.advance;
        }
    });
}

// A parameter's gradient in the parameters' type.
template <typename T, typename A>
__device__ __forceinline__ void store_gradient(void* out, bool f32, int c, A v) {
    if (f32) static_cast<float*>(out)[c] = (float)v;
    else static_cast<T*>(out)[c] = narrow<T>(v);
}

// A thread's sums to its columns; `wide`: 16-byte stores where a pack is whole.
template <typename A, int V, int K, typename P, int H>
__device__ __forceinline__ void store_sums(A* at, const P& place, const Two<A> (&pairs)[H], bool wide) {
    constexpr int W = 16 / sizeof(A);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const Pack<A, V> sums = narrow_pack<A, V>(pairs, k);
        A* const to = at + k * place.hop();
        if (V % W == 0 && wide && k < place.solid) {
#pragma unroll
            for (int i = 0; i < V; i += W) *reinterpret_cast<Pack<A, W>*>(to + i) = *reinterpret_cast<const Pack<A, W>*>(&sums.v[i]);
        } else {
            store_pack<A, 1>(to, place.count(k), Pack<A, 1>{{sums.v[0]}});
#pragma unroll
            for (int i = 1; i < V; ++i) store_pack<A, 1>(to + i, place.count(k) - i, Pack<A, 1>{{sums.v[i]}});
        }
    }
}

// RESIDUAL: dh is added to the row's gradient, which goes to dresidual, and through dropout's mask to dx.
// Threads keep their columns' share of dweight and dbias in registers over all rows of the CTA; at the end the CTA's
// groups are added up through shared memory, in order, and the CTA writes one row of partial sums (the gradients
// themselves where there is only one).
// 262144 x 128 float32: 70 us with the joining kernel, 88 % (63 without the parameters' gradients); 8192 x 8192 bfloat16 72 to
// 78 us, 79 to 86 %.  The residual form at 8192 x 5120 bfloat16 96 us, 67 %, 76 without dropout: rows of 4097 to 5120 columns
// take 320 threads of the 512 that fit an SM's registers, too few warps to hide the draws.  Clusters of two CTAs for such
// rows, one row at a time with 96 registers, and masks drawn before the sums measured slower.
template <typename T, int V, int SPAN, bool RESIDUAL>
__global__ void __maxnreg__(128)
norm_backward_kernel(const __grid_constant__ NormBackwardArgs p, const RowShape shape) {
    using A = typename Accumulator<T>::type;
    constexpr bool WIDE = V * sizeof(T) == 16;
    constexpr int ARRAYS = RESIDUAL ? 3 : 2, R = norm_backward_rows(sizeof(T), WIDE, SPAN == 32), STAGES = norm_backward_stages(RESIDUAL);
    using Ring = RowRing<T, V, ARRAYS, R, STAGES>;
    constexpr int E = Ring::E, K = Ring::K;
    __shared__ typename RowSum<A, 2 * R, SPAN>::Shared shared;
    extern __shared__ __align__(16) char dynamic[];
    const Ring ring(dynamic);
    RowSum<A, 2 * R, SPAN> row_sum(shared, shape);
    const Place<T, V, SPAN, R> place(shape, p.cols, p.rows);
    const bool whole = place.whole(), added = RESIDUAL && p.dh.data != nullptr;
    long long row = place.row;
    const T* dy = static_cast<const T*>(p.dy.data) + row * p.dy.stride + place.at;
    const T* h = static_cast<const T*>(p.h.data) + row * p.h.stride + place.at;
    const T* dh = static_cast<const T*>(p.dh.data) + row * p.dh.stride + place.at;
    T* dx = static_cast<T*>(p.dx.data) + row * p.dx.stride + place.at;
    T* dresidual = static_cast<T*>(p.dresidual.data) + row * p.dresidual.stride + place.at;

    typename Ring::Pending pending[R];
    auto fetch = [&](char* stage, int turn) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const T* from[ARRAYS];
            if (RESIDUAL) from[ARRAYS - 1] = dh + r * p.dh.stride;
            from[0] = dy + r * p.dy.stride;
            from[1] = h + r * p.h.stride;
            ring.fetch_row(stage, r, from, !RESIDUAL || added, place, turn < place.there[r], pending[r]);
        }
        ring.commit();
        dy += p.dy.advance;
        h += p.h.advance;
        if (RESIDUAL) dh += p.dh.advance;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(ring.stage(s), s);

    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale, inverse = (A)1 / (A)p.cols;
    Two<A> weight[E / 2], dweight[E / 2], dbias[E / 2];
    load_columns<T, V>(place, p.weight, p.params_f32, (A)1, weight);
#pragma unroll
    for (int q = 0; q < E / 2; ++q) dweight[q] = dbias[q] = Two<A>((A)0);

    const A* means = static_cast<const A*>(p.mean) + row;
    const A* rstds = static_cast<const A*>(p.rstd) + row;
    A next_mean[R], next_rstd[R];
    auto fetch_statistics = [&](int turn) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            next_mean[r] = turn < place.there[r] ? means[r] : (A)0;
            next_rstd[r] = turn < place.there[r] ? rstds[r] : (A)0;
        }
        means += place.step;
        rstds += place.step;
    };
    fetch_statistics(0);
    row_sum.meet();
    by_draws<V, RESIDUAL>(draws, p.cols, [&](auto how) {
        const int turns = place.turns(p.rows);
        char *now = ring.stage(0), *free = ring.stage(STAGES - 1);
        for (int turn = 0; turn < turns; ++turn) {
            fetch(free, turn + STAGES - 1);
            Two<A> away[R], rstd[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                away[r] = Two<A>(-next_mean[r]);
                rstd[r] = Two<A>(next_rstd[r]);
            }
            fetch_statistics(turn + 1);
            ring.wait();
            A sums[2 * R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                Two<A> d[E / 2], normal[E / 2], one((A)0), along((A)0);
                ring.read(now, r, 0, d);
                ring.read(now, r, 1, normal);
#pragma unroll
                for (int q = 0; q < E / 2; ++q) {
                    normal[q] = (normal[q] + away[r]) * rstd[r];
                    const Two<A> g = d[q] * weight[q];
                    dweight[q] = fma(d[q], normal[q], dweight[q]);
                    dbias[q] = dbias[q] + d[q];
                    one = one + g;
                    along = fma(g, normal[q], along);
                }
                sums[2 * r] = one.sum();
                sums[2 * r + 1] = along.sum();
            }
            row_sum(sums);
            // The rows are read from their slots once more: the registers hold the parameters' gradients.
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const Two<A> along_one(-sums[2 * r] * inverse), along_normal(-sums[2 * r + 1] * inverse);
                Two<A> d[E / 2], normal[E / 2];
                ring.read(now, r, 0, d);
                ring.read(now, r, 1, normal);
#pragma unroll
                for (int q = 0; q < E / 2; ++q)
                    d[q] = rstd[r] * fma((normal[q] + away[r]) * rstd[r], along_normal, fma(d[q], weight[q], along_one));
                const bool live = turn < place.there[r];
                if (RESIDUAL) {
                    if (added) {
                        ring.read(now, r, ARRAYS - 1, normal);
#pragma unroll
                        for (int q = 0; q < E / 2; ++q) d[q] = d[q] + normal[q];
                    }
                    if (p.dresidual.data != nullptr && live) place.store(dresidual + r * p.dresidual.stride, d, whole);
                    drop<V, K, decltype(how)::value>(draws, (row + r) * p.cols + place.at, place.hop(), scale, d);
                }
                if (live) place.store(dx + r * p.dx.stride, d, whole);
            }
            free = now;
            now = now == ring.stage(STAGES - 1) ? ring.stage(0) : now + Ring::STAGE_BYTES;
            row += place.step;
            dx += p.dx.advance;
            if (RESIDUAL) dresidual += p.dresidual.advance;
        }
    });

    asm volatile("griddepcontrol.launch_dependents;");  // the joining kernel's CTAs may take the places of those that end
    if (p.dweight == nullptr && p.dbias == nullptr) return;
    const bool final = gridDim.x == (unsigned)shape.cluster;  // no other CTA has these columns
    A* const partial = static_cast<A*>(p.partial) + (long long)(blockIdx.x / shape.cluster) * 2 * p.cols;
    // Groups within a warp by shuffles, those of different warps (or warp groups) through shared memory, [team][2][width].
    const int threads = shape.threads_per_row, width = threads * E;
    if (SPAN != 32)
        for (int offset = 16; offset >= threads; offset /= 2)
#pragma unroll
            for (int q = 0; q < E / 2; ++q) {
                const auto w = dweight[q].both(), b = dbias[q].both();
                dweight[q] = dweight[q] + Two<A>(__shfl_xor_sync(0xffffffffu, w.x, offset), __shfl_xor_sync(0xffffffffu, w.y, offset));
                dbias[q] = dbias[q] + Two<A>(__shfl_xor_sync(0xffffffffu, b.x, offset), __shfl_xor_sync(0xffffffffu, b.y, offset));
            }
    const int teams = SPAN != 32 ? (int)blockDim.x / 32 : shape.groups;
    if (teams == 1 && !final) {  // straight to the CTA's partial row
        store_sums<A, V, K>(partial + place.at, place, dweight, p.cols % 4 == 0);
        store_sums<A, V, K>(partial + p.cols + place.at, place, dbias, p.cols % 4 == 0);
        return;
    }
    const int team = SPAN != 32 ? (int)threadIdx.x / 32 : place.group;
    A* const tile = reinterpret_cast<A*>(dynamic);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring is no longer read or written
    if (SPAN == 32 || (int)(threadIdx.x % 32) < threads) {
        store_sums<A, V, K>(tile + team * 2 * width + place.at - place.begin, place, dweight, true);
        store_sums<A, V, K>(tile + team * 2 * width + width + place.at - place.begin, place, dbias, true);
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

// dweight and dbias from the partial rows: 8 threads across the columns of one of the two, W columns each (16 bytes where
// the rows allow), 32 threads along the rows, so that all loads of a thread are under way at once; added in double in a
// fixed order.
template <typename T, int W>
__global__ void __launch_bounds__(256) norm_join_kernel(const __grid_constant__ NormBackwardArgs p, int partials) {
    using A = typename Accumulator<T>::type;
    __shared__ double sums[8][8 * W];
    const int across = threadIdx.x % 8, lane = threadIdx.x / 8, c = (blockIdx.x * 8 + across) * W;
    void* out = blockIdx.y == 0 ? p.dweight : p.dbias;
    if (out == nullptr) return;
    const A* partial = static_cast<const A*>(p.partial) + (long long)blockIdx.y * p.cols + c;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the partial rows are there
    double sum[W] = {};
    if (c < p.cols) {
#pragma unroll 10
        for (int r = lane; r < partials; r += 32) {
            const Pack<A, W> part = *reinterpret_cast<const Pack<A, W>*>(partial + (long long)r * 2 * p.cols);
#pragma unroll
            for (int i = 0; i < W; ++i) sum[i] += (double)part.v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 8);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 16);
        if (threadIdx.x % 32 < 8) sums[threadIdx.x / 32][across * W + i] = sum[i];
    }
    __syncthreads();
    const int column = blockIdx.x * 8 * W + threadIdx.x;
    if (threadIdx.x >= 8 * W || column >= p.cols) return;
    double total = sums[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 8; ++w) total += sums[w][threadIdx.x];
    store_gradient<T>(out, p.params_f32, column, (A)total);
}

// Elements [low, high) of a pack, the others as zeros.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_part(const T* from, int low, int high) {
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = i >= low && i < high ? from[i] : narrow<T>((typename Accumulator<T>::type)0);
    return p;
}

template <typename T, int V, int PACKS, typename A>
__device__ __forceinline__ void drop_packs(const DrawStream& draws, long long index, int hop, A scale, Pack<T, V> (&v)[PACKS]) {
    if (!draws.active) return;
    if constexpr (V == 1) {
#pragma unroll
        for (int d = 0; d < PACKS; ++d) v[d].v[0] = narrow<T>(draws.kept(index + d * hop) ? widen(v[d].v[0]) * scale : (A)0);
    } else {
        Two<A> pairs[PACKS * V / 2];
        widen_packs<T, V>(v, pairs);
        drop<V, PACKS>(draws, index, hop, scale, pairs);
#pragma unroll
        for (int d = 0; d < PACKS; ++d) v[d] = narrow_pack<T, V>(pairs, d);
    }
}

// Dropout alone.  Rows are taken in 16-byte packs from 16-byte boundary to boundary wherever they start, as long as x and y
// start at the same distance from one (V > 1): pack i of a row holds columns [i * V - shift, (i + 1) * V - shift).  One
// long row (what a contiguous array is) and many rows are two kernels: in the one row the four packs that a thread has on
// their way are a constant distance apart in the stream of words; of many rows a thread has two (8192 x 4095 bfloat16 55 us, with
// four 62).
// 16384 x 8192 bfloat16: 108 us, 76 %: the integer units are 71 % busy (10 of 17.5 instructions for an element, 4 bytes of
// traffic); 8192 x 8192 float32 86 us, 95 %.
__host__ __device__ constexpr int dropout_depth(bool one_row) { return one_row ? 4 : 2; }
template <typename T, int V, bool ONE_ROW>
__global__ void __launch_bounds__(256, ONE_ROW ? 4 : 6)
dropout_kernel(const __grid_constant__ DropoutArgs p, long long packs, long long packs_per_row) {
    using A = typename Accumulator<T>::type;
    constexpr int DEPTH = dropout_depth(ONE_ROW);
    const DrawStream draws(p.draw);
    const A scale = (A)p.draw.scale;
    const int hop = (int)(gridDim.x * blockDim.x);
    auto shift_of = [](const T* x) { return V == 1 ? 0 : (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % V); };
    for (long long first = (long long)blockIdx.x * blockDim.x + threadIdx.x; first < packs; first += (long long)DEPTH * hop) {
        if constexpr (ONE_ROW) {
            const T* const x = static_cast<const T*>(p.x.data);
            T* const y = static_cast<T*>(p.y.data);
            const long long c = first * V - shift_of(x);
            if (c >= 0 && c + (long long)(DEPTH - 1) * hop * V + V <= p.cols) {
                Pack<T, V> v[DEPTH];
#pragma unroll
                for (int d = 0; d < DEPTH; ++d) v[d] = *reinterpret_cast<const Pack<T, V>*>(x + c + d * hop * V);
                drop_packs(draws, c, hop * V, scale, v);
#pragma unroll
                for (int d = 0; d < DEPTH; ++d) *reinterpret_cast<Pack<T, V>*>(y + c + d * hop * V) = v[d];
                continue;
            }
        }
        Pack<T, V> v[DEPTH];
        long long row[DEPTH], c[DEPTH];
        int low[DEPTH], high[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const long long pack = first + (long long)d * hop;
            if (ONE_ROW) row[d] = 0;
            else row[d] = packs <= 0xffffffffll ? (long long)((unsigned int)pack / (unsigned int)packs_per_row) : pack / packs_per_row;
            const T* x = static_cast<const T*>(p.x.data) + row[d] * p.x.stride;
            c[d] = (pack - row[d] * packs_per_row) * V - shift_of(x);
            const long long left = p.cols - c[d];
            low[d] = c[d] < 0 ? (int)-c[d] : 0;
            high[d] = pack >= packs || left <= 0 ? 0 : left < V ? (int)left : V;
            if (low[d] == 0 && high[d] == V) v[d] = *reinterpret_cast<const Pack<T, V>*>(x + c[d]);
            else v[d] = load_part<T, V>(x + c[d], low[d], high[d]);
        }
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (high[d] == 0) continue;
            Pack<T, V> one[1] = {v[d]};
            drop_packs(draws, row[d] * p.cols + c[d], 0, scale, one);
            T* y = static_cast<T*>(p.y.data) + row[d] * p.y.stride + c[d];
            if (low[d] == 0 && high[d] == V) {
                *reinterpret_cast<Pack<T, V>*>(y) = one[0];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i >= low[d] && i < high[d]) y[i] = one[0].v[i];
            }
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------

// Whether rows start on boundaries of `bytes`, so that a thread can take that much at a time.
inline bool rows_aligned(const RowArray& a, long long rows, size_t element, size_t bytes) {
    return reinterpret_cast<uintptr_t>(a.data) % bytes == 0 && (rows <= 1 || a.stride * element % bytes == 0);
}

// Elements that are taken at a time: 16 bytes, two elements (even strides that are no multiple of that), or one.  Two
// elements are half the instructions of one: 8192 x 4090 bfloat16, layer norm 39 us against 62, the residual form 71
// against 120.
template <typename T>
int pack_of(std::initializer_list<const RowArray*> arrays, long long rows) {
    for (const int pack : {(int)(16 / sizeof(T)), 2}) {
        bool all = true;
        for (const RowArray* a : arrays) all = all && rows_aligned(*a, rows, sizeof(T), pack * sizeof(T));
        if (all) return pack;
    }
    return 1;
}

template <typename... P, typename... Q>
cudaError_t launch_rows(void (*kernel)(P...), unsigned grid, unsigned threads, size_t shared, int cluster, cudaStream_t stream,
                        const Q&... args) {
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

template <typename T, int V, bool RESIDUAL>
cudaError_t launch_forward(NormForwardArgs a, cudaStream_t stream) {
    const RowShape s = row_shape(a.cols, norm_elements(sizeof(T)));
    constexpr bool WIDE = V * sizeof(T) == 16;
    const int threads = s.threads_per_row * s.groups, together = s.groups * norm_forward_rows(sizeof(T), WIDE);
    const long long batches = (a.rows + together - 1) / together, resident = NORM_SMS * (NORM_MAX_THREADS / threads) / s.cluster;
    const long long clusters = std::min(batches, resident);
    for (RowArray* r : {&a.x, &a.residual, &a.h, &a.y}) r->advance = clusters * together * r->stride;
    auto kernel = s.threads_per_row >= 32 ? norm_forward_kernel<T, V, 32, RESIDUAL> : norm_forward_kernel<T, V, 0, RESIDUAL>;
    const size_t each = norm_forward_shared(sizeof(T), WIDE, RESIDUAL);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(each * NORM_MAX_THREADS));
    return e != cudaSuccess ? e : launch_rows(kernel, (unsigned)(clusters * s.cluster), threads, each * threads, s.cluster, stream, a, s);
}

template <typename T, bool RESIDUAL>
cudaError_t launch_forward(const NormForwardArgs& a, cudaStream_t stream) {
    constexpr int WIDE = 16 / sizeof(T);
    const int pack = pack_of<T>({&a.x, &a.residual, &a.h, &a.y}, a.rows);
    if (pack == WIDE) return launch_forward<T, WIDE, RESIDUAL>(a, stream);
    if constexpr (WIDE > 2)
        if (pack == 2) return launch_forward<T, 2, RESIDUAL>(a, stream);
    return launch_forward<T, 1, RESIDUAL>(a, stream);
}

template <typename T>
cudaError_t norm_forward_launch(const NormForwardArgs& a, cudaStream_t stream) {
    const bool residual = a.residual.data != nullptr || a.h.data != nullptr || a.draw.active;
    return residual ? launch_forward<T, true>(a, stream) : launch_forward<T, false>(a, stream);
}

template <typename T, int V, bool RESIDUAL>
cudaError_t launch_backward(NormBackwardArgs a, cudaStream_t stream) {
    using A = typename Accumulator<T>::type;
    const RowShape s = row_shape(a.cols, norm_elements(sizeof(T)));
    constexpr bool WIDE = V * sizeof(T) == 16;
    const bool whole_warps = s.threads_per_row >= 32;
    const int threads = s.threads_per_row * s.groups, rows_at_once = norm_backward_rows(sizeof(T), WIDE, whole_warps);
    const int partials = norm_partials(a.rows, rows_at_once, s);
    for (RowArray* r : {&a.dy, &a.dh, &a.h, &a.dx, &a.dresidual}) r->advance = (long long)partials * s.groups * rows_at_once * r->stride;
    auto kernel = whole_warps ? norm_backward_kernel<T, V, 32, RESIDUAL> : norm_backward_kernel<T, V, 0, RESIDUAL>;
    // The ring's space later holds the groups' shares of the parameters' gradients: two values for each element.
    const size_t each = std::max(norm_backward_shared(sizeof(T), WIDE, whole_warps, RESIDUAL), 2 * norm_elements(sizeof(T)) * sizeof(A));
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(each * NORM_MAX_THREADS));
    if (e == cudaSuccess) e = launch_rows(kernel, (unsigned)(partials * s.cluster), threads, each * threads, s.cluster, stream, a, s);
    if (e != cudaSuccess || partials == 1 || (a.dweight == nullptr && a.dbias == nullptr)) return e;
    cudaLaunchConfig_t config{};
    constexpr int W = 16 / sizeof(A);
    const bool vectors = a.cols % W == 0;
    const int columns = vectors ? 8 * W : 8;
    config.gridDim = dim3((a.cols + columns - 1) / columns, 2);
    config.blockDim = dim3(256);
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, vectors ? norm_join_kernel<T, W> : norm_join_kernel<T, 1>, a, partials);
}

template <typename T, bool RESIDUAL>
cudaError_t launch_backward(const NormBackwardArgs& a, cudaStream_t stream) {
    constexpr int WIDE = 16 / sizeof(T);
    const int pack = pack_of<T>({&a.dy, &a.dh, &a.h, &a.dx, &a.dresidual}, a.rows);
    if (pack == WIDE) return launch_backward<T, WIDE, RESIDUAL>(a, stream);
    if constexpr (WIDE > 2)
        if (pack == 2) return launch_backward<T, 2, RESIDUAL>(a, stream);
    return launch_backward<T, 1, RESIDUAL>(a, stream);
}

template <typename T>
cudaError_t norm_backward_launch(const NormBackwardArgs& a, cudaStream_t stream) {
    const bool residual = a.dh.data != nullptr || a.dresidual.data != nullptr || a.draw.active;
    return residual ? launch_backward<T, true>(a, stream) : launch_backward<T, false>(a, stream);
}

template <typename T>
cudaError_t dropout_launch(const DropoutArgs& given, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    DropoutArgs a = given;
    if (a.x.stride == a.cols && a.y.stride == a.cols) {  // rows that follow on each other are one long row
        a.cols *= a.rows;
        a.rows = 1;
    }
    const bool wide = (reinterpret_cast<uintptr_t>(a.x.data) - reinterpret_cast<uintptr_t>(a.y.data)) % 16 == 0 &&
                      (a.rows <= 1 || (a.x.stride - a.y.stride) * (long long)sizeof(T) % 16 == 0);
    const long long per_row = wide ? (a.cols + V - 1) / V + 1 : a.cols;  // one more where a row starts between boundaries
    const long long packs = per_row * a.rows, each = 256 * dropout_depth(a.rows == 1);
    // Small arrays: a pack for each thread and as many CTAs as that takes.  Large ones: 16-bit rows are bound by the integer
    // units and 8 CTAs for each SM do best (16384 x 8192 bfloat16 108 us, with 24 119), others by memory and 24 (8192 x 8192
    // float32 86 us, with 8 95).
    const long long spread = (packs + 255) / 256, deep = (packs + each - 1) / each;
    const long long most = NORM_SMS * (sizeof(T) == 2 && a.rows == 1 ? 8 : 24), least = NORM_SMS * 4;
    const unsigned grid = (unsigned)(spread <= least ? spread : std::max(least, std::min(deep, most)));
    auto kernel = a.rows == 1 ? (wide ? dropout_kernel<T, V, true> : dropout_kernel<T, 1, true>)
                              : (wide ? dropout_kernel<T, V, false> : dropout_kernel<T, 1, false>);
    return launch_rows(kernel, grid, 256, 0, 1, stream, a, packs, per_row);
}

#define QB_INSTANTIATE_NORM(T)                                                              \
    template cudaError_t norm_forward_launch<T>(const NormForwardArgs&, cudaStream_t);      \
    template cudaError_t norm_backward_launch<T>(const NormBackwardArgs&, cudaStream_t);    \
    template cudaError_t dropout_launch<T>(const DropoutArgs&, cudaStream_t);

}  // namespace qb
