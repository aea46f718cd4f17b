// Arguments and launch shapes of the stand-alone layer norm, dropout and residual-form kernels, shared by the entry
// points (norm.cu) and the kernels' translation units (norm_f32.cu, norm_f64.cu, norm_f16.cu, norm_bf16.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "draws.cuh"

namespace qb {

struct RowArray {
    void* data = nullptr;
    long long stride = 0;   // elements between rows
    long long advance = 0;  // elements from a thread's row to its next one
};

struct NormForwardArgs {
    RowArray x, residual, h, y;  // residual and h may be absent
    const void* weight = nullptr;
    const void* bias = nullptr;
    void* mean = nullptr;
    void* rstd = nullptr;
    double epsilon = 0.0;
    Draw draw;
    long long rows = 0;
    int cols = 0;
    bool params_f32 = false;  // weight and bias are float32 beside 16-bit rows
};

struct NormBackwardArgs {
    RowArray dy, dh, h, dx, dresidual;  // dh and dresidual may be absent
    const void* weight = nullptr;
    const void* mean = nullptr;
    const void* rstd = nullptr;
    void* dweight = nullptr;
    void* dbias = nullptr;
    void* partial = nullptr;  // [partials][2][cols] in the accumulation type
    Draw draw;
    long long rows = 0;
    int cols = 0;
    bool params_f32 = false;
};

struct DropoutArgs {
    RowArray x, y;
    Draw draw;
    long long rows = 0;
    long long cols = 0;
};

// Elements of a row that one thread keeps in registers.
__host__ __device__ constexpr int norm_elements(size_t element_bytes) { return element_bytes == 8 ? 8 : 16; }
// Rows that a group works on at once.  16-bit rows that come 16 bytes at a time are bound by instruction issue: two
// rows share a turn's reductions, barrier and addresses.
__host__ __device__ constexpr int norm_forward_rows(size_t element_bytes, bool wide) { return element_bytes == 2 && wide ? 2 : 1; }
// Rows that share a warp have no barrier to share and are worked on one at a time in the backward pass, whose registers
// two would not fit (262144 x 128 bfloat16 42 us, with two 50).
__host__ __device__ constexpr int norm_backward_rows(size_t element_bytes, bool wide, bool whole_warps) {
    return element_bytes == 2 && wide && whole_warps ? 2 : 1;
}
// Turns whose rows are on their way or in work in a thread's slots: as many as 512 threads' slots fit beside each other for
// the backward pass; forward, two rows at once take three turns (8192 x 4096 bfloat16 26.7 us, with two 28.7).
__host__ __device__ constexpr int norm_forward_stages(size_t element_bytes, bool wide, bool residual) {
    return residual || norm_forward_rows(element_bytes, wide) == 2 ? 3 : 4;
}
__host__ __device__ constexpr int norm_backward_stages(bool residual) { return residual ? 2 : 3; }
// Bytes of a thread's slots.
constexpr size_t norm_forward_shared(size_t element_bytes, bool wide, bool residual) {
    return norm_forward_stages(element_bytes, wide, residual) * norm_forward_rows(element_bytes, wide) * (residual ? 2 : 1) *
           norm_elements(element_bytes) * element_bytes;
}
constexpr size_t norm_backward_shared(size_t element_bytes, bool wide, bool whole_warps, bool residual) {
    return norm_backward_stages(residual) * norm_backward_rows(element_bytes, wide, whole_warps) * (residual ? 3 : 2) *
           norm_elements(element_bytes) * element_bytes;
}
constexpr int NORM_MAX_THREADS = 512;  // at the kernels' 128 registers, what an SM holds
constexpr int NORM_MAX_CLUSTER = 8;
constexpr int NORM_SMS = 148;

// How the rows of an array are laid over threads: `threads_per_row` threads of each of `cluster` CTAs hold a row
// (columns [rank * slice, (rank + 1) * slice) in CTA `rank`), `groups` rows at once in a CTA.  A row is spread over CTAs
// only where one cannot hold it: a cluster's sums cost more than its warps bring (8192 x 8192 bfloat16 forward 57 us in one
// CTA, 82 in two).
struct RowShape {
    int threads_per_row, groups, cluster, slice;
};

inline RowShape row_shape(int cols, int elements) {
    RowShape s{};
    const int capacity = NORM_MAX_THREADS * elements;
    s.cluster = 1;
    while (s.cluster * capacity < cols) s.cluster *= 2;
    s.slice = ((cols + s.cluster - 1) / s.cluster + elements - 1) / elements * elements;
    const int needed = s.slice / elements;
    if (needed <= 32) {
        s.threads_per_row = 1;
        while (s.threads_per_row < needed) s.threads_per_row *= 2;
    } else {
        s.threads_per_row = (needed + 31) / 32 * 32;
    }
    s.groups = s.threads_per_row >= 256 ? 1 : 256 / s.threads_per_row;
    return s;
}

// Rows of partial weight gradients that a backward pass leaves (one per cluster of CTAs); the most with one row at once.
inline int norm_partials(long long rows, int rows_at_once, const RowShape& s) {
    const int together = s.groups * rows_at_once;
    const long long batches = (rows + together - 1) / together;
    const int resident = NORM_SMS * (s.threads_per_row * s.groups <= 256 ? 2 : 1) / s.cluster;
    return (int)(batches < resident ? batches : resident);
}

template <typename T> cudaError_t norm_forward_launch(const NormForwardArgs& a, cudaStream_t stream);
template <typename T> cudaError_t norm_backward_launch(const NormBackwardArgs& a, cudaStream_t stream);
template <typename T> cudaError_t dropout_launch(const DropoutArgs& a, cudaStream_t stream);

}  // namespace qb
