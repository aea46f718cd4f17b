// Entry points of the stand-alone layer norm, dropout and their residual form: argument checks, launch on the device
// that holds the arrays.  The kernels are in norm_kernels.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <initializer_list>

#include "common.h"
#include "norm.h"

namespace {

using qb::fail;

struct Named {
    const char* name;
    const void* data;
    bool required;
};

size_t element_bytes(int32_t dtype) { return dtype == QB200_F64 ? 8 : dtype == QB200_F32 ? 4 : 2; }

// float64 rows fill half as many columns of a thread's registers.
int max_columns(int32_t dtype) {
    return qb::NORM_MAX_CLUSTER * qb::NORM_MAX_THREADS * qb::norm_elements(element_bytes(dtype));
}

qb200_status check_dtype(const char* op, int32_t dtype) {
    if (dtype < QB200_F32 || dtype > QB200_BF16) return fail(QB200_INVALID, "%s: unknown dtype %d", op, dtype);
    return QB200_OK;
}

qb200_status check_param_dtype(const char* op, int32_t dtype, int32_t param_dtype) {
    if (param_dtype == dtype || (param_dtype == QB200_F32 && element_bytes(dtype) == 2)) return QB200_OK;
    return fail(QB200_INVALID, "%s: parameters are of the rows' dtype, or float32 beside 16-bit rows; got dtype %d and param_dtype %d",
                op, dtype, param_dtype);
}

qb200_status check_extents(const char* op, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1)
        return fail(QB200_INVALID, "%s needs rows >= 0 and cols >= 1; got %lld x %lld", op, (long long)rows, (long long)cols);
    if (rows > 0 && cols > (int64_t(1) << 56) / rows)
        return fail(QB200_TOO_LARGE, "%s: %lld x %lld elements", op, (long long)rows, (long long)cols);
    return QB200_OK;
}

qb200_status check_columns(const char* op, int32_t dtype, int64_t rows, int32_t cols) {
    QB_TRY(check_extents(op, rows, cols));
    if (cols > max_columns(dtype))
        return fail(QB200_TOO_LARGE, "%s: rows of at most %d elements in this dtype, got %d", op, max_columns(dtype), cols);
    return QB200_OK;
}

// Rows that are read may overlap or repeat (stride 0 broadcasts one row); rows that are written may not.
qb200_status check_rows(const char* op, const char* name, const void* data, int64_t stride, int64_t rows, int64_t cols,
                        int32_t dtype, bool written) {
    if (data == nullptr || rows == 0) return QB200_OK;
    if (reinterpret_cast<uintptr_t>(data) % element_bytes(dtype) != 0)
        return fail(QB200_INVALID, "%s: %s is not aligned to its elements", op, name);
    if (rows > 1 && (stride < (written ? cols : 0) || stride > (int64_t(1) << 56) / rows))
        return fail(QB200_INVALID, "%s: %s has a row stride of %lld elements for %lld columns", op, name, (long long)stride,
                    (long long)cols);
    return QB200_OK;
}

qb200_status check_present(const char* op, std::initializer_list<Named> arrays) {
    for (const Named& a : arrays)
        if (a.required && a.data == nullptr) return fail(QB200_INVALID, "%s needs %s", op, a.name);
    return QB200_OK;
}

qb200_status check_aligned(const char* op, std::initializer_list<Named> arrays, size_t bytes) {
    for (const Named& a : arrays)
        if (reinterpret_cast<uintptr_t>(a.data) % bytes != 0)
            return fail(QB200_INVALID, "%s: %s is not aligned to its elements", op, a.name);
    return QB200_OK;
}

qb200_status check_epsilon(const char* op, int32_t dtype, double epsilon) {
    const double least = dtype == QB200_F64 ? 2.2250738585072014e-308 : 1.1754943508222875e-38;  // of the statistics' type
    if (!(std::isfinite(epsilon) && epsilon >= least && (dtype == QB200_F64 || epsilon <= 3.4e38)))
        return fail(QB200_INVALID, "%s: epsilon must be positive, finite and a normal number of the statistics' type; got %g", op, epsilon);
    return QB200_OK;
}

qb200_status make_draw(const char* op, double rate, uint64_t key, uint64_t counter, const uint64_t* d_counter, int64_t rows,
                       int64_t cols, qb::Draw* out) {
    if (!(rate >= 0.0 && rate < 1.0)) return fail(QB200_INVALID, "%s: rate must be in [0, 1); got %g", op, rate);
    if (reinterpret_cast<uintptr_t>(d_counter) % 8 != 0) return fail(QB200_INVALID, "%s: d_counter is not aligned to 8 bytes", op);
    if (counter > UINT64_MAX - (uint64_t)(rows * cols))
        return fail(QB200_INVALID, "%s: counter %llu leaves no room for %lld elements below 2^64", op, (unsigned long long)counter,
                    (long long)(rows * cols));
    out->key = key;
    out->counter = counter;
    out->d_counter = reinterpret_cast<const unsigned long long*>(d_counter);
    out->active = rate > 0.0;
    out->threshold = (unsigned int)std::floor(rate * 4294967296.0);
    out->scale = 1.0 / (1.0 - rate);
    return QB200_OK;
}

// Makes the device that holds `data` the current one for the time of a call.
class DeviceOf {
public:
    ~DeviceOf() {
        if (previous_ >= 0) cudaSetDevice(previous_);
    }
    qb200_status enter(const char* op, const void* data) {
        cudaPointerAttributes attributes{};
        QB_CUDA(cudaPointerGetAttributes(&attributes, data));
        if (attributes.type == cudaMemoryTypeUnregistered)
            return fail(QB200_INVALID, "%s: an array is not device memory (nor managed or page-locked)", op);
        if (attributes.type != cudaMemoryTypeDevice) return QB200_OK;
        int current = -1;
        QB_CUDA(cudaGetDevice(&current));
        if (attributes.device == current) return QB200_OK;
        QB_CUDA(cudaSetDevice(attributes.device));
        previous_ = current;
        return QB200_OK;
    }

private:
    int previous_ = -1;
};

qb200_status finish(const char* op, cudaError_t e) {
    return e == cudaSuccess ? QB200_OK : fail(QB200_CUDA_ERROR, "%s failed: %s", op, cudaGetErrorString(e));
}

#define QB_BY_DTYPE(dtype, launch, args, stream)                                    \
    ((dtype) == QB200_F32   ? qb::launch<float>(args, stream)                       \
     : (dtype) == QB200_F64 ? qb::launch<double>(args, stream)                      \
     : (dtype) == QB200_F16 ? qb::launch<__half>(args, stream)                      \
                            : qb::launch<__nv_bfloat16>(args, stream))

// An absent array's stride is not looked at, and one row's neither, whatever it is: no address is formed with it and no
// width chosen by it.  (Groups and turns without a row name a source in their copies of no bytes; it has to be aligned all
// the same.)
qb::RowArray rows_of(const void* data, int64_t stride, int64_t rows) {
    return {const_cast<void*>(data), data != nullptr && rows > 1 ? (long long)stride : 0, 0};
}

size_t workspace_bytes_for(int32_t dtype, int64_t rows, int32_t cols) {
    if (rows == 0) return 0;
    const qb::RowShape s = qb::row_shape(cols, qb::norm_elements(element_bytes(dtype)));
    return (size_t)qb::norm_partials(rows, 1, s) * 2 * (size_t)cols * (dtype == QB200_F64 ? 8 : 4);
}

qb200_status run_forward(const char* op, int32_t dtype, int32_t param_dtype, qb::NormForwardArgs& a, const void* d_weight,
                         const void* d_bias, double epsilon, void* d_mean, void* d_rstd, int64_t rows, int32_t cols,
                         void* cuda_stream) {
    QB_TRY(check_epsilon(op, dtype, epsilon));
    if (rows == 0) return QB200_OK;
    QB_TRY(check_present(op, {{"x", a.x.data, true}, {"y", a.y.data, true}}));
    QB_TRY(check_rows(op, "x", a.x.data, a.x.stride, rows, cols, dtype, false));
    QB_TRY(check_rows(op, "residual", a.residual.data, a.residual.stride, rows, cols, dtype, false));
    QB_TRY(check_rows(op, "h", a.h.data, a.h.stride, rows, cols, dtype, true));
    QB_TRY(check_rows(op, "y", a.y.data, a.y.stride, rows, cols, dtype, true));
    QB_TRY(check_aligned(op, {{"weight", d_weight, false}, {"bias", d_bias, false}}, element_bytes(param_dtype)));
    QB_TRY(check_aligned(op, {{"mean", d_mean, false}, {"rstd", d_rstd, false}}, dtype == QB200_F64 ? 8 : 4));
    a.weight = d_weight;
    a.bias = d_bias;
    a.mean = d_mean;
    a.rstd = d_rstd;
    a.epsilon = epsilon;
    a.rows = rows;
    a.cols = cols;
    a.params_f32 = param_dtype != dtype;
    DeviceOf device;
    QB_TRY(device.enter(op, a.x.data));
    return finish(op, QB_BY_DTYPE(dtype, norm_forward_launch, a, static_cast<cudaStream_t>(cuda_stream)));
}

qb200_status run_backward(const char* op, int32_t dtype, int32_t param_dtype, qb::NormBackwardArgs& a, const void* d_weight,
                          const void* d_mean, const void* d_rstd, void* d_dweight, void* d_dbias, void* d_workspace,
                          size_t workspace_bytes, int64_t rows, int32_t cols, void* cuda_stream) {
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const size_t param_bytes = element_bytes(param_dtype);
    QB_TRY(check_aligned(op, {{"weight", d_weight, false}, {"dweight", d_dweight, false}, {"dbias", d_dbias, false}}, param_bytes));
    if (rows == 0) {  // sums over no rows
        for (void* out : {d_dweight, d_dbias}) {
            if (out == nullptr) continue;
            DeviceOf device;
            QB_TRY(device.enter(op, out));
            QB_CUDA(cudaMemsetAsync(out, 0, (size_t)cols * param_bytes, stream));
        }
        return QB200_OK;
    }
    QB_TRY(check_present(op, {{"dy", a.dy.data, true}, {"the normalised rows", a.h.data, true}, {"mean", d_mean, true},
                              {"rstd", d_rstd, true}, {"dx", a.dx.data, true}}));
    QB_TRY(check_rows(op, "dy", a.dy.data, a.dy.stride, rows, cols, dtype, false));
    QB_TRY(check_rows(op, "dh", a.dh.data, a.dh.stride, rows, cols, dtype, false));
    QB_TRY(check_rows(op, "the array of normalised rows", a.h.data, a.h.stride, rows, cols, dtype, false));
    QB_TRY(check_rows(op, "dx", a.dx.data, a.dx.stride, rows, cols, dtype, true));
    QB_TRY(check_rows(op, "dresidual", a.dresidual.data, a.dresidual.stride, rows, cols, dtype, true));
    QB_TRY(check_aligned(op, {{"mean", d_mean, false}, {"rstd", d_rstd, false}}, dtype == QB200_F64 ? 8 : 4));
    if (d_dweight != nullptr || d_dbias != nullptr) {
        const size_t needed = workspace_bytes_for(dtype, rows, cols);
        if (d_workspace == nullptr || workspace_bytes < needed)
            return fail(QB200_INVALID, "%s needs a workspace of %zu bytes for %lld rows of %d, got %zu", op, needed, (long long)rows,
                        cols, d_workspace == nullptr ? (size_t)0 : workspace_bytes);
        if (reinterpret_cast<uintptr_t>(d_workspace) % 16 != 0)
            return fail(QB200_INVALID, "%s: the workspace is not aligned to 16 bytes", op);
    }
    a.weight = d_weight;
    a.mean = d_mean;
    a.rstd = d_rstd;
    a.dweight = d_dweight;
    a.dbias = d_dbias;
    a.partial = d_workspace;
    a.rows = rows;
    a.cols = cols;
    a.params_f32 = param_dtype != dtype;
    DeviceOf device;
    QB_TRY(device.enter(op, a.dy.data));
    return finish(op, QB_BY_DTYPE(dtype, norm_backward_launch, a, stream));
}

}  // namespace

extern "C" {

qb200_status qb200_layer_norm(int32_t dtype, int32_t param_dtype, const void* d_x, int64_t x_stride, int64_t rows, int32_t cols,
                              const void* d_weight, const void* d_bias, double epsilon, void* d_y, int64_t y_stride,
                              void* d_mean, void* d_rstd, void* cuda_stream) {
    const char* op = "layer_norm";
    QB_TRY(check_dtype(op, dtype));
    QB_TRY(check_param_dtype(op, dtype, param_dtype));
    QB_TRY(check_columns(op, dtype, rows, cols));
    qb::NormForwardArgs a;
    a.x = rows_of(d_x, x_stride, rows);
    a.y = rows_of(d_y, y_stride, rows);
    return run_forward(op, dtype, param_dtype, a, d_weight, d_bias, epsilon, d_mean, d_rstd, rows, cols, cuda_stream);
}

qb200_status qb200_dropout_layer_norm(int32_t dtype, int32_t param_dtype, const void* d_x, int64_t x_stride, const void* d_residual,
                                      int64_t residual_stride, int64_t rows, int32_t cols, double rate, uint64_t key,
                                      uint64_t counter, const uint64_t* d_counter, const void* d_weight, const void* d_bias,
                                      double epsilon, void* d_h, int64_t h_stride, void* d_y, int64_t y_stride, void* d_mean,
                                      void* d_rstd, void* cuda_stream) {
    const char* op = "dropout_layer_norm";
    QB_TRY(check_dtype(op, dtype));
    QB_TRY(check_param_dtype(op, dtype, param_dtype));
    QB_TRY(check_columns(op, dtype, rows, cols));
    qb::NormForwardArgs a;
    QB_TRY(make_draw(op, rate, key, counter, d_counter, rows, cols, &a.draw));
    a.x = rows_of(d_x, x_stride, rows);
    a.residual = rows_of(d_residual, residual_stride, rows);
    a.h = rows_of(d_h, h_stride, rows);
    a.y = rows_of(d_y, y_stride, rows);
    return run_forward(op, dtype, param_dtype, a, d_weight, d_bias, epsilon, d_mean, d_rstd, rows, cols, cuda_stream);
}

qb200_status qb200_layer_norm_workspace(int32_t dtype, int64_t rows, int32_t cols, size_t* nbytes) {
    const char* op = "layer_norm_workspace";
    QB_TRY(check_dtype(op, dtype));
    QB_TRY(check_columns(op, dtype, rows, cols));
    if (nbytes == nullptr) return fail(QB200_INVALID, "%s needs an output", op);
    *nbytes = workspace_bytes_for(dtype, rows, cols);
    return QB200_OK;
}

qb200_status qb200_layer_norm_backward(int32_t dtype, int32_t param_dtype, const void* d_dy, int64_t dy_stride, const void* d_x,
                                       int64_t x_stride, int64_t rows, int32_t cols, const void* d_weight, const void* d_mean,
                                       const void* d_rstd, void* d_dx, int64_t dx_stride, void* d_dweight, void* d_dbias,
                                       void* d_workspace, size_t workspace_bytes, void* cuda_stream) {
    const char* op = "layer_norm_backward";
    QB_TRY(check_dtype(op, dtype));
    QB_TRY(check_param_dtype(op, dtype, param_dtype));
    QB_TRY(check_columns(op, dtype, rows, cols));
    qb::NormBackwardArgs a;
    a.dy = rows_of(d_dy, dy_stride, rows);
    a.h = rows_of(d_x, x_stride, rows);
    a.dx = rows_of(d_dx, dx_stride, rows);
    return run_backward(op, dtype, param_dtype, a, d_weight, d_mean, d_rstd, d_dweight, d_dbias, d_workspace, workspace_bytes, rows,
                        cols, cuda_stream);
}

qb200_status qb200_dropout_layer_norm_backward(int32_t dtype, int32_t param_dtype, const void* d_dy, int64_t dy_stride,
                                               const void* d_dh, int64_t dh_stride, const void* d_h, int64_t h_stride,
                                               int64_t rows, int32_t cols, const void* d_weight, const void* d_mean,
                                               const void* d_rstd, double rate, uint64_t key, uint64_t counter,
                                               const uint64_t* d_counter, void* d_dx, int64_t dx_stride, void* d_dresidual,
                                               int64_t dresidual_stride, void* d_dweight, void* d_dbias, void* d_workspace,
                                               size_t workspace_bytes, void* cuda_stream) {
    const char* op = "dropout_layer_norm_backward";
    QB_TRY(check_dtype(op, dtype));
    QB_TRY(check_param_dtype(op, dtype, param_dtype));
    QB_TRY(check_columns(op, dtype, rows, cols));
    qb::NormBackwardArgs a;
    QB_TRY(make_draw(op, rate, key, counter, d_counter, rows, cols, &a.draw));
    a.dy = rows_of(d_dy, dy_stride, rows);
    a.dh = rows_of(d_dh, dh_stride, rows);
    a.h = rows_of(d_h, h_stride, rows);
    a.dx = rows_of(d_dx, dx_stride, rows);
    a.dresidual = rows_of(d_dresidual, dresidual_stride, rows);
    return run_backward(op, dtype, param_dtype, a, d_weight, d_mean, d_rstd, d_dweight, d_dbias, d_workspace, workspace_bytes, rows,
                        cols, cuda_stream);
}

qb200_status qb200_dropout(int32_t dtype, const void* d_x, int64_t x_stride, int64_t rows, int64_t cols, double rate, uint64_t key,
                           uint64_t counter, const uint64_t* d_counter, void* d_y, int64_t y_stride, void* cuda_stream) {
    const char* op = "dropout";
    QB_TRY(check_dtype(op, dtype));
    QB_TRY(check_extents(op, rows, cols));
    qb::DropoutArgs a;
    QB_TRY(make_draw(op, rate, key, counter, d_counter, rows, cols, &a.draw));
    if (rows == 0) return QB200_OK;
    QB_TRY(check_present(op, {{"x", d_x, true}, {"y", d_y, true}}));
    QB_TRY(check_rows(op, "x", d_x, x_stride, rows, cols, dtype, false));
    QB_TRY(check_rows(op, "y", d_y, y_stride, rows, cols, dtype, true));
    a.x = rows_of(d_x, x_stride, rows);
    a.y = rows_of(d_y, y_stride, rows);
    a.rows = rows;
    a.cols = cols;
    DeviceOf device;
    QB_TRY(device.enter(op, d_x));
    return finish(op, QB_BY_DTYPE(dtype, dropout_launch, a, static_cast<cudaStream_t>(cuda_stream)));
}

}  // extern "C"
