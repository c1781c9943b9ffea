// Host entry points of the NVFP4 linear with its epilogue and of its grouped
// form (linear_fused.cuh has the formula), and the upload of grouped weights.
#include "linear_fused.cuh"

#include <climits>
#include <memory>
#include <vector>

namespace nvfp4 {
namespace {

// Scale rows at their device pitch, sanitised as at every other upload (sign
// cleared, 0x7F -> 0), and the inverse divisors.
__global__ void grouped_scales_kernel(uint8_t *dst, int pitch, const uint8_t *src, int row_scales, long long rows) {
    const long long n = rows * pitch;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / pitch;
        const int c = (int)(i - r * pitch);
        const uint8_t b = c < row_scales ? src[r * row_scales + c] & 0x7Fu : 0;
        dst[i] = b == 0x7Fu ? 0u : b;
    }
}

__global__ void inverse_kernel(float *v, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) v[i] = 1.0f / v[i];
}

struct device_memory {
    void *p = nullptr;
    ~device_memory() {
        if (p) cudaFree(p);
    }
};

bool valid_type(int type) { return type == NVFP4_TYPE_BF16 || type == NVFP4_TYPE_F16 || type == NVFP4_TYPE_F32; }

bool aligned_to_type(const void *p, int type) {
    return (reinterpret_cast<uintptr_t>(p) & (type == NVFP4_TYPE_F32 ? 3u : 1u)) == 0;
}

// The call's arguments, or the message of the check that failed.
const char *fused_args(FusedLinearArgs &a, const nvfp4_runtime *runtime, const nvfp4_matrix *matrix, const void *x,
                       int type, int64_t x_stride, int vectors, const void *bias, int bias_type, int activation,
                       void *out, int64_t out_stride) {
    if (!runtime || !matrix || matrix->runtime != runtime || !x || !out || vectors <= 0 || !valid_type(type))
        return "invalid linear arguments or mismatched runtime/matrix";
    if (vectors > (1 << 30)) return "linear: at most 2^30 rows of x";
    const int act = activation & ~NVFP4_ACT_GATED;
    const bool gated = (activation & NVFP4_ACT_GATED) != 0;
    if (act < NVFP4_ACT_NONE || act > NVFP4_ACT_GELU_TANH) return "unknown activation";
    if (gated && matrix->rows % 2 != 0) return "a gated activation needs an even number of weight rows";
    if (bias && !valid_type(bias_type)) return "unknown bias type";
    a.out_rows = gated ? matrix->rows / 2 : matrix->rows;
    if (x_stride < 0 || out_stride < a.out_rows) return "invalid row stride";
    if (!aligned_to_type(x, type) || !aligned_to_type(out, type) || (bias && !aligned_to_type(bias, bias_type)))
        return "linear arguments must be aligned to their elements";
    const long long e = type == NVFP4_TYPE_F32 ? 4 : 2;
    if (spans_overlap({x, vectors, matrix->cols * e, x_stride * e}, {out, vectors, a.out_rows * e, out_stride * e}))
        return "linear: out must not overlap x";
    a.packed = matrix->packed;
    a.scales = matrix->scales;
    a.packed_pitch = matrix->packed_pitch;
    a.scale_pitch = matrix->scale_pitch;
    a.inv_globals = matrix->inv_globals;
    a.inv_global = matrix->inv_global;
    a.groups = matrix->groups;
    a.rows = matrix->rows;
    a.cols = matrix->cols;
    a.x = x;
    a.x_stride = x_stride;
    a.type = type;
    a.vectors = vectors;
    a.bias = bias;
    a.bias_type = bias_type;
    a.act = act;
    a.gated = gated ? 1 : 0;
    a.out = out;
    a.out_stride = out_stride;
    a.err = matrix->tc.err;
    a.host_err = matrix->tc.host_err_dev;
    return nullptr;
}

nvfp4_status run_fused(nvfp4_runtime *runtime, const nvfp4_matrix *matrix, const FusedLinearArgs &a, void *workspace,
                       size_t workspace_bytes, void *stream, const char *operation) {
    const bool few = linear_gemv_serves(a);
    const size_t needed = few ? 0 : linear_gemm_workspace(a.type, a.x, a.x_stride, a.vectors, a.cols);
    if (needed && (!workspace || workspace_bytes < needed))
        return fail_invalid("the linear's workspace is missing or too small (nvfp4_linear_workspace_bytes)");
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail_invalid("the linear's workspace must be 256-byte aligned");
    try {
        const device_scope scope(runtime);
        check_on_device(runtime, {a.x, a.out}, operation);
        std::lock_guard<std::mutex> lock(runtime->queue_mutex);
        runtime->direct_call(static_cast<cudaStream_t>(stream), [&](cudaStream_t os) {
            runtime->profiled_kernel(operation, os, [&](cudaStream_t s) {
                if (few) launch_linear_gemv(a, runtime->device, runtime->sm_count, s);
                else launch_linear_gemm(a, *matrix, workspace, runtime->sm_count, s);
            });
        });
        clear_last_error();
        return NVFP4_STATUS_OK;
    } catch (const std::exception &error) {
        return fail_exception(error);
    }
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" NVFP4_API nvfp4_status nvfp4_matrix_upload_grouped(nvfp4_runtime *runtime, const void *packed,
                                                              size_t packed_bytes, const void *scales_e4m3,
                                                              size_t scale_bytes, const float *divisors, int groups,
                                                              int rows, int cols, nvfp4_matrix **out_matrix) {
    if (!runtime || !packed || !scales_e4m3 || !divisors || !out_matrix || rows <= 0 || cols <= 0 || cols % 16 != 0)
        return fail_invalid("invalid native NVFP4 matrix arguments");
    if (groups < 1 || groups > kLinMaxGroups) return fail_invalid("a grouped NVFP4 matrix holds 1 to 1024 groups");
    if (cols > kLinMaxCols) return fail_invalid("NVFP4 linear supports at most 49152 columns on this backend");
    const long long all_rows = static_cast<long long>(groups) * rows;
    if (all_rows > INT_MAX - 4096) return fail_invalid("NVFP4 matrix has too many rows");
    const size_t row_packed = static_cast<size_t>(cols / 2), row_scales = static_cast<size_t>(cols / 16);
    if (packed_bytes != static_cast<size_t>(all_rows) * row_packed ||
        scale_bytes != static_cast<size_t>(all_rows) * row_scales)
        return fail_invalid("packed/scales byte counts do not match groups, rows and cols");
    *out_matrix = nullptr;
    try {
        const device_scope scope(runtime);
        auto m = std::make_unique<nvfp4_matrix>();
        m->runtime = runtime;
        m->groups = groups;
        m->rows = rows;
        m->cols = cols;
        m->packed_pitch = packed_pitch_of(cols);
        m->scale_pitch = static_cast<int>((row_scales + 15) / 16 * 16);
        const size_t packed_total = static_cast<size_t>(all_rows) * m->packed_pitch;
        std::lock_guard<std::mutex> lock(runtime->queue_mutex);
        cudaStream_t s = runtime->stream;
        std::vector<float> divisor(groups);
        check_cuda(cudaMemcpyAsync(divisor.data(), divisors, sizeof(float) * groups, cudaMemcpyDefault, s),
                   "cudaMemcpyAsync(divisors)");
        check_cuda(cudaStreamSynchronize(s), "cudaStreamSynchronize(divisors)");
        for (float d : divisor)
            if (d == 0.0f) throw invalid_argument_error("a divisor of a grouped NVFP4 matrix is zero");
        device_memory raw;
        check_cuda(cudaMalloc(&m->packed, packed_total), "cudaMalloc(matrix packed)");
        check_cuda(cudaMalloc(&m->scales, static_cast<size_t>(all_rows) * m->scale_pitch), "cudaMalloc(matrix scales)");
        check_cuda(cudaMalloc(&m->inv_globals, sizeof(float) * groups), "cudaMalloc(matrix divisors)");
        check_cuda(cudaMalloc(&m->tc.err, sizeof(int)), "cudaMalloc(matrix error word)");
        check_cuda(cudaMalloc(&raw.p, scale_bytes), "cudaMalloc(matrix scale staging)");
        if (static_cast<size_t>(m->packed_pitch) != row_packed)
            check_cuda(cudaMemsetAsync(m->packed, 0, packed_total, s), "cudaMemsetAsync(matrix packed)");
        check_cuda(cudaMemcpy2DAsync(m->packed, m->packed_pitch, packed, row_packed, row_packed, all_rows,
                                     cudaMemcpyDefault, s),
                   "cudaMemcpy2DAsync(matrix packed)");
        check_cuda(cudaMemcpyAsync(raw.p, scales_e4m3, scale_bytes, cudaMemcpyDefault, s),
                   "cudaMemcpyAsync(matrix scales)");
        check_cuda(cudaMemcpyAsync(m->inv_globals, divisors, sizeof(float) * groups, cudaMemcpyDefault, s),
                   "cudaMemcpyAsync(matrix divisors)");
        check_cuda(cudaMemsetAsync(m->tc.err, 0, sizeof(int), s), "cudaMemsetAsync(matrix error word)");
        grouped_scales_kernel<<<runtime->sm_count * 8, 256, 0, s>>>(m->scales, m->scale_pitch,
                                                                   static_cast<const uint8_t *>(raw.p),
                                                                   static_cast<int>(row_scales), all_rows);
        check_cuda(cudaGetLastError(), "grouped_scales_kernel");
        inverse_kernel<<<1, 256, 0, s>>>(m->inv_globals, groups);
        check_cuda(cudaGetLastError(), "inverse_kernel");
        make_matrix_maps(*m);
        int *host_err = nullptr;
        check_cuda(cudaHostAlloc(reinterpret_cast<void **>(&host_err), sizeof(int), cudaHostAllocMapped),
                   "cudaHostAlloc(matrix error word)");
        m->host_err = host_err;
        *host_err = 0;
        check_cuda(cudaHostGetDevicePointer(reinterpret_cast<void **>(&m->tc.host_err_dev), host_err, 0),
                   "cudaHostGetDevicePointer(matrix error word)");
        check_cuda(cudaStreamSynchronize(s), "cudaStreamSynchronize(matrix upload)");
        runtime->error_words.emplace_back(m->host_err, m->tc.err);
        *out_matrix = m.release();
        clear_last_error();
        return NVFP4_STATUS_OK;
    } catch (const std::exception &error) {
        return fail_exception(error);
    }
}

extern "C" NVFP4_API size_t nvfp4_linear_workspace_bytes(const nvfp4_matrix *matrix, const void *x, int type,
                                                         int64_t x_stride, int vectors, int grouped) {
    if (!matrix || !valid_type(type) || vectors <= 0) return 0;
    FusedLinearArgs a{};
    a.type = type;
    a.vectors = vectors;
    a.cols = matrix->cols;
    a.groups = matrix->groups;
    static const int any = 0;
    a.offsets = grouped ? &any : nullptr;  // only whether there are offsets counts here
    if (linear_gemv_serves(a)) return 0;
    return linear_gemm_workspace(type, x, x_stride, vectors, matrix->cols);
}

extern "C" NVFP4_API nvfp4_status nvfp4_linear_fused(nvfp4_runtime *runtime, const nvfp4_matrix *matrix, const void *x,
                                                     int type, int64_t x_stride, int vectors, const void *bias,
                                                     int bias_type, int activation, const void *residual,
                                                     int64_t residual_stride, void *out, int64_t out_stride,
                                                     void *workspace, size_t workspace_bytes, void *stream) {
    FusedLinearArgs a{};
    if (const char *message = fused_args(a, runtime, matrix, x, type, x_stride, vectors, bias, bias_type, activation,
                                         out, out_stride))
        return fail_invalid(message);
    if (matrix->groups != 1) return fail_invalid("a matrix of several groups runs through nvfp4_linear_grouped");
    if (residual && (residual_stride < 0 || !aligned_to_type(residual, type)))
        return fail_invalid("invalid residual stride or alignment");
    const long long e = type == NVFP4_TYPE_F32 ? 4 : 2;
    if (residual && !(residual == out && (residual_stride == out_stride || vectors == 1)) &&
        spans_overlap({residual, vectors, a.out_rows * e, residual_stride * e},
                      {out, vectors, a.out_rows * e, out_stride * e}))
        return fail_invalid("linear: the residual is out itself or does not overlap it");
    a.residual = residual;
    a.residual_stride = residual_stride;
    return run_fused(runtime, matrix, a, workspace, workspace_bytes, stream, "linear_fused");
}

extern "C" NVFP4_API nvfp4_status nvfp4_linear_grouped(nvfp4_runtime *runtime, const nvfp4_matrix *matrix,
                                                       const void *x, int type, int64_t x_stride, int vectors,
                                                       const int32_t *offsets, const void *bias, int bias_type,
                                                       int activation, void *out, int64_t out_stride, int zero_rest,
                                                       void *workspace, size_t workspace_bytes, void *stream) {
    FusedLinearArgs a{};
    if (const char *message = fused_args(a, runtime, matrix, x, type, x_stride, vectors, bias, bias_type, activation,
                                         out, out_stride))
        return fail_invalid(message);
    if (!offsets || (reinterpret_cast<uintptr_t>(offsets) & 3u)) return fail_invalid("grouped linear needs offsets");
    a.offsets = offsets;
    a.zero_rest = zero_rest != 0;
    return run_fused(runtime, matrix, a, workspace, workspace_bytes, stream, "linear_grouped");
}
