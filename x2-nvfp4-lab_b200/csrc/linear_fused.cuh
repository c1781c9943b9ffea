// The NVFP4 linear with its epilogue: arguments shared by the host entry
// points (linear_fused.cu) and the two kernels (linear_gemv.cu, few rows;
// linear_gemm.cu, many).
//
//   out[v, r] = residual[v, r] + act(inv * sum_c W[r, c] x[v, c] + bias[r])
//
// and with a gate, for r < rows / 2,
//
//   out[v, r] = residual[v, r] + act(z[v, r]) * z[v, rows / 2 + r].
//
// W = E2M1 * E4M3(block) has at most six significant bits, so it is exact in
// FP16 and in BF16; products are exact and sums FP32 in both kernels.
#pragma once

#include "linear_matrix.cuh"
#include "nvfp4_common.cuh"

namespace nvfp4 {

struct FusedLinearArgs {
    const uint8_t *packed;
    const uint8_t *scales;
    int packed_pitch, scale_pitch;
    const float *inv_globals;  // device [groups], or NULL:
    float inv_global;
    int groups;
    int rows, cols;            // of a group's weights
    int out_rows;              // rows, or rows / 2 with a gate
    const void *x;
    long long x_stride;        // elements
    int type;                  // of x, residual and out
    int vectors;               // rows of x
    const int *offsets;        // device [groups + 1] row ranges of the groups, or NULL: one group of all rows
    const void *bias;          // [groups, rows] or NULL
    int bias_type;
    int act;                   // NVFP4_ACT_*, without the gate flag
    int gated;
    const void *residual;
    long long residual_stride;
    void *out;
    long long out_stride;
    int zero_rest;             // rows outside the groups' ranges get zeros
    int *err, *host_err;       // wait-timeout words of the matrix
};

__device__ __forceinline__ float load_as_f32(const void *p, int type, size_t i) {
    if (type == NVFP4_TYPE_F32) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return type == NVFP4_TYPE_F16 ? __half2float(__ushort_as_half(h)) : bf16_bits_to_f32(h);
}

// The one rounding to the output's type.
__device__ __forceinline__ void store_from_f32(void *p, int type, size_t i, float v) {
    if (type == NVFP4_TYPE_F32)
        static_cast<float *>(p)[i] = v;
    else
        static_cast<uint16_t *>(p)[i] =
            type == NVFP4_TYPE_F16 ? __half_as_ushort(__float2half_rn(v)) : f32_to_bf16_bits(v);
}

// z / (1 + exp(-u)). Of 16-bit types exp and the division are the fast ones:
// off by a few units of 2^-23 near zero and by 2e-6 of the result at z = -40,
// far below half a step of FP16 (2^-11), and zero where exp passes 2^126
// (results below 2^-119). FP32 takes the exact exp, of -|u|, so that the
// denominator stays in [1, 2], where the fast division is off by two units:
// five in all. (The exact division, a branch for each value, made 301 rows of
// 1,008 with GELU's tanh form 21.0 us; this takes 15.8, the fast exp 15.4.)
template <bool FP32>
__device__ __forceinline__ float times_sigmoid(float z, float u) {
    if constexpr (!FP32) return __fdividef(z, 1.0f + __expf(-u));
    const float e = expf(-fabsf(u));
    return __fdividef(u < 0.0f ? z * e : z, 1.0f + e);
}

template <int ACT, bool FP32>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == NVFP4_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
    if constexpr (ACT == NVFP4_ACT_SILU) return times_sigmoid<FP32>(z, z);
    // z Phi(z); erfc keeps the small tail of negative z that 1 + erf rounds away.
    if constexpr (ACT == NVFP4_ACT_GELU) return 0.5f * z * erfcf(-0.70710678118654752f * z);
    // 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v)), v = sqrt(2 / pi) (z + 0.044715 z^3).
    if constexpr (ACT == NVFP4_ACT_GELU_TANH)
        return times_sigmoid<FP32>(z, 1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
    return z;
}

template <bool FP32>
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case NVFP4_ACT_RELU: return activate<NVFP4_ACT_RELU, FP32>(z);
        case NVFP4_ACT_SILU: return activate<NVFP4_ACT_SILU, FP32>(z);
        case NVFP4_ACT_GELU: return activate<NVFP4_ACT_GELU, FP32>(z);
        case NVFP4_ACT_GELU_TANH: return activate<NVFP4_ACT_GELU_TANH, FP32>(z);
        default: return z;
    }
}

// First row and count of a group, whatever the offsets hold kept inside the call's rows.
__device__ __forceinline__ void group_range(const FusedLinearArgs &a, int g, int *first, int *count) {
    if (!a.offsets) {
        *first = 0;
        *count = a.vectors;
        return;
    }
    const int lo = min(max(__ldg(a.offsets + g), 0), a.vectors);
    *first = lo;
    *count = min(max(__ldg(a.offsets + g + 1), lo), a.vectors) - lo;
}

// Zeros to the rows before the first group's and past the last one's (the
// rows that no group owns when the offsets do not decrease).
__device__ __forceinline__ void zero_other_rows(const FusedLinearArgs &a) {
    if (!a.zero_rest || !a.offsets) return;
    const int head = min(max(__ldg(a.offsets), 0), a.vectors);
    const int tail = min(max(__ldg(a.offsets + a.groups), head), a.vectors);
    const long long n = (long long)(head + a.vectors - tail) * a.out_rows;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        long long v = i / a.out_rows;
        const long long r = i - v * a.out_rows;
        if (v >= head) v += tail - head;
        store_from_f32(a.out, a.type, (size_t)(v * a.out_stride + r), 0.0f);
    }
}

// Whether the few-row kernel takes the call (x and out need not be set).
bool linear_gemv_serves(const FusedLinearArgs &a);
void launch_linear_gemv(const FusedLinearArgs &a, int device, int sm_count, cudaStream_t stream);

// Device workspace of launch_linear_gemm for this call: 0 when the kernel can
// read x where it lies.
size_t linear_gemm_workspace(int type, const void *x, long long x_stride, int vectors, int cols);
void launch_linear_gemm(const FusedLinearArgs &a, const nvfp4_matrix &matrix, void *workspace, int sm_count,
                        cudaStream_t stream);

}  // namespace nvfp4
