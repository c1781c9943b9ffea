// The resident NVFP4 weights behind nvfp4_matrix handles, shared by the
// linear entry points (linear.cu: dense FP32; linear_fused.cu: epilogues and
// groups).
#pragma once

#include "internal.h"
#include "linear_tc.cuh"
#include "tma_util.cuh"

struct nvfp4_matrix {
    nvfp4_runtime *runtime = nullptr;
    int groups = 1;        // weight matrices of the same shape, one after the other
    int rows = 0;          // per group
    int cols = 0;
    int packed_pitch = 0;  // bytes per packed row (multiple of 32: one load of a lane)
    int scale_pitch = 0;   // bytes per scale row (multiple of 16)
    uint8_t *packed = nullptr;   // [groups * rows][packed_pitch]
    uint8_t *scales = nullptr;   // [groups * rows][scale_pitch]
    float inv_global = 0.0f;     // of a matrix uploaded on its own
    float *inv_globals = nullptr;          // device [groups], of a grouped upload (NULL otherwise)
    nvfp4::LinearTcState tc;               // FP32 tensor-core path (not of a grouped upload): scale atoms, terms, maps
    CUtensorMap map_w;                     // packed rows: box 128 B x 64 rows, 128-byte swizzle (linear_gemm.cu)
    CUtensorMap map_s;                     // scale rows: box 16 B x 64 rows
    volatile int *host_err = nullptr;      // pinned, device-mapped wait-timeout word (read at synchronize)

    // Whether nvfp4_linear_* (FP32, no epilogue) can run it.
    bool has_terms() const { return tc.w_atoms != nullptr; }

    ~nvfp4_matrix() {
        nvfp4::free_linear_tc(tc);
        if (host_err) cudaFreeHost(const_cast<int *>(host_err));
        if (packed) cudaFree(packed);
        if (scales) cudaFree(scales);
        if (inv_globals) cudaFree(inv_globals);
    }
};

namespace nvfp4 {

constexpr int kLinMaxCols = 49152;

inline int packed_pitch_of(int cols) { return (cols / 2 + 31) / 32 * 32; }

// The tensor maps of a matrix whose arrays are allocated.
inline void make_matrix_maps(nvfp4_matrix &m) {
    const uint64_t rows = static_cast<uint64_t>(m.groups) * m.rows;
    check_cuda(make_tensor_map_u8(&m.map_w, m.packed, m.packed_pitch, m.packed_pitch, rows, 128, 64,
                                  CU_TENSOR_MAP_SWIZZLE_128B),
               "cuTensorMapEncodeTiled(packed)");
    check_cuda(make_tensor_map_u8(&m.map_s, m.scales, m.scale_pitch, m.scale_pitch, rows, 16, 64,
                                  CU_TENSOR_MAP_SWIZZLE_NONE),
               "cuTensorMapEncodeTiled(scales)");
}
constexpr int kLinMaxGroups = 1024;

}  // namespace nvfp4
