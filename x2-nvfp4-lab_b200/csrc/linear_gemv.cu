// NVFP4 linear with epilogue for few rows: a weight stream.
//
// A warp owns 16 weight rows (with a gate eight gate rows and their eight up
// rows, so that a lane holds both) and 128 columns at a time: lane (g, t)
// loads 16 bytes (32 columns) of rows g and g + 8, decodes them to FP16 in
// registers (E2M1 x E4M3 is exact there) and feeds them straight into
// mma.sync m16n8k16 as the A operand; the rows of x, as FP16 in shared memory,
// are its B columns. The order of K inside an MMA is free as long as both
// operands agree: MMA i of a chunk takes columns 32 t + 4 i .. + 3 of lane t's
// 32, so that a lane's 16 bytes feed eight MMAs without a shuffle.
//
// Rows of x in FP16: FP16 as they are; BF16 scaled by a power of two per row
// (largest finite value to [2^14, 2^15)), which is exact for every element
// down to 2^-31 of the row's largest and off by less than 2^-39 of it below;
// FP32 scaled the same way as two columns, high and low half (22 bits and a
// sign, 2^-23 of an element). The scale comes back in the epilogue.
//
// Every 256 columns the MMAs' sums are added to FP32 registers: the tensor
// core rounds its running sum towards zero, which over long rows would grow
// into a bias.
//
// Bound by the weight stream (9/16 byte a weight) and, on B200, nearly as
// much by the decode: about 12 instructions per lane and eight weights. Loads
// run one batch (256 columns) ahead of the arithmetic. K is split over the
// warps of a CTA when there are too few row tiles to give every warp its own;
// their sums meet in shared memory in warp order.
#include "linear_fused.cuh"
#include "tma_util.cuh"

#include <algorithm>

namespace nvfp4 {
namespace {

constexpr int kGvThreads = 256;
constexpr int kGvWarps = kGvThreads / 32;
constexpr int kGvBatch = 2;                        // 128-column chunks loaded together
constexpr int kGvRedPitch = 20;                    // floats per column of a partial tile: conflict-free stores
constexpr size_t kGvSmem = 232448;                 // shared memory of a CTA

struct GemvArgs {
    FusedLinearArgs f;
    int chunks;       // 128-column chunks
    int tiles;        // 16-row weight tiles of a group (eight outputs each with a gate)
    int warps_k;      // warps that share a tile's columns (a power of two)
    int units;        // ceil(tiles / (warps / warps_k)): tiles a CTA takes together
    int pass_rows;    // rows of x staged at a time
    int pass_cols;    // their MMA columns (two per row for FP32)
    int token_stride; // bytes of a staged column
};

struct Batch {
    uint4 q[kGvBatch][2];
    uint16_t s[kGvBatch][2];
};

__device__ __forceinline__ float finite_abs_bits(float v) {
    const float m = fabsf(v);
    return m <= 3.402823466e38f ? m : 0.0f;  // infinities and NaN do not set the scale
}

// Eight consecutive elements of a row of x as FP32.
template <int TYPE>
__device__ __forceinline__ void load8(const FusedLinearArgs &f, long long row, int col, bool wide, float (&v)[8]) {
    const size_t at = (size_t)(row * f.x_stride + col);
    if constexpr (TYPE == NVFP4_TYPE_F32) {
        const float *p = static_cast<const float *>(f.x) + at;
        if (wide) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(f.x) + at;
        uint16_t h[8];
        if (wide) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
            memcpy(h, &w, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = __ldg(p + i);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = TYPE == NVFP4_TYPE_F16 ? __half2float(__ushort_as_half(h[i])) : bf16_bits_to_f32(h[i]);
    }
}

// Rows [row0, row0 + n) of x as FP16 columns in shared memory, and their scales.
template <int TYPE>
__device__ __forceinline__ void stage_rows(const GemvArgs &a, uint8_t *xs, uint32_t *amax, float *back, int row0, int n) {
    const FusedLinearArgs &f = a.f;
    const int oct = a.chunks * 16, valid = f.cols / 8;  // groups of eight columns, padded and real
    const bool wide = ((reinterpret_cast<uintptr_t>(f.x) | (uintptr_t)(f.x_stride * (TYPE == NVFP4_TYPE_F32 ? 4 : 2))) & 15u) == 0;
    if constexpr (TYPE != NVFP4_TYPE_F16) {
        for (int i = threadIdx.x; i < n; i += kGvThreads) amax[i] = 0u;
        __syncthreads();
        // Whole warps per (row, 32 groups): one shared-memory maximum per warp.
        const int spans = (valid + 31) / 32;
        for (int i = threadIdx.x >> 5; i < n * spans; i += kGvWarps) {
            const int r = i / spans, o = (i - r * spans) * 32 + (threadIdx.x & 31);
            float m = 0.0f;
            if (o < valid) {
                float v[8];
                load8<TYPE>(f, row0 + r, o * 8, wide, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs_bits(v[j]));
            }
            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
            if ((threadIdx.x & 31) == 0) atomicMax(amax + r, top);
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n * oct; i += kGvThreads) {
        const int r = i / oct, o = i - r * oct;
        float v[8];
        if (o < valid) {
            load8<TYPE>(f, row0 + r, o * 8, wide, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        }
        const int off = act_tile_offset(0, 0, o >> 4, (o >> 2) & 3, o & 3);
        uint32_t hi[4], lo[4];
        if constexpr (TYPE == NVFP4_TYPE_F16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) hi[j] = __half_as_ushort(__float2half_rn(v[2 * j])) |
                                               ((uint32_t)__half_as_ushort(__float2half_rn(v[2 * j + 1])) << 16);
            *reinterpret_cast<uint4 *>(xs + r * a.token_stride + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (o == 0) back[r] = 1.0f;
        } else {
            // 2^(14 - e) with e the exponent of the row's largest finite value, kept where both it and its inverse
            // are normal numbers.
            const uint32_t top = amax[r];
            const int e = top ? max((int)(top >> 23) - 127, -112) : 14;
            const float scale = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            if (o == 0) back[r] = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t h2 = 0, l2 = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const float y = v[2 * j + b] * scale;
                    const __half h = __float2half_rn(y);
                    h2 |= (uint32_t)__half_as_ushort(h) << (16 * b);
                    if constexpr (TYPE == NVFP4_TYPE_F32) {
                        const bool fin = fabsf(y) <= 65504.0f;
                        l2 |= (uint32_t)__half_as_ushort(__float2half_rn(fin ? y - __half2float(h) : 0.0f)) << (16 * b);
                    }
                }
                hi[j] = h2;
                lo[j] = l2;
            }
            if constexpr (TYPE == NVFP4_TYPE_F32) {
                *reinterpret_cast<uint4 *>(xs + (2 * r) * a.token_stride + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(xs + (2 * r + 1) * a.token_stride + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            } else {
                *reinterpret_cast<uint4 *>(xs + r * a.token_stride + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            }
        }
    }
    __syncthreads();
}

template <int NT, int TYPE>
__global__ void __launch_bounds__(kGvThreads) linear_gemv_kernel(const __grid_constant__ GemvArgs a) {
    constexpr int kCols = 8 * NT;
    extern __shared__ __align__(16) uint8_t gv_smem[];
    const FusedLinearArgs &f = a.f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int warps_k = a.warps_k, tiles_at_once = kGvWarps / warps_k;
    const int kw = warp & (warps_k - 1), wr = warp / warps_k;

    uint8_t *xs = gv_smem;
    float *red = reinterpret_cast<float *>(gv_smem + (size_t)a.pass_cols * a.token_stride);  // [2][warps][kCols][pitch]
    uint32_t *amax = reinterpret_cast<uint32_t *>(red + 2 * kGvWarps * kCols * kGvRedPitch);
    float *back = reinterpret_cast<float *>(amax + kCols);
    int *active = reinterpret_cast<int *>(back + kCols);  // [groups] groups with rows (grouped calls)
    __shared__ int warp_sum[kGvWarps];
    __shared__ int s_active;

    int n_active = 1;
    if (f.offsets) {
        // Compact list of the groups that have rows.
        const int per = (f.groups + kGvThreads - 1) / kGvThreads;
        const int g0 = min((int)threadIdx.x * per, f.groups), g1 = min(g0 + per, f.groups);
        int own = 0;
        for (int i = g0; i < g1; ++i) {
            int first, count;
            group_range(f, i, &first, &count);
            own += count > 0;
        }
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        int at = upto - own;
        for (int w = 0; w < warp; ++w) at += warp_sum[w];
        for (int i = g0; i < g1; ++i) {
            int first, count;
            group_range(f, i, &first, &count);
            if (count > 0) active[at++] = i;
        }
        if (threadIdx.x == kGvThreads - 1) s_active = at;
        __syncthreads();
        n_active = s_active;
    }

    const long long work = (long long)n_active * a.units;
    long long u = work * blockIdx.x / gridDim.x;
    const long long u_end = work * (blockIdx.x + 1) / gridDim.x;
    const int batches = ((a.chunks + warps_k - 1) / warps_k + kGvBatch - 1) / kGvBatch;
    int parity = 0;

    while (u < u_end) {
        const int ai = (int)(u / a.units);
        const int unit0 = (int)(u - (long long)ai * a.units);
        const int unit1 = (int)min((long long)a.units, unit0 + (u_end - u));
        u += unit1 - unit0;
        const int group = f.offsets ? active[ai] : 0;
        int first, count;
        group_range(f, group, &first, &count);
        const uint8_t *packed = f.packed + (size_t)group * f.rows * f.packed_pitch;
        const uint8_t *scales = f.scales + (size_t)group * f.rows * f.scale_pitch;
        const float inv = f.inv_globals ? __ldg(f.inv_globals + group) : f.inv_global;

        // Weight rows of this lane in tile `tile`, clamped to the last row (its sums are not stored).
        auto rows_of = [&](int tile, int &r0, int &r1) {
            if (f.gated) {
                r0 = min(tile * 8 + g, f.out_rows - 1);
                r1 = r0 + f.out_rows;
            } else {
                r0 = min(tile * 16 + g, f.rows - 1);
                r1 = min(tile * 16 + g + 8, f.rows - 1);
            }
        };
        auto load = [&](Batch &b, int unit, int batch) {
            int r0, r1;
            rows_of(unit * tiles_at_once + wr, r0, r1);
#pragma unroll
            for (int i = 0; i < kGvBatch; ++i) {
                const int c = (batch * kGvBatch + i) * warps_k + kw;
                const int byte = c * 64 + t * 16;
                const bool in = byte < f.packed_pitch;
                b.q[i][0] = in ? ldg_stream128(packed + (size_t)r0 * f.packed_pitch + byte) : make_uint4(0, 0, 0, 0);
                b.q[i][1] = in ? ldg_stream128(packed + (size_t)r1 * f.packed_pitch + byte) : make_uint4(0, 0, 0, 0);
                b.s[i][0] = in ? ldg_u16(scales + (size_t)r0 * f.scale_pitch + c * 8 + t * 2) : (uint16_t)0;
                b.s[i][1] = in ? ldg_u16(scales + (size_t)r1 * f.scale_pitch + c * 8 + t * 2) : (uint16_t)0;
            }
        };

        for (int v0 = 0; v0 < count; v0 += a.pass_rows) {
            const int n = min(a.pass_rows, count - v0);
            const int ncols = TYPE == NVFP4_TYPE_F32 ? 2 * n : n;
            Batch cur;
            load(cur, unit0, 0);
            __syncthreads();  // the rows staged before are no longer read
            stage_rows<TYPE>(a, xs, amax, back, first + v0, n);
            // MMA columns past the staged ones repeat the last: their sums are not stored.
            const uint8_t *bcol[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) bcol[j] = xs + min(8 * j + g, ncols - 1) * a.token_stride + t * 64;

            for (int unit = unit0; unit < unit1; ++unit, parity ^= 1) {
                float sum[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[j][i] = 0.0f;
                for (int batch = 0; batch < batches; ++batch) {
                    Batch nxt;
                    const bool more = batch + 1 < batches;
                    if (more || unit + 1 < unit1) load(nxt, more ? unit : unit + 1, more ? batch + 1 : 0);
                    float acc[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
#pragma unroll
                    for (int i = 0; i < kGvBatch; ++i) {
                        const int c = (batch * kGvBatch + i) * warps_k + kw;
                        if (c >= a.chunks) break;
                        const uint32_t s0 = e4m3x2_to_f16x2(cur.s[i][0]), s1 = e4m3x2_to_f16x2(cur.s[i][1]);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t q0 = w == 0 ? cur.q[i][0].x : w == 1 ? cur.q[i][0].y : w == 2 ? cur.q[i][0].z : cur.q[i][0].w;
                            const uint32_t q1 = w == 0 ? cur.q[i][1].x : w == 1 ? cur.q[i][1].y : w == 2 ? cur.q[i][1].z : cur.q[i][1].w;
                            const uint32_t k0 = w < 2 ? f16x2_lo_lo(s0) : f16x2_hi_hi(s0);
                            const uint32_t k1 = w < 2 ? f16x2_lo_lo(s1) : f16x2_hi_hi(s1);
                            uint32_t h0[4], h1[4];
                            e2m1x8_to_f16x8(q0, h0);
                            e2m1x8_to_f16x8(q1, h1);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                h0[e] = hmul2_u32(h0[e], k0);
                                h1[e] = hmul2_u32(h1[e], k1);
                            }
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                const uint4 b = *reinterpret_cast<const uint4 *>(bcol[j] + c * 256 + ((w ^ (t >> 1)) << 4));
                                mma_16816(acc[j], h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                                mma_16816(acc[j], h0[2], h1[2], h0[3], h1[3], b.z, b.w);
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum[j][i] += acc[j][i];
                    if (more || unit + 1 < unit1) cur = nxt;
                }

                // Partial tiles meet in shared memory; the warps of a tile share its epilogue.
                float *mine = red + ((size_t)parity * kGvWarps + warp) * kCols * kGvRedPitch;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float *p = mine + (8 * j + 2 * t) * kGvRedPitch + g;
                    p[0] = sum[j][0];
                    p[kGvRedPitch] = sum[j][1];
                    p[8] = sum[j][2];
                    p[kGvRedPitch + 8] = sum[j][3];
                }
                if (warps_k > 1) named_barrier(1 + wr, warps_k * 32);
                else __syncwarp();
                const int tile = unit * tiles_at_once + wr;
                const int per_col = f.gated ? 8 : 16;
                const float *part = red + ((size_t)parity * kGvWarps + wr * warps_k) * kCols * kGvRedPitch;
                for (int i = kw * 32 + lane; i < n * per_col; i += warps_k * 32) {
                    const int v = i / per_col, r = i - v * per_col;
                    const int row = tile * per_col + r;
                    if (row >= f.out_rows) continue;
                    const int c0 = (TYPE == NVFP4_TYPE_F32 ? 2 * v : v) * kGvRedPitch + r;
                    float z = 0.0f, z_up = 0.0f;
                    for (int k = 0; k < warps_k; ++k) {
                        const float *p = part + (size_t)k * kCols * kGvRedPitch + c0;
                        z += TYPE == NVFP4_TYPE_F32 ? p[0] + p[kGvRedPitch] : p[0];
                        if (f.gated) z_up += TYPE == NVFP4_TYPE_F32 ? p[8] + p[kGvRedPitch + 8] : p[8];
                    }
                    const float scale = inv * back[v];
                    z *= scale;
                    const size_t b0 = (size_t)group * f.rows + row;
                    if (f.bias) z += load_as_f32(f.bias, f.bias_type, b0);
                    z = activate(z, f.act);
                    if (f.gated) {
                        z_up *= scale;
                        if (f.bias) z_up += load_as_f32(f.bias, f.bias_type, b0 + f.out_rows);
                        z *= z_up;
                    }
                    const long long vec = (long long)first + v0 + v;
                    if (f.residual) z += load_as_f32(f.residual, f.type, (size_t)(vec * f.residual_stride + row));
                    store_from_f32(f.out, f.type, (size_t)(vec * f.out_stride + row), z);
                }
            }
        }
    }
    zero_other_rows(f);
}

// Shared memory besides the staged rows: partial tiles, scales, the list of groups.
size_t other_smem(const FusedLinearArgs &f, int nt) {
    return sizeof(float) * 2 * kGvWarps * 8 * nt * kGvRedPitch + 8 * 8 * nt + (f.offsets ? sizeof(int) * f.groups : 0);
}

template <int NT, int TYPE>
void launch(GemvArgs &a, int sm_count, cudaStream_t stream) {
    const size_t smem = (size_t)a.pass_cols * a.token_stride + other_smem(a.f, NT);
    check_cuda(cudaFuncSetAttribute(linear_gemv_kernel<NT, TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(smem)),
               "cudaFuncSetAttribute(linear_gemv_kernel)");
    int per_sm = 0;
    check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, linear_gemv_kernel<NT, TYPE>, kGvThreads, smem),
               "cudaOccupancyMaxActiveBlocksPerMultiprocessor(linear_gemv_kernel)");
    const long long work = (long long)a.units * (a.f.offsets ? std::min(a.f.groups, a.f.vectors) : 1);
    const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>(work, (long long)sm_count * std::max(1, per_sm))));
    linear_gemv_kernel<NT, TYPE><<<grid, kGvThreads, smem, stream>>>(a);
    check_cuda(cudaGetLastError(), "linear_gemv_kernel");
}

template <int TYPE>
void launch_type(GemvArgs &a, int nt, int sm_count, cudaStream_t stream) {
    if (nt == 1) launch<1, TYPE>(a, sm_count, stream);
    else if (nt == 2) launch<2, TYPE>(a, sm_count, stream);
    else launch<4, TYPE>(a, sm_count, stream);
}

}  // namespace

void launch_linear_gemv(const FusedLinearArgs &f, int sm_count, cudaStream_t stream) {
    GemvArgs a{};
    a.f = f;
    a.chunks = (f.cols + 127) / 128;
    a.tiles = f.gated ? (f.out_rows + 7) / 8 : (f.rows + 15) / 16;
    a.token_stride = act_tile_stride_bytes(a.chunks * 128);
    const int per_row = f.type == NVFP4_TYPE_F32 ? 2 : 1;
    // Columns of the MMAs: enough for the call's rows, at most 32; as many staged rows as shared memory holds.
    auto fit = [&](int nt) { return static_cast<int>((kGvSmem - other_smem(f, nt)) / a.token_stride) / per_row; };
    const int want = f.offsets ? std::max(1, (f.vectors + f.groups - 1) / f.groups * 2) : f.vectors;
    int nt = 1;
    while (nt < 4 && 8 * nt / per_row < want && fit(2 * nt) > 8 * nt / per_row) nt *= 2;
    a.pass_rows = std::max(1, std::min({8 * nt / per_row, fit(nt), f.vectors}));
    a.pass_cols = a.pass_rows * per_row;
    // Each warp its own tile when that fills the GPU four times over; else the warps of a CTA split K.
    const long long tiles = (long long)a.tiles * (f.offsets ? std::min(f.groups, f.vectors) : 1);
    a.warps_k = kGvWarps;
    while (a.warps_k > 1 && (a.warps_k > a.chunks || tiles * a.warps_k > (long long)sm_count * 64)) a.warps_k >>= 1;
    a.units = (a.tiles + kGvWarps / a.warps_k - 1) / (kGvWarps / a.warps_k);
    if (f.type == NVFP4_TYPE_BF16) launch_type<NVFP4_TYPE_BF16>(a, nt, sm_count, stream);
    else if (f.type == NVFP4_TYPE_F16) launch_type<NVFP4_TYPE_F16>(a, nt, sm_count, stream);
    else launch_type<NVFP4_TYPE_F32>(a, nt, sm_count, stream);
}

}  // namespace nvfp4
