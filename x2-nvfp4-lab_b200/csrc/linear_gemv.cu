// NVFP4 linear with epilogue for few rows: a weight stream.
//
// A warp owns 16 weight rows (with a gate eight gate rows and their eight up
// rows, so that a lane holds both) and 256 columns at a time: lane (g, t)
// loads 32 bytes (64 columns) of rows g and g + 8 and their four block scales,
// decodes them to FP16 in registers (E2M1 x E4M3 is exact there) and feeds
// them straight into mma.sync m16n8k16 as the A operand; the rows of x, as
// FP16 in shared memory, are its B columns. The order of K inside an MMA is
// free as long as both operands agree: an MMA takes four consecutive columns
// of each lane's 64, so that a lane's 32 bytes feed 16 MMAs without a shuffle.
//
// Rows of x in FP16: FP16 as they are; BF16 scaled by a power of two per row
// (largest finite value to [2^14, 2^15)), which is exact for every element
// down to 2^-31 of the row's largest and off by less than 2^-39 of it below;
// FP32 scaled the same way as two columns, high and low half (22 bits and a
// sign): off by 2^-23 of an element at most down to 2^-16 of the row's largest,
// where the low half becomes subnormal, and by 2^-39 of that largest below it.
// The scale comes back in the epilogue.
//
// Every 512 columns the MMAs' sums are added to FP32 registers: the tensor
// core rounds its running sum towards zero, which over long rows would grow
// into a bias.
//
// Bound by the weight stream (9/16 byte a weight) and, on B200, nearly as
// much by the decode (80 weights per cycle and SM with nothing else to do; HBM
// brings 41). Two batches of loads are in flight per warp, two CTAs on an SM: 78-81%
// of the copy bandwidth at 248,320 x 2,048 weights (53.9-55.9 us in replayed graphs, as
// all times here, 61.6 as a call in a row of calls; three batches were no faster, nor
// were asynchronous copies of the weights into shared memory). K is
// split over the warps of a CTA when there are too few row tiles to give every
// warp its own; their sums meet in shared memory in warp order.
#include "linear_fused.cuh"
#include "tma_util.cuh"

#include <algorithm>

namespace nvfp4 {
namespace {

constexpr int kGvThreads = 256;
constexpr int kGvWarps = kGvThreads / 32;
constexpr int kGvCols = 8;                          // columns of an MMA: rows of x, or halves of FP32 rows
constexpr int kGvStaged = 16;                       // most rows of x staged at a time
constexpr int kGvRedPitch = 20;                     // floats per column of a partial tile: conflict-free stores
constexpr size_t kGvSmem = 232384;                 // dynamic shared memory of a CTA (64 bytes are static)
constexpr size_t kGvSmemSm = 233472;               // and of an SM, of which every CTA takes 1 KB more

struct GemvArgs {
    FusedLinearArgs f;
    int chunks;       // 256-column chunks
    int tiles;        // 16-row weight tiles of a group (eight outputs each with a gate)
    int warps_k;      // warps that share a tile's columns (a power of two)
    int pass_rows;    // rows of a group that the MMA columns hold
    int seg_rows;     // rows of x staged at a time, of several groups: pass_rows or more
    int token_stride; // bytes of a staged column
};

// A lane's part of 16 rows x 256 columns: 64 codes and four scales of two rows.
struct Batch {
    uint32_t q[2][8];
    uint32_t s[2];
};

// With the line after it into L2: the warp's next chunk (248,320 x 2,048 weights 53.9 us, 60.6 without; L2 prefetches of
// whole tiles or of the first ones behind the staging of x were slower than that).
__device__ __forceinline__ void load_codes(const uint8_t *p, uint32_t (&q)[8]) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7])
                 : "l"(p));
}

__device__ __forceinline__ uint32_t load_scales(const uint8_t *p) {
    uint32_t s;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(s) : "l"(p));  // volatile: not moved to its use
    return s;
}

// Byte of column octet `o` in a staged row: lane quarter t = (o / 8) % 4 has 128 of every 640 bytes, 160 apart, and
// staged rows are 16 bytes apart modulo 128, so the LDS.128 of a B fragment (two rows, four quarters per phase) touches
// eight different 16-byte units, at constant offsets from one address per lane.
constexpr int kGvStagedChunk = 640;
__device__ __forceinline__ int staged_byte(int o) {
    return (o >> 5) * kGvStagedChunk + ((o >> 3) & 3) * 160 + (o & 7) * 16;
}

// mma_16816 with a zero addend.
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ float finite_abs(float v) {
    const float m = fabsf(v);
    return m <= 3.402823466e38f ? m : 0.0f;  // infinities and NaN do not set the scale
}

// Eight consecutive elements of a row of x as they lie in memory.
template <int TYPE>
struct Octet {
    static constexpr int kWords = TYPE == NVFP4_TYPE_F32 ? 8 : 4;
    uint32_t w[kWords];
    __device__ __forceinline__ float get(int i) const {
        if constexpr (TYPE == NVFP4_TYPE_F32) return __uint_as_float(w[i]);
        const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
        return TYPE == NVFP4_TYPE_F16 ? __half2float(__ushort_as_half((uint16_t)h)) : bf16_bits_to_f32(h);
    }
};

template <int TYPE>
__device__ __forceinline__ Octet<TYPE> load_octet(const FusedLinearArgs &f, long long row, int col, bool wide) {
    Octet<TYPE> v;
    const size_t at = (size_t)(row * f.x_stride + col);
    if (wide) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(f.x) + at * (TYPE == NVFP4_TYPE_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < Octet<TYPE>::kWords / 4; ++i) {
            const uint4 q = __ldg(p + i);
            v.w[4 * i] = q.x, v.w[4 * i + 1] = q.y, v.w[4 * i + 2] = q.z, v.w[4 * i + 3] = q.w;
        }
    } else if constexpr (TYPE == NVFP4_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.w[i] = __ldg(static_cast<const uint32_t *>(f.x) + at + i);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v.w[i] = (uint32_t)__ldg(static_cast<const uint16_t *>(f.x) + at + 2 * i) |
                     ((uint32_t)__ldg(static_cast<const uint16_t *>(f.x) + at + 2 * i + 1) << 16);
    }
    return v;
}

// One octet as FP16 (FP32: high and low halves) at its place, scaled by its row's power of two.
template <int TYPE>
__device__ __forceinline__ void stage_octet(const GemvArgs &a, uint8_t *xs, const uint32_t *amax, float *back, int r, int o,
                                            const Octet<TYPE> &v) {
    uint8_t *to = xs + (TYPE == NVFP4_TYPE_F32 ? 2 * r : r) * a.token_stride + staged_byte(o);
    if constexpr (TYPE == NVFP4_TYPE_F16) {
        *reinterpret_cast<uint4 *>(to) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
        if (o == 0) back[r] = 1.0f;
        return;
    }
    // 2^(14 - e) with e the exponent of the row's largest finite value, kept where both it and its inverse are normal
    // numbers.
    const uint32_t top = amax[r];
    const int e = top ? max((int)(top >> 23) - 127, -112) : 14;
    const float scale = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
    if (o == 0) back[r] = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hi[j] = lo[j] = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float y = v.get(2 * j + b) * scale;
            const __half h = __float2half_rn(y);
            hi[j] |= (uint32_t)__half_as_ushort(h) << (16 * b);
            if constexpr (TYPE == NVFP4_TYPE_F32)
                lo[j] |= (uint32_t)__half_as_ushort(__float2half_rn(fabsf(y) <= 65504.0f ? y - __half2float(h) : 0.0f)) << (16 * b);
        }
    }
    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if constexpr (TYPE == NVFP4_TYPE_F32)
        *reinterpret_cast<uint4 *>(to + a.token_stride) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// Rows [row0, row0 + n) of x as FP16 columns in shared memory, and their scales. A warp's 32 octets are of one row
// (rows are padded to 256 columns). What a thread loads for the rows' maxima it keeps for the conversion; where that
// does not fit its registers the rows are read a second time.
template <int TYPE>
__device__ __forceinline__ void stage_rows(const GemvArgs &a, uint8_t *xs, uint32_t *amax, float *back, int row0, int n) {
    constexpr int kHeld = 16 / Octet<TYPE>::kWords;
    const FusedLinearArgs &f = a.f;
    const int oct = a.chunks * 32, valid = f.cols / 8;  // groups of eight columns, padded and real
    const int items = n * oct;
    const bool wide = ((reinterpret_cast<uintptr_t>(f.x) | (uintptr_t)(f.x_stride * (TYPE == NVFP4_TYPE_F32 ? 4 : 2))) & 15u) == 0;
    const bool once = items <= kHeld * kGvThreads;
    Octet<TYPE> v[kHeld];
    auto load_held = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const int i = i0 + u * kGvThreads, r = i / oct, o = i - r * oct;
            if (i < items && o < valid) {
                v[u] = load_octet<TYPE>(f, row0 + r, o * 8, wide);
            } else {
#pragma unroll
                for (int j = 0; j < Octet<TYPE>::kWords; ++j) v[u].w[j] = 0u;
            }
        }
    };
    if constexpr (TYPE != NVFP4_TYPE_F16) {
        for (int i = threadIdx.x; i < n; i += kGvThreads) amax[i] = 0u;
        __syncthreads();
        for (int i0 = threadIdx.x; i0 < items; i0 += kHeld * kGvThreads) {
            load_held(i0);
#pragma unroll
            for (int u = 0; u < kHeld; ++u) {
                const int i = i0 + u * kGvThreads;
                if (i >= items) break;
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[u].get(j)));
                const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
                if ((threadIdx.x & 31) == 0) atomicMax(amax + i / oct, top);
            }
        }
        __syncthreads();
    }
    for (int i0 = threadIdx.x; i0 < items; i0 += kHeld * kGvThreads) {
        if (TYPE == NVFP4_TYPE_F16 || !once) load_held(i0);
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const int i = i0 + u * kGvThreads, r = i / oct;
            if (i < items) stage_octet<TYPE>(a, xs, amax, back, r, i - r * oct, v[u]);
        }
    }
    __syncthreads();
}

// The same for 16-bit rows through asynchronous copies: the raw bytes go to their places, all in flight at once; then
// every thread looks for the rows' maxima in what it copied itself, and last converts it in place.
template <int TYPE>
__device__ __forceinline__ void stage_rows_async(const GemvArgs &a, uint8_t *xs, uint32_t *amax, float *back, int row0, int n) {
    const FusedLinearArgs &f = a.f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool wide = ((reinterpret_cast<uintptr_t>(f.x) | (uintptr_t)(f.x_stride * 2)) & 15u) == 0;
    // work(row, octet, place) for this thread's octets.
    auto each = [&](auto &&work) {
        int r = warp / a.chunks, c = warp - r * a.chunks;
        while (r < n) {
            work(r, 32 * c + lane, xs + r * a.token_stride + staged_byte(32 * c + lane));
            for (c += kGvWarps; c >= a.chunks; c -= a.chunks) ++r;
        }
    };
    if (threadIdx.x < n) amax[threadIdx.x] = 0u;
    each([&](int r, int o, uint8_t *to) {
        if (8 * o >= f.cols) {
            *reinterpret_cast<uint4 *>(to) = make_uint4(0, 0, 0, 0);
        } else if (wide) {
            cp_async16(to, static_cast<const uint16_t *>(f.x) + (row0 + r) * f.x_stride + 8 * o);
        } else {
            const Octet<TYPE> v = load_octet<TYPE>(f, row0 + r, 8 * o, false);
            *reinterpret_cast<uint4 *>(to) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
        }
    });
    cp_async_wait_all();
    if constexpr (TYPE == NVFP4_TYPE_F16) {
        if (threadIdx.x < n) back[threadIdx.x] = 1.0f;
    } else {
        auto read = [&](const uint8_t *at) {
            const uint4 q = *reinterpret_cast<const uint4 *>(at);
            return Octet<TYPE>{{q.x, q.y, q.z, q.w}};
        };
        __syncthreads();  // amax is zero
        each([&](int r, int, const uint8_t *at) {
            const Octet<TYPE> v = read(at);
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v.get(j)));
            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
            if (lane == 0) atomicMax(amax + r, top);
        });
        __syncthreads();
        each([&](int r, int o, const uint8_t *at) { stage_octet<TYPE>(a, xs, amax, back, r, o, read(at)); });
    }
    __syncthreads();
}

template <int TYPE, bool GROUPED>
__global__ void __launch_bounds__(kGvThreads, 2) linear_gemv_kernel(const __grid_constant__ GemvArgs a) {
    constexpr int kPerRow = TYPE == NVFP4_TYPE_F32 ? 2 : 1;  // MMA columns
    constexpr bool kSeveral = GROUPED && TYPE != NVFP4_TYPE_F32;  // rows of several groups staged together
    extern __shared__ __align__(16) uint8_t gv_smem[];
    const FusedLinearArgs &f = a.f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int warps_k = a.warps_k, teams = kGvWarps / warps_k;
    const int kw = warp & (warps_k - 1), wr = warp / warps_k;

    uint8_t *xs = gv_smem;
    float *red = reinterpret_cast<float *>(gv_smem + (size_t)a.seg_rows * kPerRow * a.token_stride);  // [2][warps][kGvCols][pitch]
    uint32_t *amax = reinterpret_cast<uint32_t *>(red + 2 * kGvWarps * kGvCols * kGvRedPitch);
    float *back = reinterpret_cast<float *>(amax + kGvStaged);
    int *active = reinterpret_cast<int *>(back + kGvStaged);  // [3][groups] groups with rows, their first row and count
    int *active_first = active + f.groups, *active_count = active_first + f.groups;
    __shared__ int warp_sum[kGvWarps];
    __shared__ int s_active;

    int n_active = 1;
    if constexpr (GROUPED) {
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
            if (count > 0) active[at] = i, active_first[at] = first, active_count[at++] = count;
        }
        if (threadIdx.x == kGvThreads - 1) s_active = at;
        __syncthreads();
        n_active = s_active;
    }

    // This CTA's row tiles: a run of (group, tile), taken in turn by its teams of warps_k warps.
    const long long work = (long long)n_active * a.tiles;
    int u = (int)(work * blockIdx.x / gridDim.x);
    const int u_end = (int)(work * (blockIdx.x + 1) / gridDim.x);
    const int batches = ((a.chunks - kw + warps_k - 1) / warps_k + 1) & ~1;  // of this warp; even: two buffers in turn
    int parity = 0;

    // Place of a tile of the run: its group, the tile there, and the group's rows.
    struct Place {
        int group, tile, first, count;
    };
    auto place = [&](int unit) {
        if constexpr (!GROUPED) return Place{0, unit, 0, f.vectors};
        const int ai = unit / a.tiles;
        return Place{active[ai], unit - ai * a.tiles, active_first[ai], active_count[ai]};
    };

    while (u < u_end) {
        // A piece of the run whose rows of x are staged together: of one group, in several passes if it has more rows than
        // the MMA columns hold, else of as many groups one after the other as fit, so that the teams' turn and the loads go
        // on from group to group (256 rows over 256 groups of 1,024 x 2,048 weights 44.5 us, 48.5 a group at a time).
        const Place start = place(u);
        int end = min(u_end, u - start.tile + a.tiles), rows = start.count;
        if (kSeveral && rows <= a.pass_rows) {
            while (end < u_end) {
                const Place p = place(end);
                if (p.count > a.pass_rows || rows + p.count > a.seg_rows || p.first != start.first + rows) break;
                rows += p.count;
                end = min(u_end, end + a.tiles);
            }
        }
        const bool several = kSeveral && rows > start.count;
        const int limit = several ? rows : a.pass_rows;  // rows a pass

        for (int v0 = 0; v0 < rows; v0 += limit) {
            const int n = min(limit, rows - v0), row0 = start.first + v0;

            // The loads run ahead of the arithmetic: (l_unit, l_batch) is the next batch to request.
            // A lane's chunks end with its row's pitch (zero scales follow the last column, whatever codes the padding
            // holds); past it the scales are set to zero and nothing is read.
            int l_unit = u + wr, l_batch = 0, l_chunk = kw;
            const int lane_chunks = (f.packed_pitch - t * 32 + 127) / 128;
            const uint8_t *p0, *p1, *s0, *s1;
            auto set_rows = [&]() {
                // Rows of this lane, clamped to the last (its sums are not stored).
                l_batch = 0;
                l_chunk = l_unit < end ? kw : a.chunks;
                const Place p = place(min(l_unit, end - 1));
                int r0, r1;
                if (f.gated) {
                    r0 = min(p.tile * 8 + g, f.out_rows - 1);
                    r1 = r0 + f.out_rows;
                } else {
                    r0 = min(p.tile * 16 + g, f.rows - 1);
                    r1 = min(p.tile * 16 + g + 8, f.rows - 1);
                }
                const size_t g0 = (size_t)p.group * f.rows;
                p0 = f.packed + (g0 + r0) * f.packed_pitch + kw * 128 + t * 32;
                p1 = f.packed + (g0 + r1) * f.packed_pitch + kw * 128 + t * 32;
                s0 = f.scales + (g0 + r0) * f.scale_pitch + kw * 16 + t * 4;
                s1 = f.scales + (g0 + r1) * f.scale_pitch + kw * 16 + t * 4;
            };
            set_rows();
            auto load = [&](Batch &b) {
                if (l_chunk < lane_chunks) {
                    load_codes(p0, b.q[0]);
                    load_codes(p1, b.q[1]);
                    b.s[0] = load_scales(s0);
                    b.s[1] = load_scales(s1);
                } else {
                    b.s[0] = b.s[1] = 0u;
                }
                if (++l_batch == batches) {
                    l_unit += teams;
                    set_rows();
                } else {
                    p0 += warps_k * 128;
                    p1 += warps_k * 128;
                    s0 += warps_k * 16;
                    s1 += warps_k * 16;
                    l_chunk += warps_k;
                }
            };
            Batch b0, b1;
            load(b0);
            load(b1);
            __syncthreads();  // the rows staged before are no longer read
            // 16-bit rows of more than an octet a thread go by asynchronous copies: 8 rows at 2048 x 16384 12.5 us (13.4
            // through registers), 768 rows over 256 groups 70.9 us (73.6); one row 8.6 us (8.0), and four of FP32, whose
            // halves lie apart, 14.5 us (11.0).
            bool async = false;
            if constexpr (TYPE != NVFP4_TYPE_F32) async = n * a.chunks > kGvWarps;
            if constexpr (TYPE != NVFP4_TYPE_F32) {
                if (async) stage_rows_async<TYPE>(a, xs, amax, back, row0, n);
            }
            if (!async) stage_rows<TYPE>(a, xs, amax, back, row0, n);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};

            // One output from its sum (and its up sum with a gate).
            auto output = [&](const Place &p, float inv, int col0, int row, int v, float z, float z_up) {
                // The row's power of two comes last: with the divisor first the product may be subnormal where the result
                // is not.
                const float scale = back[col0 + v];
                z = z * inv * scale;
                const size_t at = (size_t)p.group * f.rows + row;
                if (f.bias) z += load_as_f32(f.bias, f.bias_type, at);
                z = activate<TYPE == NVFP4_TYPE_F32>(z, f.act);
                if (f.gated) {
                    z_up = z_up * inv * scale;
                    if (f.bias) z_up += load_as_f32(f.bias, f.bias_type, at + f.out_rows);
                    z *= z_up;
                }
                const long long vec = (long long)row0 + col0 + v;
                if (f.residual) z += load_as_f32(f.residual, f.type, (size_t)(vec * f.residual_stride + row));
                store_from_f32(f.out, f.type, (size_t)(vec * f.out_stride + row), z);
            };
            auto finish = [&](const Place &p, int col0, int n) {
                const int per_col = f.gated ? 8 : 16, r0 = p.tile * per_col;
                const float inv = f.inv_globals ? __ldg(f.inv_globals + p.group) : f.inv_global;
                if (warps_k == 1) {
                    // The lane has rows g and g + 8 of MMA columns 2 t and 2 t + 1.
#pragma unroll
                    for (int b = 0; b < (TYPE == NVFP4_TYPE_F32 ? 1 : 2); ++b) {
                        const int v = TYPE == NVFP4_TYPE_F32 ? t : 2 * t + b;
                        if (v >= n) continue;
                        const float z = TYPE == NVFP4_TYPE_F32 ? sum[0] + sum[1] : sum[b];
                        const float y = TYPE == NVFP4_TYPE_F32 ? sum[2] + sum[3] : sum[2 + b];
                        if (r0 + g < f.out_rows) output(p, inv, col0, r0 + g, v, z, y);
                        if (!f.gated && r0 + g + 8 < f.out_rows) output(p, inv, col0, r0 + g + 8, v, y, 0.0f);
                    }
                } else {
                    // Partial tiles meet in shared memory; the warps of a tile share its epilogue.
                    float *to = red + ((size_t)parity * kGvWarps + warp) * kGvCols * kGvRedPitch + 2 * t * kGvRedPitch + g;
                    to[0] = sum[0];
                    to[kGvRedPitch] = sum[1];
                    to[8] = sum[2];
                    to[kGvRedPitch + 8] = sum[3];
                    named_barrier(1 + wr, warps_k * 32);
                    const float *part = red + ((size_t)parity * kGvWarps + wr * warps_k) * kGvCols * kGvRedPitch;
                    for (int i = kw * 32 + lane; i < n * per_col; i += warps_k * 32) {
                        const int v = f.gated ? i >> 3 : i >> 4, r = i & (per_col - 1);
                        if (r0 + r >= f.out_rows) continue;
                        const int c0 = (TYPE == NVFP4_TYPE_F32 ? 2 * v : v) * kGvRedPitch + r;
                        float z = 0.0f, z_up = 0.0f;
                        for (int k = 0; k < warps_k; ++k) {
                            const float *q = part + (size_t)k * kGvCols * kGvRedPitch + c0;
                            z += TYPE == NVFP4_TYPE_F32 ? q[0] + q[kGvRedPitch] : q[0];
                            if (f.gated) z_up += TYPE == NVFP4_TYPE_F32 ? q[8] + q[kGvRedPitch + 8] : q[8];
                        }
                        output(p, inv, col0, r0 + r, v, z, z_up);
                    }
                    parity ^= 1;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = 0.0f;
            };
            auto step = [&](const Batch &b, const uint8_t *bcol, int c, float (&acc)[2][4], bool fresh) {
                const uint32_t f0[2] = {e4m3x2_to_f16x2((uint16_t)b.s[0]), e4m3x2_to_f16x2((uint16_t)(b.s[0] >> 16))};
                const uint32_t f1[2] = {e4m3x2_to_f16x2((uint16_t)b.s[1]), e4m3x2_to_f16x2((uint16_t)(b.s[1] >> 16))};
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    const uint32_t k0 = (w & 2) ? f16x2_hi_hi(f0[w >> 2]) : f16x2_lo_lo(f0[w >> 2]);
                    const uint32_t k1 = (w & 2) ? f16x2_hi_hi(f1[w >> 2]) : f16x2_lo_lo(f1[w >> 2]);
                    uint32_t h0[4], h1[4];
                    e2m1x8_to_f16x8(b.q[0][w], h0);
                    e2m1x8_to_f16x8(b.q[1][w], h1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h0[e] = hmul2_u32(h0[e], k0);
                        h1[e] = hmul2_u32(h1[e], k1);
                    }
                    const uint4 x = *reinterpret_cast<const uint4 *>(bcol + c * kGvStagedChunk + w * 16);
                    if (fresh && w == 0) {
                        mma_16816_first(acc[0], h0[0], h1[0], h0[1], h1[1], x.x, x.y);
                        mma_16816_first(acc[1], h0[2], h1[2], h0[3], h1[3], x.z, x.w);
                    } else {
                        mma_16816(acc[0], h0[0], h1[0], h0[1], h1[1], x.x, x.y);
                        mma_16816(acc[1], h0[2], h1[2], h0[3], h1[3], x.z, x.w);
                    }
                }
            };
            for (int unit = u + wr; unit < end; unit += teams) {
                const Place p = place(unit);
                const int col0 = several ? p.first - start.first : 0;
                const int here = several ? p.count : n;
                // MMA columns past the group's repeat the last: their sums are not stored.
                const uint8_t *bcol = xs + (col0 * kPerRow + min(g, here * kPerRow - 1)) * a.token_stride + t * 160;
                for (int c = kw; c < a.chunks; c += 2 * warps_k) {
                    float acc[2][4];  // two chains
                    step(b0, bcol, c, acc, true);
                    load(b0);
                    if (c + warps_k < a.chunks) step(b1, bcol, c + warps_k, acc, false);
                    load(b1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] += acc[0][i] + acc[1][i];
                }
                finish(p, col0, here);
            }
        }
        u = end;
    }
    zero_other_rows(f);
}

// Shared memory besides the staged rows: partial tiles, scales, the list of groups.
size_t other_smem(const FusedLinearArgs &f) {
    return sizeof(float) * 2 * kGvWarps * kGvCols * kGvRedPitch + 8 * kGvStaged +
           (f.offsets ? 3 * sizeof(int) * f.groups : 0);
}

template <int TYPE, bool GROUPED>
void launch(GemvArgs &a, int device, int sm_count, cudaStream_t stream) {
    const size_t smem = (size_t)a.seg_rows * (TYPE == NVFP4_TYPE_F32 ? 2 : 1) * a.token_stride + other_smem(a.f);
    static std::atomic<uint64_t> done{0};
    allow_shared_memory(linear_gemv_kernel<TYPE, GROUPED>, kGvSmem, done, device, "cudaFuncSetAttribute(linear_gemv_kernel)");
    // Two CTAs on an SM (the kernel's registers) where their shared memory fits.
    const int per_sm = 2 * (smem + 1024) <= kGvSmemSm ? 2 : 1;
    const long long teams = kGvWarps / a.warps_k;
    const long long work = ((long long)a.tiles * (a.f.offsets ? std::min(a.f.groups, a.f.vectors) : 1) + teams - 1) / teams;
    const long long grid = std::min(work, (long long)sm_count * per_sm);
    linear_gemv_kernel<TYPE, GROUPED><<<static_cast<int>(std::max<long long>(1, grid)), kGvThreads, smem, stream>>>(a);
    check_cuda(cudaGetLastError(), "linear_gemv_kernel");
}

template <int TYPE>
void launch_type(GemvArgs &a, int device, int sm_count, cudaStream_t stream) {
    if (a.f.offsets) launch<TYPE, true>(a, device, sm_count, stream);
    else launch<TYPE, false>(a, device, sm_count, stream);
}

// Shared memory of a staged MMA column.
int column_bytes(int cols) { return (cols + 255) / 256 * kGvStagedChunk + 16; }

// Rows of x whose MMA columns fit shared memory.
int staged_rows(const FusedLinearArgs &f) {
    return static_cast<int>((kGvSmem - other_smem(f)) / column_bytes(f.cols)) / (f.type == NVFP4_TYPE_F32 ? 2 : 1);
}

}  // namespace

// Eight rows: one pass of the MMA columns, of FP32 two passes of four rows (high and low halves). Measured against the
// tensor-memory kernel at 16,384 x 2,048 weights: 2 BF16 rows 8.9 against 12.1 us, 4 rows 10.2, 8 rows 12.9 against 12.1,
// 12 rows 20.7; 8 FP32 rows 18.7 against 22.1, 12 rows 26.7; at 65,536 x 2,048 8 BF16 rows 23.4 against 29.5, at 2,048 x
// 2,048 8.5 against 11.2 and 8 FP32 rows 11.2 against 21.3. Groups of rows whose counts are on the device go by their
// average: over 256 groups of 1,024 x 2,048 weights three BF16 rows a group 63 against 92 us, four 94 against 93, six FP32
// rows 179 against 206; over 32 groups three BF16 rows 17.6 against 18.8, four 22.1, four FP32 rows 30.6 against 37.6.
bool linear_gemv_serves(const FusedLinearArgs &f) {
    return staged_rows(f) >= 1 &&
           (f.offsets ? f.vectors <= (f.type == NVFP4_TYPE_F32 ? 6LL : 3LL) * f.groups : f.vectors <= kGvCols);
}

void launch_linear_gemv(const FusedLinearArgs &f, int device, int sm_count, cudaStream_t stream) {
    GemvArgs a{};
    a.f = f;
    a.chunks = (f.cols + 255) / 256;
    a.tiles = f.gated ? (f.out_rows + 7) / 8 : (f.rows + 15) / 16;
    a.token_stride = column_bytes(f.cols);
    const int per_row = f.type == NVFP4_TYPE_F32 ? 2 : 1;
    // Groups may have more rows than their average: further rows in further passes. (MMA columns for 16 rows made every
    // pass slower: a batch of 32 tokens over 256 groups 91 against 54 us.)
    a.pass_rows = std::max(1, std::min({8 / per_row, staged_rows(f), f.vectors}));
    // Rows of several groups staged together: 16 of up to 2,048 columns, and of more as many as that much shared memory
    // holds. More of it leaves the L1 too little for the scales, of which a load uses half a sector (with 24 rows 512 rows
    // over 256 groups of 1,024 x 2,048 weights took 70.9 us, with 16 60.1); FP32 gains nothing (66 us, 62.2 a group at a
    // time: 256 rows over 256 groups).
    a.seg_rows = a.pass_rows;
    if (f.offsets && f.type != NVFP4_TYPE_F32)
        a.seg_rows = std::max(a.pass_rows, std::min({kGvStaged, f.vectors, kGvStaged * column_bytes(2048) / a.token_stride}));
    // As few warps share a tile as leave every SM eight teams at work (half of its warps): 16,384 x 2,048 weights take
    // 8.0 us with two warps a tile and 10.2 with eight, whose barriers cost more than their even shares bring.
    const long long tiles = (long long)a.tiles * (f.offsets ? std::min(f.groups, f.vectors) : 1);
    a.warps_k = 1;
    while (a.warps_k < kGvWarps && 2 * a.warps_k <= a.chunks && tiles * a.warps_k < (long long)sm_count * 8) a.warps_k *= 2;
    if (f.type == NVFP4_TYPE_BF16) launch_type<NVFP4_TYPE_BF16>(a, device, sm_count, stream);
    else if (f.type == NVFP4_TYPE_F16) launch_type<NVFP4_TYPE_F16>(a, device, sm_count, stream);
    else launch_type<NVFP4_TYPE_F32>(a, device, sm_count, stream);
}

}  // namespace nvfp4
