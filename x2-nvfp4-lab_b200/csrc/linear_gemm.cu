// NVFP4 linear with epilogue for many rows: tcgen05 with the weights decoded on
// the way in.
//
// A weight E2M1 * E4M3 is exact in FP16 and in BF16, so the product runs as a
// plain 16-bit MMA on x as it is: no rounding but the FP32 sums'. The weights
// are the A operand (128 rows, M) and lie in tensor memory: conversion warps read
// the packed bytes from shared memory, decode a row's 64 columns in registers
// and store them with tcgen05.st, so that neither the decoded tile nor its
// reads cross shared memory, whose bandwidth the B operand needs. The rows of
// x are B (N = 16 to 160, as many as the tile has: the instruction's N is chosen per tile),
// loaded by TMA. With a gate the tile is 64 gate and 64 up rows, 16 of each in
// every lane quarter.
//
// Warps: 0 producer of x and 2 of weights (TMA), 1 MMA issuer, 4-15 conversion
// (three warpgroups, every third step of 128 columns each), 16-23 epilogue (two
// warpgroups). Tensor memory: two accumulators of
// 160 columns and three decoded steps of 64, or of 64 columns and six. The
// epilogue works in registers: a lane has a weight row, one value of bias, and
// trades with its neighbours for pairs of outputs. (Turning 32 columns a page in
// shared memory for 8-byte stores cost 3,100 cycles a page in barriers, branches
// and generic addresses, and was the bound of short rows: 9,006 FP16 rows x 512
// over 64 groups of 2,048 weight rows took 41.5 us, 33.0 without.)
//
// Persistent pairs of CTAs, one CTA per SM, walk (group, two weight tiles, x
// tile) items: each CTA decodes its own weight tile and loads half of the rows
// of x, and the even one issues the MMAs of both. x tiles of a group are of even
// size, and items of one weight tile are neighbours, so that its bytes come from
// HBM once.
//
// An MMA (of a pair: 256 x N x 16, A in tensor memory) takes N / 2 cycles and 37
// at least, measured, when the next one is issued in time; of one CTA with A in
// shared memory it takes N / 2 + 43.
//
// FP32 x enters as two FP16 halves, scaled per row by a power of two
// (linear_gemv.cu has the error), split by a kernel before; x that TMA cannot
// read (16-byte addresses and strides) is copied by the same kernel. For FP32
// the sums move to FP32 registers of the epilogue every 128 columns, and the low
// halves' products come first: the tensor core rounds its running sum towards
// zero, and the bias of a long chain would show (5.7e-7 of the result with
// segments of 256 columns, high halves first). Of 16-bit x longer than 4,096 columns
// the sums move at least that often to the second accumulator, which then carries the
// sums so far (16 columns at a time through the epilogue's registers): sums of one sign
// come out low by 1.4e-5 on average, 3.7e-5 at most, of FP16 x of any length, by less
// of BF16; in one chain it was 3.2e-5 and 7.1e-5 at 8,192 columns and 2.5e-4 and 3.4e-4
// at 49,152, near FP16's half step of 4.9e-4. 4,096 rows x 8,192 columns over 8,192
// weight rows take 388-398 us (380 in one chain), 1,024 x 28,672 over 4,096 197-204 (190-195).
#include "linear_fused.cuh"
#include "tcgen05_util.cuh"
#include "tma_util.cuh"

#include <algorithm>
#include <atomic>

namespace nvfp4 {
namespace {

constexpr int kGmConvWarp0 = 4, kGmConvGroups = 3, kGmEpiWarp0 = kGmConvWarp0 + 4 * kGmConvGroups;
constexpr int kGmEpiGroups = 2;
constexpr int kGmThreads = 32 * (kGmEpiWarp0 + 4 * kGmEpiGroups);
constexpr int kGmLargeN = 160;                      // rows of x per tile
constexpr int kGmSmallN = 64;                       // of calls with few, and of split FP32 x (32 per epilogue warpgroup)
constexpr int kGmSegment32 = 1;                     // steps per accumulator of split FP32 x
constexpr int kGmSegment16 = 32;                    // and at most of 16-bit x (with 16 of them 8,192 columns take 408-414 us)
constexpr int kGmRawBytes = 128 * 128;              // 256 columns of packed weights
constexpr int kGmRawScales = 128 * 16;
constexpr int kGmRaw = kGmRawBytes + kGmRawScales;

// Tiles of up to N rows of x: tensor memory holds two accumulators of N columns and decoded weights in the rest, so
// small tiles have six decoded 128-column steps in flight, large ones three; x has a ring of its own.
template <int N, int TERMS>
struct Shape {
    static constexpr int kStages = (512 - 2 * N) / 64;
    static constexpr int kHalfB = TERMS * N / 2 * 128;  // a CTA's half of x's rows in a tile, 64 columns of them
    static constexpr int kStageB = 2 * kHalfB;
    static constexpr int kXStages = 6;               // steps of x in flight (a multiple of kStages)
    static constexpr int kRawStages = N == kGmLargeN ? 5 : 6;  // 18 KB of weights each, as many as fit
    static constexpr int kColA = 2 * N;              // tensor-memory column of the first decoded step
    static constexpr int kOffRaw = kXStages * kStageB;
    static constexpr int kOffBars = kOffRaw + kRawStages * kGmRaw;
    static constexpr int kBars = 2 * kStages + 2 * kXStages + 2 * kRawStages + 2 + 2 + 1;
    static constexpr int kOffTiles = kOffBars + kBars * 8 + 8;
    static constexpr size_t kSmem = 1024 + kOffTiles + sizeof(int) * (3 * kLinMaxGroups + 1);
    static_assert(kXStages % kStages == 0, "the MMA warp's loop is unrolled over both rings");
    static_assert(kOffTiles % 4 == 0 && kSmem <= 232448, "shared memory overflow");
    static_assert(kColA + 64 * kStages <= 512, "tensor memory overflow");
    static_assert(kHalfB % 1024 == 0 && kOffRaw % 1024 == 0 && kGmRaw % 1024 == 0, "swizzled tiles need 1024-byte alignment");
};

enum GemmWaitSite : int {
    kSiteFusedEmpty = 71,
    kSiteFusedRawEmpty = 72,
    kSiteFusedRawFull = 73,
    kSiteFusedFull = 74,
    kSiteFusedAccEmpty = 75,
    kSiteFusedAccFull = 76,
    kSiteFusedRowsEmpty = 77,
    kSiteFusedRowsFull = 78,
};

struct GemmArgs {
    FusedLinearArgs f;
    const float *row_scale;  // [vectors] of split FP32 x (NULL: ones)
    int max_n;               // rows of x per tile
    int box_rows;            // rows of x per TMA box: a CTA's half of a tile, or more
    int segment;             // steps per accumulator
    int m_pairs;             // pairs of weight tiles of a group
    int raw_steps;           // 256-column steps over K
    int k_steps;             // 128-column steps over K
    int pairs_out;           // two neighbouring 16-bit outputs (and two of the residual) may move as one word
};

// A warp's wait: one try and a vote on the way that matters, the bounded wait
// out of line. The same answer in every lane, so that a warp stays whole.
__device__ __noinline__ bool wait_long(uint64_t *bar, uint32_t parity, int *err, int site) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, site));
}

__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, int *err, int site) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return wait_long(bar, parity, err, site);
}

__device__ __forceinline__ bool wait_drain(uint64_t *bar, uint32_t parity) {
    const unsigned long long t0 = global_ns();
    for (uint32_t i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 63u && global_ns() - t0 > kWaitLimitNs) return false;
    }
}

// Two FP16 values times their scales as a BF16 pair: the products have at most six significant bits, so the FP32
// results of the mixed-precision FMA are exact and so are their upper halves. (Shifting FP16 patterns into BF16 and
// multiplying there takes two more instructions on the half-rate integer pipe: 29 against 44 weights per cycle and SM.)
__device__ __forceinline__ uint32_t mul_f16x2_to_bf16x2(uint32_t a, uint32_t b) {
    float lo, hi;
    asm("{\n\t.reg .f16 a0, a1, b0, b1;\n\t"
        "mov.b32 {a0, a1}, %2;\n\tmov.b32 {b0, b1}, %3;\n\t"
        "fma.rn.f32.f16 %0, a0, b0, 0f00000000;\n\tfma.rn.f32.f16 %1, a1, b1, 0f00000000;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(a), "r"(b));
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

// Eight codes times their block scale (FP16, twice) as four 16-bit pairs.
template <bool BF16>
__device__ __forceinline__ void decode8(uint32_t codes, uint32_t scale, uint32_t *out) {
    uint32_t h[4];
    e2m1x8_to_f16x8(codes, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = BF16 ? mul_f16x2_to_bf16x2(h[i], scale) : hmul2_u32(h[i], scale);
}

struct Tile {
    int group, m, row0, n;  // row0, n: rows of x
};

// Tile sizes of a group of `count` rows: as many tiles as needed, even, a multiple of 16 rows each.
__device__ __forceinline__ int x_tiles(int count, int max_n) { return (count + max_n - 1) / max_n; }

// `upto` [groups + 1]: x tiles of the groups before; after it each group's first row and number of rows. `group`: one at
// or before the item's, left at the item's: a warp's items only go forward, and its lanes look at 32 groups at once.
__device__ __forceinline__ Tile tile_of(const GemmArgs &a, const int *upto, int item, int &group) {
    Tile t;
    const int at = item / a.m_pairs, groups = a.f.offsets ? a.f.groups : 1;
    // The last group with upto[g] <= at: as many steps on as following groups begin at or before it.
    if (groups > 1) {
        for (unsigned on = ~0u; on == ~0u;) {
            const int g = group + 1 + (int)(threadIdx.x & 31);
            on = __ballot_sync(0xffffffffu, g < groups && upto[min(g, groups)] <= at);
            group += __popc(on);
        }
    }
    t.group = group;
    const int first = upto[groups + 1 + group], count = upto[2 * groups + 1 + group];
    const int before = upto[group], tiles = upto[group + 1] - before;
    const int in_group = item - before * a.m_pairs;
    int m = in_group, v = 0, width = (count + 15) & ~15;
    if (tiles > 1) {
        m = in_group / tiles;
        width = ((count + tiles - 1) / tiles + 15) & ~15;
        v = (in_group - m * tiles) * width;
    }
    t.m = 2 * m + (int)cluster_rank();
    t.row0 = first + v;
    t.n = min(width, count - v);
    return t;
}

template <int TYPE>
__device__ __forceinline__ float value_of(uint16_t bits) {
    return TYPE == NVFP4_TYPE_F16 ? __half2float(__ushort_as_half(bits)) : bf16_bits_to_f32(bits);
}

template <int TYPE>
__device__ __forceinline__ uint32_t pair_of(float lo, float hi) {
    uint32_t word;
    if constexpr (TYPE == NVFP4_TYPE_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        memcpy(&word, &h, 4);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        memcpy(&word, &h, 4);
    }
    return word;
}

// What a lane of the epilogue does for a tile: it holds one weight row's sums, of 16 rows of x at a time.
struct Finish {
    int out0;      // its output (with a gate the one that its row and the row 16 lanes on make together)
    int row0, n;   // rows of x of the tile
    float inv, bias;
};

template <int ACT, bool FP32, int COUNT>
__device__ __forceinline__ void activate_all(float (&y)[COUNT]) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) y[i] = activate<ACT, FP32>(y[i]);
}

// 16 rows of x from c0 on: scale, bias, activation, gate, residual, one rounding, store. With a gate lanes 0-15 hold
// gate rows and lanes 16-31 their up rows: lanes of the first half finish the even rows of x, of the second the odd
// ones. 16-bit outputs then trade with the lane beside, so that a lane stores two neighbouring outputs of one row: a
// warp writes 64 bytes of each row (32 with a gate), whole sectors, without shared memory.
template <int TYPE, bool GATED, bool ACTIVE>
__device__ __forceinline__ void finish_rows(const GemmArgs &a, const Finish &t, int c0, const float (&sums)[16], float row_scale) {
    constexpr int kOut = GATED ? 8 : 16, kRowStep = GATED ? 2 : 1;
    constexpr bool kFp32 = TYPE == NVFP4_TYPE_F32;
    constexpr int kBytes = kFp32 ? 4 : 2;
    const FusedLinearArgs &f = a.f;
    const int lane = threadIdx.x & 31;
    float y[kOut], up[kOut];
#pragma unroll
    for (int i = 0; i < 16; i += kRowStep) {
        float z[2];
#pragma unroll
        for (int k = 0; k < kRowStep; ++k) {
            // The row's power of two comes last: with the divisor first the product may be subnormal where the result is
            // not.
            if constexpr (TYPE == NVFP4_TYPE_F32)
                z[k] = fmaf(sums[i + k] * t.inv, __shfl_sync(0xffffffffu, row_scale, (c0 & 16) + i + k), t.bias);
            else
                z[k] = fmaf(sums[i + k], t.inv, t.bias);
        }
        y[i / kRowStep] = z[0];
        if constexpr (GATED) {
            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? z[1] : z[0], 16);
            y[i / 2] = lane < 16 ? z[0] : other;
            up[i / 2] = lane < 16 ? other : z[1];
        }
    }
    if constexpr (ACTIVE) switch (f.act) {
        case NVFP4_ACT_RELU: activate_all<NVFP4_ACT_RELU, kFp32>(y); break;
        case NVFP4_ACT_SILU: activate_all<NVFP4_ACT_SILU, kFp32>(y); break;
        case NVFP4_ACT_GELU: activate_all<NVFP4_ACT_GELU, kFp32>(y); break;
        case NVFP4_ACT_GELU_TANH: activate_all<NVFP4_ACT_GELU_TANH, kFp32>(y); break;
        default: break;
    }
    if constexpr (GATED) {
#pragma unroll
        for (int i = 0; i < kOut; ++i) y[i] *= up[i];
    }
    const int first = c0 + (GATED ? lane >> 4 : 0);
    const long long out_step = kRowStep * f.out_stride * kBytes, res_step = kRowStep * f.residual_stride * kBytes;
    if (TYPE != NVFP4_TYPE_F32 && a.pairs_out) {
        // Words of two outputs: even lanes those of row i, odd lanes of row i + 1; `half` picks a lane's part of both.
        const int odd = lane & 1, row = first + odd * kRowStep, col = t.out0 - odd;
        const uint32_t half = odd ? 0x3276u : 0x5410u;
        const int left = col < f.out_rows ? t.n - row : 0;  // rows of x that this lane may store to
        if (f.residual) {
            const uint8_t *res = static_cast<const uint8_t *>(f.residual) + ((t.row0 + row) * f.residual_stride + col) * kBytes;
            uint32_t r[kOut / 2];
#pragma unroll
            for (int i = 0; i < kOut; i += 2) {
                r[i / 2] = 0;
                if (i * kRowStep < left) r[i / 2] = *reinterpret_cast<const uint32_t *>(res + i * res_step);
            }
#pragma unroll
            for (int i = 0; i < kOut; i += 2) {
                const uint32_t mine = __byte_perm(r[i / 2], __shfl_xor_sync(0xffffffffu, r[i / 2], 1), half);
                y[i] += value_of<TYPE>(static_cast<uint16_t>(mine));
                y[i + 1] += value_of<TYPE>(static_cast<uint16_t>(mine >> 16));
            }
        }
        uint8_t *out = static_cast<uint8_t *>(f.out) + ((t.row0 + row) * f.out_stride + col) * kBytes;
        uint32_t words[kOut / 2];
#pragma unroll
        for (int i = 0; i < kOut; i += 2) {
            const uint32_t mine = pair_of<TYPE>(y[i], y[i + 1]);
            words[i / 2] = __byte_perm(mine, __shfl_xor_sync(0xffffffffu, mine, 1), half);
        }
        // Whole pages without a predicate a store, and calls without an activation without its branch: 9,006 rows x 512 over
        // 64 groups of 2,048 weight rows 37.3 us, 40.1 with them.
        if (__all_sync(0xffffffffu, left > (kOut - 2) * kRowStep)) {
#pragma unroll
            for (int i = 0; i < kOut; i += 2) {
                *reinterpret_cast<uint32_t *>(out) = words[i / 2];
                out += 2 * out_step;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kOut; i += 2) {
            const uint32_t word = words[i / 2];
            if (i * kRowStep < left) *reinterpret_cast<uint32_t *>(out + i * out_step) = word;
        }
        return;
    }
    const int left = t.out0 < f.out_rows ? t.n - first : 0;
    if (f.residual) {
        const uint8_t *res = static_cast<const uint8_t *>(f.residual) + ((t.row0 + first) * f.residual_stride + t.out0) * kBytes;
        float r[kOut];
#pragma unroll
        for (int i = 0; i < kOut; ++i) r[i] = i * kRowStep < left ? load_as_f32(res + i * res_step, TYPE, 0) : 0.0f;
#pragma unroll
        for (int i = 0; i < kOut; ++i) y[i] += r[i];
    }
    uint8_t *out = static_cast<uint8_t *>(f.out) + ((t.row0 + first) * f.out_stride + t.out0) * kBytes;
#pragma unroll
    for (int i = 0; i < kOut; ++i)
        if (i * kRowStep < left) store_from_f32(out + i * out_step, TYPE, 0, y[i]);
}

template <int TYPE>
__device__ __forceinline__ void finish_rows(const GemmArgs &a, const Finish &t, int c0, const float (&sums)[16], float row_scale) {
    if (a.f.gated) finish_rows<TYPE, true, true>(a, t, c0, sums, row_scale);
    else if (TYPE == NVFP4_TYPE_F32 || a.f.act != NVFP4_ACT_NONE) finish_rows<TYPE, false, true>(a, t, c0, sums, row_scale);
    else finish_rows<TYPE, false, false>(a, t, c0, sums, row_scale);
}

// TYPE: of x, residual and out; FP32 x arrives as FP16 parts. CARRIED: rows of 16-bit x too long for one accumulator; the
// second one carries the sums of the segments before.
template <int TYPE, int N, bool CARRIED>
__global__ void __launch_bounds__(kGmThreads, 1)
    linear_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_s,
                       const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ GemmArgs a) {
    constexpr bool kBf16 = TYPE == NVFP4_TYPE_BF16;
    constexpr int kTerms = TYPE == NVFP4_TYPE_F32 ? 2 : 1;
    using Z = Shape<N, kTerms>;
    constexpr int S = Z::kStages, X = Z::kXStages, R = Z::kRawStages;
    extern __shared__ uint8_t gm_smem_raw[];
    uint8_t *smem = gm_smem_raw + (-smem_u32(gm_smem_raw) & 1023u);
    const FusedLinearArgs &f = a.f;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + Z::kOffBars);    // [S] weights are decoded (four warps); even CTA: and the odd one's weights and rows of x are there
    uint64_t *empty = full + S;                                          // [S] the step's MMAs are done with the weights
    uint64_t *x_full = empty + S;                                        // [X] rows of x have landed
    uint64_t *x_empty = x_full + X;                                      // [X] the step's MMAs are done with them
    uint64_t *raw_full = x_empty + X;                                      // [R] packed weights and scales have landed
    uint64_t *raw_empty = raw_full + R;                                  // [R] (four conversion warps for each of its two steps)
    uint64_t *acc_full = raw_empty + R;                                  // [2]
    uint64_t *acc_empty = acc_full + 2;                                  // [2] (every epilogue warp of both CTAs; even CTA)
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    int *upto = reinterpret_cast<int *>(smem + Z::kOffTiles);             // [groups + 1] x tiles of the groups before (tile_of)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err = f.err;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(full + i, 4 + (rank == 0 ? 1 : 0));
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < X; ++i) {
            mbar_init(x_full + i, 1);
            mbar_init(x_empty + i, 1);
        }
        for (int i = 0; i < R; ++i) {
            mbar_init(raw_full + i, 1);
            mbar_init(raw_empty + i, 2 * 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, 2 * 4 * kGmEpiGroups);
        }
        mbar_init(drain, 1);
        fence_barrier_init();
        prefetch_tensormap(&tm_w);
        prefetch_tensormap(&tm_s);
        prefetch_tensormap(&tm_x);
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(tmem_slot, 512);
    }
    if (warp == 2) {
        const int groups = f.offsets ? f.groups : 1;
        const int per = (groups + 31) / 32, g0 = min(lane * per, groups), g1 = min(g0 + per, groups);
        int own = 0;
        for (int g = g0; g < g1; ++g) {
            int first, count;
            group_range(f, g, &first, &count);
            own += x_tiles(count, a.max_n);
        }
        int before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (lane == 31) upto[groups] = before;
        before -= own;
        for (int g = g0; g < g1; ++g) {
            int first, count;
            group_range(f, g, &first, &count);
            upto[g] = before;
            upto[groups + 1 + g] = first;
            upto[2 * groups + 1 + g] = count;
            before += x_tiles(count, a.max_n);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    cluster_sync();  // the other CTA's barriers are ready too
    tc::fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int items = upto[f.offsets ? f.groups : 1] * a.m_pairs;
    if (warp != 2) pdl_wait();  // the rows that the split kernel wrote; the weights wait for nothing

    if (warp == 0) {
        // ----------------------------------------------- producer of x
        uint32_t it = 0;
        int group = 0;
        bool ok = true;
        for (int item = pair; item < items && ok; item += pairs) {
            const Tile t = tile_of(a, upto, item, group);
            // The pair splits the tile's rows: this CTA's are the first or the second half of N.
            const int half = ((t.n + 15) & ~15) / 2, row0 = t.row0 + (int)rank * half;
            for (int ks = 0; ks < a.k_steps; ++ks, ++it) {
                const int st = it % X;
                if (!wait_warp(x_empty + st, ((it / X) & 1u) ^ 1u, err, kSiteFusedRowsEmpty)) {
                    ok = false;
                    break;
                }
                uint8_t *b = smem + st * Z::kStageB;
                if (tc::elect_one()) {
                    mbar_arrive_expect_tx(x_full + st, 2 * kTerms * a.box_rows * 128);
#pragma unroll
                    for (int j = 0; j < kTerms; ++j) {
                        uint8_t *to = b + j * (kGmSmallN / 2) * 128;
                        const int row = j * f.vectors + row0;
                        tma_load_2d(to, &tm_x, x_full + st, ks * 256, row);
                        tma_load_2d(to + Z::kHalfB, &tm_x, x_full + st, ks * 256 + 128, row);
                    }
                }
                __syncwarp();
            }
        }
        // After a failure the copies of the last stages issued land before the CTA ends.
        if (!ok || *reinterpret_cast<volatile int *>(err) != 0)
            for (uint32_t k = it > (uint32_t)X ? it - X : 0u; k < it; ++k) wait_drain(x_full + k % X, (k / X) & 1u);
        __syncwarp();
    } else if (warp == 2) {
        // ----------------------------------------- producer of weights
        uint32_t rt = 0;
        int group = 0;
        bool ok = true;
        for (int item = pair; item < items && ok; item += pairs) {
            const Tile t = tile_of(a, upto, item, group);
            const int w0 = t.group * f.rows + t.m * (f.gated ? 64 : 128), w1 = w0 + (f.gated ? f.out_rows : 64);
            for (int rs = 0; rs < a.raw_steps; ++rs, ++rt) {
                const int st = rt % R;
                if (!wait_warp(raw_empty + st, ((rt / R) & 1u) ^ 1u, err, kSiteFusedRawEmpty)) {
                    ok = false;
                    break;
                }
                uint8_t *raw = smem + Z::kOffRaw + st * kGmRaw;
                if (tc::elect_one()) {
                    mbar_arrive_expect_tx(raw_full + st, kGmRaw);
                    tma_load_2d(raw, &tm_w, raw_full + st, rs * 128, w0);
                    tma_load_2d(raw + kGmRawBytes / 2, &tm_w, raw_full + st, rs * 128, w1);
                    tma_load_2d(raw + kGmRawBytes, &tm_s, raw_full + st, rs * 16, w0);
                    tma_load_2d(raw + kGmRawBytes + kGmRawScales / 2, &tm_s, raw_full + st, rs * 16, w1);
                }
                __syncwarp();
            }
        }
        if (!ok || *reinterpret_cast<volatile int *>(err) != 0)
            for (uint32_t k = rt > (uint32_t)R ? rt - R : 0u; k < rt; ++k) wait_drain(raw_full + k % R, (k / R) & 1u);
        __syncwarp();
    } else if (warp == 1) {
        // ---------------------------------------------------------- MMA
        // Everything an instruction takes is the same in every lane and known to be (reductions, loop counters).
        const uint64_t desc = tc::smem_desc_sw128(smem_u32(smem));  // its address field cannot overflow
        const int last = __reduce_max_sync(0xffffffffu, items);
        uint32_t st = 0, ph = 0, x_ph = 0;  // step in the ring of x; phases of the weights' ring and of x's
        bool ok = true;
        uint32_t use = 0;  // accumulators filled so far
        if (rank == 1) {
            // The odd CTA tells the even one, which issues for both, when its half of a step is there.
            uint32_t wst = 0;
            for (int item = pair; item < last && ok; item += pairs) {
                for (int ks = 0; ks < a.k_steps; ++ks) {
                    if (!wait_warp(x_full + st, x_ph, err, kSiteFusedRowsFull) || !wait_warp(full + wst, ph, err, kSiteFusedFull)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    tc::fence_before_sync();
                    if (tc::elect_one()) mbar_arrive_at(full + wst, 0);
                    __syncwarp();
                    if (++wst == S) wst = 0, ph ^= 1;
                    if (++st == X) st = 0, x_ph ^= 1;
                }
            }
        } else {
            int group = 0;
            for (int item = pair; item < last && ok; item += pairs) {
                const uint32_t n = __reduce_max_sync(0xffffffffu, tile_of(a, upto, item, group).n);
                const uint32_t idesc = tc::idesc_16bit_pair((n + 15) & ~15u, kBf16 ? 1u : 0u);
                for (int left = a.k_steps; left > 0 && ok; left -= a.segment, ++use) {
                    const uint32_t buf = use & 1, acc = tmem + (CARRIED ? 0 : buf * N);
                    // The last use of this accumulator: two before, or the one before.
                    const uint32_t prior = use - (CARRIED ? 1 : 2);
                    if ((int)prior >= 0 && !wait_warp(acc_empty + (prior & 1), (prior >> 1) & 1u, err, kSiteFusedAccEmpty)) {
                        ok = false;
                        break;
                    }
                    uint32_t more = 0;
                    // Unrolled over the ring, so that barriers and descriptors are constants away from a base (230
                    // against 150 cycles of a step's issue, measured alone).
                    for (int todo = min(left, a.segment); todo > 0 && ok;) {
#pragma unroll
                        for (int stage = 0; stage < X; ++stage) {
                            constexpr int kS = S;
                            const int ws = stage % kS;
                            if (st != stage || todo == 0 || !ok) continue;
                            if (!wait_warp(x_full + stage, x_ph, err, kSiteFusedRowsFull) ||
                                !wait_warp(full + ws, ph, err, kSiteFusedFull)) {
                                ok = false;
                                continue;
                            }
                            tc::fence_after_sync();
                            if (tc::elect_one()) {
#pragma unroll
                                for (int j = kTerms - 1; j >= 0; --j)  // the small halves first
#pragma unroll
                                    for (int i = 0; i < 8; ++i)
                                        tc::mma_16bit_ts_pair(
                                            acc, tmem + Z::kColA + 64 * ws + 8 * i,
                                            desc + ((stage * Z::kStageB + (i >> 2) * Z::kHalfB + j * (kGmSmallN / 2) * 128 +
                                                     32 * (i & 3)) >> 4),
                                            idesc, j != kTerms - 1 || i != 0 ? 1u : more);
                                tc::commit_pair(empty + ws);
                                tc::commit_pair(x_empty + stage);
                            }
                            __syncwarp();
                            more = 1;
                            --todo;
                            st = (stage + 1) % X;
                            if (ws + 1 == kS) ph ^= 1;
                            if (stage + 1 == X) x_ph ^= 1;
                        }
                    }
                    if (ok && tc::elect_one()) tc::commit_pair(acc_full + buf);
                    __syncwarp();
                }
            }
        }
        // Every MMA has completed before tensor memory is freed. The last commit arrives at the same place in both CTAs:
        // each waits for its own arrival, the odd one after the cluster's barrier, by which it has been issued.
        if (rank == 0) {
            if (tc::elect_one()) tc::commit_pair(drain);
            __syncwarp();
            wait_drain(drain, 0);
        }
        __syncwarp();
    } else if (warp >= kGmConvWarp0 && warp < kGmEpiWarp0) {
        // --------------------------------------------------- conversion
        const int mine = (warp - kGmConvWarp0) >> 2;  // the warpgroup's first step
        const int quarter = warp & 3;
        // Row of the raw tile that this lane decodes into its tensor-memory lane.
        const int row = f.gated ? (lane & 15) + 16 * quarter + (lane >= 16 ? 64 : 0) : 32 * quarter + lane;
        const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16) + Z::kColA;
        uint32_t it = 0, rt = 0;  // steps and raw stages of the tiles before
        int ks = mine;
        bool ok = true;
        for (int item = pair; item < items && ok; item += pairs) {
            for (; ks < a.k_steps; ks += kGmConvGroups) {
                const uint32_t step = it + ks, raw_no = rt + (ks >> 1);
                const int st = step % S, rs = raw_no % R;
                if (!wait_warp(raw_full + rs, (raw_no / R) & 1u, err, kSiteFusedRawFull)) {
                    ok = false;
                    break;
                }
                const uint8_t *raw = smem + Z::kOffRaw + rs * kGmRaw;
                const uint2 sc = *reinterpret_cast<const uint2 *>(raw + kGmRawBytes + row * 16 + 8 * (ks & 1));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int unit = 4 * (ks & 1) + 2 * half;  // 16-byte unit of the row's 128
                    const uint4 q0 = *reinterpret_cast<const uint4 *>(raw + row * 128 + ((unit ^ (row & 7)) << 4));
                    const uint4 q1 = *reinterpret_cast<const uint4 *>(raw + row * 128 + (((unit + 1) ^ (row & 7)) << 4));
                    const uint32_t word = half ? sc.y : sc.x;
                    const uint32_t s01 = e4m3x2_to_f16x2((uint16_t)word), s23 = e4m3x2_to_f16x2((uint16_t)(word >> 16));
                    const uint32_t s0 = f16x2_lo_lo(s01), s1 = f16x2_hi_hi(s01), s2 = f16x2_lo_lo(s23), s3 = f16x2_hi_hi(s23);
                    uint32_t r[32];
                    decode8<kBf16>(q0.x, s0, r);
                    decode8<kBf16>(q0.y, s0, r + 4);
                    decode8<kBf16>(q0.z, s1, r + 8);
                    decode8<kBf16>(q0.w, s1, r + 12);
                    decode8<kBf16>(q1.x, s2, r + 16);
                    decode8<kBf16>(q1.y, s2, r + 20);
                    decode8<kBf16>(q1.z, s3, r + 24);
                    decode8<kBf16>(q1.w, s3, r + 28);
                    if (half == 0) {
                        if (!wait_warp(empty + st, ((step / S) & 1u) ^ 1u, err, kSiteFusedEmpty)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after_sync();
                    }
                    tc::st_32x32b_x32(lanes + 64 * st + 32 * half, r);
                }
                if (!ok) break;
                // The raw stage may be refilled; one that holds a row's last, odd step has no second reader.
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(raw_empty + rs);
                    if ((ks & 1) == 0 && ks + 1 == a.k_steps) mbar_arrive(raw_empty + rs);
                }
                tc::wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + st);
            }
            ks -= a.k_steps;
            it += a.k_steps;
            rt += a.raw_steps;
        }
    } else if (warp >= kGmEpiWarp0) {
        // ----------------------------------------------------- epilogue
        const int piece = (warp - kGmEpiWarp0) >> 2, quarter = warp & 3;
        const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
        const int tile_rows = f.gated ? 64 : 128, own = f.gated ? 16 * quarter + (lane & 15) : 32 * quarter + lane;
        int use = 0;
        auto filled = [&]() {
            const bool is = wait_warp(acc_full + (use & 1), (use >> 1) & 1u, err, kSiteFusedAccFull);
            tc::fence_after_sync();
            return is;
        };
        // With more tiles than pairs the warpgroups take whole tiles in turn (each its accumulator; what one waits for at
        // the start of a tile hides behind the other's work), else every other 16 columns of the one tile. FP32 always
        // does the latter, its sums are in registers, and so do rows of several segments.
        const bool whole = TYPE != NVFP4_TYPE_F32 && items > pairs && !CARRIED;
        auto release = [&]() {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_at(acc_empty + (use & 1), 0);
                if (whole) mbar_arrive_at(acc_empty + (use & 1), 0);  // for the other warpgroup
            }
        };
        bool ok = true;
        int group = 0;
        for (int item = pair; item < items && ok; item += pairs) {
            if (whole && (use & 1) != piece) {
                ++use;
                continue;
            }
            const Tile t = tile_of(a, upto, item, group);
            Finish to{t.m * tile_rows + own, t.row0, t.n, f.inv_globals ? __ldg(f.inv_globals + t.group) : f.inv_global, 0.0f};
            if (f.bias && to.out0 < f.out_rows)
                to.bias = load_as_f32(f.bias, f.bias_type,
                                      (size_t)t.group * f.rows + to.out0 + (f.gated && lane >= 16 ? f.out_rows : 0));
            if constexpr (TYPE == NVFP4_TYPE_F32) {
                const float row_scale = 32 * piece + lane < t.n ? __ldcg(a.row_scale + t.row0 + 32 * piece + lane) : 0.0f;
                float sum[2][16];
#pragma unroll
                for (int i = 0; i < 32; ++i) sum[i >> 4][i & 15] = 0.0f;
                for (int ks = 0; ks < a.k_steps; ks += a.segment, ++use) {
                    if (!filled()) {
                        ok = false;
                        break;
                    }
                    uint32_t r[32];
                    tc::ld_32x32b_x32(lanes + (use & 1) * N + 32 * piece, r);
                    tc::wait_ld();
                    release();
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[i >> 4][i & 15] += __uint_as_float(r[i]);
                }
                if (!ok) break;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (32 * piece + 16 * h < t.n) finish_rows<TYPE>(a, to, 32 * piece + 16 * h, sum[h], row_scale);
            } else {
                uint32_t from = lanes + (use & 1) * N;
                if constexpr (CARRIED) {
                    // Each segment's sums to those of the segments before, which the rest of the tile is made of.
                    from = lanes + N;
                    for (int ks = 0; ks < a.k_steps && ok; ks += a.segment) {
                        ok = filled();
                        if (!ok) break;
                        for (int c0 = 16 * piece; c0 < t.n; c0 += 16 * kGmEpiGroups) {
                            uint32_t r[16], before[16];
                            tc::ld_32x32b_x16(lanes + c0, r);
                            if (ks != 0) tc::ld_32x32b_x16(from + c0, before);
                            tc::wait_ld();
                            if (ks != 0) {
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    r[i] = __float_as_uint(__uint_as_float(before[i]) + __uint_as_float(r[i]));
                            }
                            tc::st_32x32b_x16(from + c0, r);
                        }
                        tc::wait_st();
                        release();
                        ++use;
                    }
                } else {
                    ok = filled();
                }
                if (!ok) break;
                const int step = whole ? 16 : 16 * kGmEpiGroups, c_first = whole ? 0 : 16 * piece;
                for (int c0 = c_first; c0 < t.n; c0 += step) {
                    uint32_t r[16];
                    float sum[16];
                    tc::ld_32x32b_x16(from + c0, r);
                    tc::wait_ld();
                    if (!CARRIED && c0 + step >= t.n) release();
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[i] = __uint_as_float(r[i]);
                    finish_rows<TYPE>(a, to, c0, sum, 1.0f);
                }
                if (!CARRIED) {
                    if (c_first >= t.n) release();
                    ++use;
                }
            }
        }
    }
    zero_other_rows(f);

    tc::fence_before_sync();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other may reach its shared memory
    if (warp == 1) {
        if (rank == 1) wait_drain(drain, 0);  // no arrival is on its way to this shared memory when the CTA ends
        __syncwarp();
        tc::fence_after_sync();
        tc::tmem_dealloc_pair(tmem, 512);
    }
    if (threadIdx.x == 0 && *reinterpret_cast<volatile int *>(err) != 0 && f.host_err) {
        const int code = *reinterpret_cast<volatile int *>(err);
        *reinterpret_cast<volatile int *>(f.host_err) = code != 0 ? code : kErrWaitTimeout;
    }
}

// ------------------------------------------------------------------ rows of x that TMA cannot read as they are

struct SplitArgs {
    const void *x;
    long long x_stride;
    int type, vectors, cols;
    uint16_t *parts;    // [2][vectors][cols] FP16 halves of FP32 x, or [vectors][cols] as it is
    float *row_scale;   // [vectors]
};

// A CTA per row. FP32: the largest finite value to [2^14, 2^15) by a power of
// two, then the high half and what it leaves over (linear_gemv.cu's parts).
__global__ void __launch_bounds__(128) linear_split_kernel(SplitArgs a) {
    __shared__ uint32_t warp_top[4];
    pdl_launch_dependents();
    const int row = blockIdx.x;
    const size_t to = (size_t)row * a.cols;
    if (a.type != NVFP4_TYPE_F32) {
        const uint16_t *x = static_cast<const uint16_t *>(a.x) + row * a.x_stride;
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) a.parts[to + c] = x[c];
        return;
    }
    // Four columns at a time; a row's first 2,048 are read once and held (scalar loads, twice, made calls of 301 x 1,008 17.8 instead
    // of 16.2 us and of 40 x 8,192 71 instead of 60).
    const float *x = static_cast<const float *>(a.x) + row * a.x_stride;
    const bool wide = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
    auto load = [&](int c) {
        return wide ? *reinterpret_cast<const float4 *>(x + c) : make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]);
    };
    auto largest = [](const float4 &v) {
        auto finite = [](float f) { return fabsf(f) <= 3.402823466e38f ? fabsf(f) : 0.0f; };
        return fmaxf(fmaxf(finite(v.x), finite(v.y)), fmaxf(finite(v.z), finite(v.w)));
    };
    constexpr int kHeld = 4, kStep = 4 * 128;
    const int c0 = 4 * threadIdx.x;
    float4 held[kHeld];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        held[i] = c0 + i * kStep < a.cols ? load(c0 + i * kStep) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) m = fmaxf(m, largest(held[i]));
    for (int c = c0 + kHeld * kStep; c < a.cols; c += kStep) m = fmaxf(m, largest(load(c)));
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
    top = max(max(warp_top[0], warp_top[1]), max(warp_top[2], warp_top[3]));
    const int e = top ? max((int)(top >> 23) - 127, -112) : 14;
    const float scale = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
    if (threadIdx.x == 0) a.row_scale[row] = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
    uint16_t *low = a.parts + (size_t)a.vectors * a.cols;
    auto split = [&](int c, const float4 &v) {
        const float y[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
        uint16_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half hi = __float2half_rn(y[i]);
            h[i] = __half_as_ushort(hi);
            l[i] = __half_as_ushort(__float2half_rn(fabsf(y[i]) <= 65504.0f ? y[i] - __half2float(hi) : 0.0f));
        }
        memcpy(__builtin_assume_aligned(a.parts + to + c, 8), h, 8);
        memcpy(__builtin_assume_aligned(low + to + c, 8), l, 8);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (c0 + i * kStep < a.cols) split(c0 + i * kStep, held[i]);
    for (int c = c0 + kHeld * kStep; c < a.cols; c += kStep) split(c, load(c));
}

// TMA reads 16-bit rows in place when their addresses and stride are multiples of 16 bytes.
bool in_place(int type, const void *x, long long x_stride, int cols) {
    return type != NVFP4_TYPE_F32 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && x_stride % 8 == 0 && x_stride >= cols;
}

size_t parts_bytes(int type, int vectors, int cols) {
    return ((size_t)vectors * cols * (type == NVFP4_TYPE_F32 ? 4 : 2) + 255) & ~size_t(255);
}

template <int TYPE, int N, bool CARRIED>
void launch_as(const GemmArgs &g, const nvfp4_matrix &matrix, const CUtensorMap &map_x, int grid, bool dependent,
            cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    allow_shared_memory(linear_gemm_kernel<TYPE, N, CARRIED>, Shape<N, TYPE == NVFP4_TYPE_F32 ? 2 : 1>::kSmem, done,
                        matrix.runtime->device, "cudaFuncSetAttribute(linear_gemm_kernel)");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kGmThreads);
    cfg.dynamicSmemBytes = Shape<N, TYPE == NVFP4_TYPE_F32 ? 2 : 1>::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    check_cuda(cudaLaunchKernelEx(&cfg, linear_gemm_kernel<TYPE, N, CARRIED>, matrix.map_w, matrix.map_s, map_x, g),
               "linear_gemm_kernel");
}

template <int TYPE, int N>
void launch(const GemmArgs &g, const nvfp4_matrix &matrix, const CUtensorMap &map_x, int grid, bool dependent,
            cudaStream_t stream) {
    if constexpr (TYPE == NVFP4_TYPE_F32) launch_as<TYPE, N, false>(g, matrix, map_x, grid, dependent, stream);
    else if (g.segment < g.k_steps) launch_as<TYPE, N, true>(g, matrix, map_x, grid, dependent, stream);
    else launch_as<TYPE, N, false>(g, matrix, map_x, grid, dependent, stream);
}

}  // namespace

size_t linear_gemm_workspace(int type, const void *x, long long x_stride, int vectors, int cols) {
    if (in_place(type, x, x_stride, cols)) return 0;
    return parts_bytes(type, vectors, cols) + (type == NVFP4_TYPE_F32 ? sizeof(float) * (size_t)vectors : 0);
}

void launch_linear_gemm(const FusedLinearArgs &f, const nvfp4_matrix &matrix, void *workspace, int sm_count,
                        cudaStream_t stream) {
    GemmArgs g{};
    g.f = f;
    const int terms = f.type == NVFP4_TYPE_F32 ? 2 : 1;  // 16-bit parts of x
    const bool small = f.type == NVFP4_TYPE_F32 || (f.offsets ? (long long)f.vectors <= 32LL * f.groups : f.vectors <= kGmSmallN);
    g.max_n = small ? kGmSmallN : kGmLargeN;
    g.m_pairs = f.gated ? (f.out_rows + 127) / 128 : (f.rows + 255) / 256;
    g.k_steps = (f.cols + 127) / 128;
    g.raw_steps = (f.cols + 255) / 256;
    const int segments = (g.k_steps + kGmSegment16 - 1) / kGmSegment16;
    g.segment = f.type == NVFP4_TYPE_F32 ? kGmSegment32 : (g.k_steps + segments - 1) / segments;
    // A CTA's half of a tile in one box (a piece that hangs over loads rows that no sum of the tile uses): fitted to the
    // even tiles of a single group, the most that a tile holds where the counts are on the device (boxes of 16 rows
    // instead: 8,192 rows over 64 groups 39.3 against 38.4 us).
    const int tiles = (f.vectors + g.max_n - 1) / g.max_n;
    g.box_rows = f.offsets ? g.max_n / 2 : ((f.vectors + tiles - 1) / tiles + 15) / 16 * 8;
    auto words = [](const void *p, long long stride) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0 && (stride & 1) == 0; };
    g.pairs_out = (f.out_rows & 1) == 0 && words(f.out, f.out_stride) && (!f.residual || words(f.residual, f.residual_stride));
    const bool direct = in_place(f.type, f.x, f.x_stride, f.cols);
    const void *rows = f.x;
    long long stride = f.x_stride;
    if (!direct) {
        SplitArgs s{};
        s.x = f.x;
        s.x_stride = f.x_stride;
        s.type = f.type;
        s.vectors = f.vectors;
        s.cols = f.cols;
        s.parts = static_cast<uint16_t *>(workspace);
        if (f.type == NVFP4_TYPE_F32)
            s.row_scale = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + parts_bytes(f.type, f.vectors, f.cols));
        g.row_scale = s.row_scale;
        linear_split_kernel<<<f.vectors, 128, 0, stream>>>(s);
        check_cuda(cudaGetLastError(), "linear_split_kernel");
        rows = workspace;
        stride = f.cols;
    }
    CUtensorMap map_x;
    check_cuda(make_tensor_map_u8(&map_x, rows, (uint64_t)f.cols * 2, (uint64_t)stride * 2,
                                  (uint64_t)f.vectors * terms, 128, g.box_rows,
                                  CU_TENSOR_MAP_SWIZZLE_128B),
               "cuTensorMapEncodeTiled(rows of x)");
    // Items the call can have: every group may end inside a tile.
    const long long x_tiles_most = tiles + (f.offsets ? std::min(f.groups, f.vectors) : 0);
    const int grid = 2 * static_cast<int>(std::min<long long>(sm_count / 2, x_tiles_most * g.m_pairs));
    if (f.type == NVFP4_TYPE_F32)
        launch<NVFP4_TYPE_F32, kGmSmallN>(g, matrix, map_x, grid, !direct, stream);
    else if (f.type == NVFP4_TYPE_BF16)
        small ? launch<NVFP4_TYPE_BF16, kGmSmallN>(g, matrix, map_x, grid, !direct, stream)
              : launch<NVFP4_TYPE_BF16, kGmLargeN>(g, matrix, map_x, grid, !direct, stream);
    else
        small ? launch<NVFP4_TYPE_F16, kGmSmallN>(g, matrix, map_x, grid, !direct, stream)
              : launch<NVFP4_TYPE_F16, kGmLargeN>(g, matrix, map_x, grid, !direct, stream);
}

}  // namespace nvfp4
