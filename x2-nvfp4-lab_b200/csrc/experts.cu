// Token rows sorted by expert and brought back, with the gradients of both.
//
//   sort      rows[p] = x[perm[p] / K]          perm: the T*K picks in expert order, stable (token order within an
//                                               expert), -1 past the last expert's rows; inverse[t, k] = the row of
//                                               pick (t, k), -1 where its id is no expert; offsets[e] = the first
//                                               row of expert e, offsets[E] = the number of rows in use
//   its dx    dx[t]   = sum_k drows[inverse[t, k]]                          (the return with weights of one)
//   return    out[t]  = residual[t] + sum_k w[t, k] * rows[inverse[t, k]]
//   its dX    drows[inverse[t, k]] = w[t, k] * dout[t],  dw[t, k] = <dout[t], rows[inverse[t, k]]>; zero in rows that
//             no pick names (a pick may be set to -1 after the sort)
//
// Every kernel moves T*K rows of H values once and does next to nothing with them, so HBM bounds them. One group of
// threads owns a token: the sort reads a token's row once and stores it K times, the return reads its K rows and
// stores one, the gradient reads dout once beside K rows. Sums are FP32 in the order of k (of columns, for dw, in a
// fixed tree): no atomics touch a result, so two calls give the same bits.
#include "internal.h"
#include "nvfp4_common.cuh"
#include "tma_util.cuh"

#include <algorithm>
#include <climits>

namespace nvfp4 {
namespace {

constexpr int kExThreads = 256;
constexpr int kExMaxTopk = 64;
constexpr int kExMaxExperts = 1024;
constexpr int kExWarps = kExThreads / 32;
constexpr int kExRows = 8;  // picks of a token that a thread handles together
// Picks whose ranks one launch finds by comparing every pick with every other (a warp per pick): each CTA does it for
// its own token from a shared-memory copy of the ids, so nothing waits on another launch.
constexpr int kExSmallPicks = 4096;

// Row of a pick: -1 for a dropped one, and for a number that no sort of this many picks writes.
__device__ __forceinline__ int row_of(const int *inverse, long long pick, int picks) {
    const int p = __ldg(inverse + pick);
    return static_cast<unsigned>(p) < static_cast<unsigned>(picks) ? p : -1;
}

// Expert of a pick, `experts` where the id names none.
__device__ __forceinline__ int pick_key(const void *ids, int wide, long long ids_stride, int topk, int pick,
                                        int experts) {
    long long at = pick;
    if (ids_stride != topk) {
        const int t = pick / topk;
        at = (long long)t * ids_stride + (pick - t * topk);
    }
    const long long id = wide ? static_cast<const long long *>(ids)[at] : (long long)static_cast<const int *>(ids)[at];
    return id >= 0 && id < experts ? (int)id : experts;
}

// ------------------------------------------------------------------ vectors of B bytes

template <int B>
struct Vec;
template <>
struct Vec<16> {
    using type = uint4;
};
template <>
struct Vec<8> {
    using type = uint2;
};
template <>
struct Vec<4> {
    using type = uint32_t;
};
template <>
struct Vec<2> {
    using type = uint16_t;
};

enum : int { kBf16 = NVFP4_TYPE_BF16, kF16 = NVFP4_TYPE_F16, kF32 = NVFP4_TYPE_F32 };

template <int TYPE>
__device__ __forceinline__ float get1(const void *p, size_t i) {
    if constexpr (TYPE == kF32) return static_cast<const float *>(p)[i];
    if constexpr (TYPE == kF16) return __half2float(static_cast<const __half *>(p)[i]);
    if constexpr (TYPE == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

__device__ __forceinline__ float get_any(const void *p, int type, size_t i) {
    return type == kF32 ? get1<kF32>(p, i) : type == kF16 ? get1<kF16>(p, i) : get1<kBf16>(p, i);
}

__device__ __forceinline__ void put_any(void *p, int type, size_t i, float v) {
    if (type == kF32) static_cast<float *>(p)[i] = v;
    else if (type == kF16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// B bytes as FP32 values, and back with one rounding each.
template <int TYPE, int B>
struct Lane {
    static constexpr int kN = B / (TYPE == kF32 ? 4 : 2);
    using V = typename Vec<B>::type;
    __device__ static __forceinline__ void unpack(const V &v, float (&f)[kN]) {
        if constexpr (TYPE == kF32) {
            memcpy(f, &v, B);
        } else {
            uint16_t h[kN];
            memcpy(h, &v, B);
#pragma unroll
            for (int i = 0; i < kN; ++i)
                f[i] = TYPE == kF16 ? __half2float(__ushort_as_half(h[i])) : bf16_bits_to_f32(h[i]);
        }
    }
    __device__ static __forceinline__ V pack(const float (&f)[kN]) {
        V v;
        if constexpr (TYPE == kF32) {
            memcpy(&v, f, B);
        } else {
            uint16_t h[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i)
                h[i] = TYPE == kF16 ? __half_as_ushort(__float2half_rn(f[i])) : f32_to_bf16_bits(f[i]);
            memcpy(&v, h, B);
        }
        return v;
    }
};

template <typename V>
__device__ __forceinline__ V zero_vec() {
    V v;
    memset(&v, 0, sizeof(V));
    return v;
}

// ------------------------------------------------------------------ sort

struct SortArgs {
    const uint8_t *x;
    uint8_t *rows;
    const void *ids;
    int *perm;
    int *inverse;
    int *offsets;
    long long x_stride;    // bytes
    long long ids_stride;  // elements
    int ids_wide;
    int tokens, topk, experts, picks;
    int row_bytes;
    int per_warp;           // picks a warp ranks, a multiple of 32
    int group;              // threads that share a token in the copy launch
};

// One launch for few picks: CTA t ranks token t's picks and copies its row; the last CTA writes the offsets.
template <int B>
__global__ void __launch_bounds__(kExThreads) expert_sort_small_kernel(SortArgs a) {
    using V = typename Vec<B>::type;
    __shared__ int key[kExSmallPicks];
    __shared__ int count[kExMaxExperts + 1];
    __shared__ int place[kExMaxTopk];
    __shared__ int warp_sum[kExWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool totals = (int)blockIdx.x == a.tokens;
    if (totals)
        for (int e = threadIdx.x; e <= a.experts; e += kExThreads) count[e] = 0;
    for (int i = threadIdx.x; i < a.picks; i += kExThreads)
        key[i] = pick_key(a.ids, a.ids_wide, a.ids_stride, a.topk, i, a.experts);
    __syncthreads();
    if (totals) {
        for (int i = threadIdx.x; i < a.picks; i += kExThreads) atomicAdd(&count[key[i]], 1);
        __syncthreads();
        // Exclusive sum over the experts: each thread a run of them, then the warps' sums.
        const int per = (a.experts + kExThreads) / kExThreads;
        const int e0 = threadIdx.x * per, e1 = min(e0 + per, a.experts + 1);
        int own = 0;
        for (int e = e0; e < e1; ++e) own += count[e];
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        int base = upto - own;
        for (int w = 0; w < warp; ++w) base += warp_sum[w];
        for (int e = e0; e < e1; ++e) {
            a.offsets[e] = base;
            base += count[e];
        }
        return;
    }
    const int t = blockIdx.x;
    for (int k = warp; k < a.topk; k += kExWarps) {
        const int pick = t * a.topk + k, mine = key[pick];
        int before = 0;
        for (int i = lane; i < a.picks; i += 32) before += key[i] < mine || (key[i] == mine && i < pick) ? 1 : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
        if (lane == 0) {
            const bool used = mine < a.experts;
            place[k] = used ? before : ~before;  // a dropped pick's row, past the last expert's, is zero
            a.inverse[pick] = used ? before : -1;
            a.perm[before] = used ? pick : -1;
        }
    }
    __syncthreads();
    const int nvec = a.row_bytes / B;
    const V *src = reinterpret_cast<const V *>(a.x + (long long)t * a.x_stride);
    for (int v = threadIdx.x; v < nvec; v += kExThreads) {
        const V val = src[v];
        for (int k = 0; k < a.topk; ++k) {
            const int p = place[k];
            const bool used = p >= 0;
            reinterpret_cast<V *>(a.rows + (long long)(used ? p : ~p) * a.row_bytes)[v] = used ? val : zero_vec<V>();
        }
    }
}

constexpr int kRankCtas = 8, kRankThreads = 1024, kRankWarps = kRankThreads / 32;
constexpr int kRankKeys = 8;  // picks a lane holds at a time

// Lanes of the warp with this lane's key, a ballot per bit (match.any takes about 80 cycles an SM for each warp).
__device__ __forceinline__ unsigned lanes_with(int key, int bits) {
    unsigned same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool one = (key >> b) & 1;
        const unsigned ones = __ballot_sync(0xffffffffu, one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// Many picks, first launch: one cluster ranks them all. A warp owns consecutive picks and counts them; the warps' counts
// add up in the CTA, the CTAs' through distributed shared memory; then every warp walks its picks again, 32 at a time,
// and places them in order.
__global__ void __launch_bounds__(kRankThreads, 1) expert_rank_kernel(SortArgs a) {
    extern __shared__ int rank_smem[];
    const int n = a.experts + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = (int)cluster_rank();
    int *block = rank_smem;       // [experts + 1] picks of this CTA, read by the others
    int *base = block + n;        // [experts + 1] first row of this CTA's picks
    int *counts = base + n;       // [warps][experts + 1] a warp's picks, then the place of its next one
    __shared__ int warp_sum[kRankWarps];
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < kRankWarps * n; i += kRankThreads) counts[i] = 0;
    __syncthreads();
    const long long first = (long long)(cta * kRankWarps + warp) * a.per_warp;
    const long long last = min(first + a.per_warp, (long long)a.picks);
    int *mine = counts + warp * n;
    const int bits = 32 - __clz(n);
    int key[kRankKeys];
    auto load_keys = [&](long long i) {
#pragma unroll
        for (int u = 0; u < kRankKeys; ++u) {
            const long long pick = i + 32 * u + lane;
            key[u] = pick < last ? pick_key(a.ids, a.ids_wide, a.ids_stride, a.topk, (int)pick, a.experts) : -1;
        }
    };
    for (long long i = first; i < last; i += 32 * kRankKeys) {
        load_keys(i);
#pragma unroll
        for (int u = 0; u < kRankKeys; ++u) {
            if (key[u] >= 0) atomicAdd(mine + key[u], 1);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += kRankThreads) {
        int run = 0;
#pragma unroll 8
        for (int w = 0; w < kRankWarps; ++w) {
            const int c = counts[w * n + e];
            counts[w * n + e] = run;
            run += c;
        }
        block[e] = run;
    }
    cluster_sync();
    // A thread's experts are consecutive (one, or two past 1023), so that the sum over earlier experts is a scan.
    const int per = (n + kRankThreads - 1) / kRankThreads;
    const int e0 = min((int)threadIdx.x * per, n), e1 = min(e0 + per, n);
    int own = 0;
    for (int e = e0; e < e1; ++e) {
        int before = 0, all = 0;
#pragma unroll
        for (int r = 0; r < kRankCtas; ++r) {
            const int c = load_cluster(block + e, r);
            before += r < cta ? c : 0;
            all += c;
        }
        base[e] = own + before;
        own += all;
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int start = upto - own;
    for (int w = 0; w < warp; ++w) start += warp_sum[w];
    for (int e = e0; e < e1; ++e) {
        base[e] += start;
        if (cta == 0) a.offsets[e] = base[e];  // no CTA's picks come before the first one's
    }
    __syncthreads();
    for (long long i = first; i < last; i += 32 * kRankKeys) {
        if (a.per_warp > 32 * kRankKeys) load_keys(i);  // else they are still in registers
#pragma unroll
        for (int u = 0; u < kRankKeys; ++u) {
            if (i + 32 * u >= last) break;
            // Picks past the last have a key of their own.
            const unsigned same = lanes_with(key[u] >= 0 ? key[u] : n, bits);
            const int row = key[u] >= 0 ? base[key[u]] + mine[key[u]] + __popc(same & ((1u << lane) - 1u)) : 0;
            __syncwarp();
            if (key[u] >= 0) {
                const int pick = (int)(i + 32 * u) + lane;
                const bool used = key[u] < a.experts;
                a.inverse[pick] = used ? row : -1;
                a.perm[row] = used ? pick : -1;
                if (lane == __ffs(same) - 1) mine[key[u]] += __popc(same);
            }
            __syncwarp();
        }
    }
    cluster_sync();  // no CTA leaves while another may read its counts
}

// Second launch: each token's row to its picks' rows, and zeros to the rows past the last expert's. A group of
// threads owns a token.
template <int B>
__global__ void __launch_bounds__(kExThreads) expert_copy_kernel(SortArgs a) {
    using V = typename Vec<B>::type;
    const int per_cta = kExThreads / a.group;
    const int t = blockIdx.x * per_cta + threadIdx.x / a.group, lane = threadIdx.x % a.group;
    if (t >= a.tokens) return;
    const int nvec = a.row_bytes / B;
    const V *src = reinterpret_cast<const V *>(a.x + (long long)t * a.x_stride);
    V val = lane < nvec ? src[lane] : zero_vec<V>();  // x depends on no earlier launch of this call
    pdl_wait();
    const int used = __ldcg(a.offsets + a.experts);
    for (int k0 = 0; k0 < a.topk; k0 += kExRows) {
        int p[kExRows];
#pragma unroll
        for (int j = 0; j < kExRows; ++j) p[j] = k0 + j < a.topk ? __ldcg(a.inverse + (long long)t * a.topk + k0 + j) : -1;
        for (int v = lane; v < nvec; v += a.group) {
            if (v != lane || k0 > 0) val = src[v];
#pragma unroll
            for (int j = 0; j < kExRows; ++j) {
                if (p[j] >= 0) reinterpret_cast<V *>(a.rows + (long long)p[j] * a.row_bytes)[v] = val;
                const int r = t * a.topk + k0 + j;
                if (k0 + j < a.topk && r >= used) reinterpret_cast<V *>(a.rows + (long long)r * a.row_bytes)[v] = zero_vec<V>();
            }
        }
    }
}

// ------------------------------------------------------------------ return and its gradient

struct ReturnArgs {
    const uint8_t *rows;
    const uint8_t *residual;
    const uint8_t *dout;
    const int *inverse;
    const int *offsets;
    const void *weights;
    void *dweights;
    uint8_t *out;
    uint8_t *drows;
    long long rows_stride, residual_stride, out_stride, dout_stride;  // bytes
    int weight_type;
    int tokens, topk, experts;
    int row_bytes;
    int group;
};


template <int TYPE, int B>
__global__ void __launch_bounds__(kExThreads) expert_return_kernel(ReturnArgs a) {
    using L = Lane<TYPE, B>;
    using V = typename Vec<B>::type;
    const int per_cta = kExThreads / a.group;
    const int t = blockIdx.x * per_cta + threadIdx.x / a.group, lane = threadIdx.x % a.group;
    if (t >= a.tokens) return;
    const int nvec = a.row_bytes / B;
    const long long pick0 = (long long)t * a.topk;
    for (int v = lane; v < nvec; v += a.group) {
        float sum[L::kN];
        if (a.residual) {
            L::unpack(reinterpret_cast<const V *>(a.residual + (long long)t * a.residual_stride)[v], sum);
        } else {
#pragma unroll
            for (int i = 0; i < L::kN; ++i) sum[i] = 0.0f;
        }
        for (int k0 = 0; k0 < a.topk; k0 += kExRows) {
            V val[kExRows];
            int p[kExRows];
#pragma unroll
            for (int j = 0; j < kExRows; ++j) {
                p[j] = k0 + j < a.topk ? row_of(a.inverse, pick0 + k0 + j, a.tokens * a.topk) : -1;
                if (p[j] >= 0) val[j] = reinterpret_cast<const V *>(a.rows + (long long)p[j] * a.rows_stride)[v];
            }
#pragma unroll
            for (int j = 0; j < kExRows; ++j) {
                if (p[j] < 0) continue;
                float f[L::kN];
                L::unpack(val[j], f);
                const float w = a.weights ? get_any(a.weights, a.weight_type, pick0 + k0 + j) : 1.0f;
#pragma unroll
                for (int i = 0; i < L::kN; ++i) sum[i] = fmaf(w, f[i], sum[i]);
            }
        }
        reinterpret_cast<V *>(a.out + (long long)t * a.out_stride)[v] = L::pack(sum);
    }
}

// Zeros to the rows of drows below offsets[experts] that no pick names: those of picks dropped after the sort. There are
// none in an order as the sort made it, and then the kernel only counts: a cluster's CTAs a share of the picks each, their
// counts added up through distributed shared memory, and the gradient kernel, launched behind it, waits for that before
// its first store, with its loads under way (4,096 tokens with eight BF16 rows of 2,048: 54.1 us both, 54.6 without the
// count and the loads ahead; 32 tokens 6.1 against 5.3). Else each CTA marks which of its own rows are named, a bit a row,
// from the picks of all (61.8 us with a tenth of the picks dropped).
constexpr int kUnnamedThreads = 512, kUnnamedCluster = 8;
constexpr int kUnnamedWords = 8192;  // 262,144 rows marked at a time

template <int B>
__global__ void __launch_bounds__(kUnnamedThreads) expert_unnamed_rows_kernel(ReturnArgs a) {
    using V = typename Vec<B>::type;
    __shared__ uint32_t named[kUnnamedWords];
    __shared__ int count;
    pdl_launch_dependents();
    const int picks = a.tokens * a.topk, rank = (int)cluster_rank();
    const int used = min(max(__ldg(a.offsets + a.experts), 0), picks);
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    int own = 0;
#pragma unroll 4
    for (long long i = rank * kUnnamedThreads + (int)threadIdx.x; i < picks; i += kUnnamedCluster * kUnnamedThreads)
        own += (unsigned)__ldg(a.inverse + i) < (unsigned)used ? 1 : 0;
    own = __reduce_add_sync(0xffffffffu, own);
    if ((threadIdx.x & 31) == 0 && own != 0) atomicAdd(&count, own);
    cluster_sync();
    int all = 0;
#pragma unroll
    for (int r = 0; r < kUnnamedCluster; ++r) all += load_cluster(&count, r);
    cluster_sync();  // no CTA leaves while another may read its count
    if (all == used) return;
    const long long first = (long long)used * blockIdx.x / gridDim.x, last = (long long)used * (blockIdx.x + 1) / gridDim.x;
    const int nvec = a.row_bytes / B;
    for (long long r0 = first; r0 < last; r0 += 32 * kUnnamedWords) {
        const int n = (int)min(last - r0, 32LL * kUnnamedWords);
        for (int i = threadIdx.x; i < (n + 31) / 32; i += kUnnamedThreads) named[i] = 0u;
        __syncthreads();
        for (long long i = threadIdx.x; i < picks; i += kExRows * kUnnamedThreads) {
            unsigned at[kExRows];
#pragma unroll
            for (int u = 0; u < kExRows; ++u) {
                const long long pick = i + u * kUnnamedThreads;
                at[u] = (pick < picks ? (unsigned)__ldg(a.inverse + pick) : ~0u) - (unsigned)r0;
            }
#pragma unroll
            for (int u = 0; u < kExRows; ++u)
                if (at[u] < (unsigned)n) atomicOr(named + (at[u] >> 5), 1u << (at[u] & 31));
        }
        __syncthreads();
        for (int r = threadIdx.x >> 5; r < n; r += kUnnamedThreads / 32) {
            if ((named[r >> 5] >> (r & 31)) & 1u) continue;
            V *to = reinterpret_cast<V *>(a.drows + (r0 + r) * a.row_bytes);
            for (int v = threadIdx.x & 31; v < nvec; v += 32) to[v] = zero_vec<V>();
        }
        __syncthreads();
    }
}

// The gradient keeps four rows' loads in flight per thread and four CTAs on an SM: with eight rows its 166 registers
// left one CTA, and 4,096 tokens with eight BF16 rows of 2,048 took 136 us instead of 59.
constexpr int kExBackRows = 4;

template <int TYPE, int B>
__global__ void __launch_bounds__(kExThreads, 4) expert_return_backward_kernel(ReturnArgs a) {
    using L = Lane<TYPE, B>;
    using V = typename Vec<B>::type;
    __shared__ float part[kExWarps][kExBackRows];
    const int per_cta = kExThreads / a.group;
    const int sub = threadIdx.x / a.group;
    const int t = blockIdx.x * per_cta + sub, lane = threadIdx.x % a.group;
    const bool live = t < a.tokens;
    const int nvec = live ? a.row_bytes / B : 0;
    const long long pick0 = (long long)t * a.topk;
    const V *dout = reinterpret_cast<const V *>(a.dout + (long long)t * a.dout_stride);
    const int used = a.drows ? __ldg(a.offsets + a.experts) : INT_MAX;
    for (int k0 = 0; k0 < a.topk; k0 += kExBackRows) {
        int p[kExBackRows];
        float w[kExBackRows], dot[kExBackRows];
#pragma unroll
        for (int j = 0; j < kExBackRows; ++j) {
            p[j] = live && k0 + j < a.topk ? row_of(a.inverse, pick0 + k0 + j, a.tokens * a.topk) : -1;
            w[j] = p[j] >= 0 && a.weights ? get_any(a.weights, a.weight_type, pick0 + k0 + j) : 1.0f;
            dot[j] = 0.0f;
        }
        for (int v = lane; v < nvec; v += a.group) {
            V val[kExBackRows];
            if (a.dweights) {
#pragma unroll
                for (int j = 0; j < kExBackRows; ++j)
                    if (p[j] >= 0) val[j] = reinterpret_cast<const V *>(a.rows + (long long)p[j] * a.rows_stride)[v];
            }
            const V dv = dout[v];
            pdl_wait();  // the zeros of rows that no pick names; what is read above depends on no launch of this call
            float g[L::kN];
            L::unpack(dv, g);
#pragma unroll
            for (int j = 0; j < kExBackRows; ++j) {
                if (a.drows && p[j] >= 0) {
                    float d[L::kN];
#pragma unroll
                    for (int i = 0; i < L::kN; ++i) d[i] = w[j] * g[i];
                    reinterpret_cast<V *>(a.drows + (long long)p[j] * a.row_bytes)[v] = L::pack(d);
                }
                // Rows past the last expert's have no gradient.
                if (k0 + j < a.topk && pick0 + k0 + j >= used)
                    reinterpret_cast<V *>(a.drows + (pick0 + k0 + j) * a.row_bytes)[v] = zero_vec<V>();
            }
            if (a.dweights) {
#pragma unroll
                for (int j = 0; j < kExBackRows; ++j) {
                    if (p[j] < 0) continue;
                    float f[L::kN];
                    L::unpack(val[j], f);
#pragma unroll
                    for (int i = 0; i < L::kN; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
                }
            }
        }
        if (a.dweights) {
            // The rows' sums over the lanes that share the token: two halving steps leave each lane one row, the rest add.
            int o = min(a.group, 32) >> 1, row = 0;
            float sum[kExBackRows];
#pragma unroll
            for (int j = 0; j < kExBackRows; ++j) sum[j] = dot[j];
#pragma unroll
            for (int half = kExBackRows / 2; half > 0; half >>= 1, o >>= 1) {
                const bool upper = (threadIdx.x & o) != 0;
                row += upper ? half : 0;
#pragma unroll
                for (int j = 0; j < half; ++j) {
                    const float send = upper ? sum[j] : sum[j + half], keep = upper ? sum[j + half] : sum[j];
                    sum[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
            }
            const bool first_of_row = (threadIdx.x & (2 * o - 1)) == 0;  // of the lanes that hold the same row
            for (; o > 0; o >>= 1) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
            if (a.group > 32) {
                if (first_of_row) part[threadIdx.x >> 5][row] = sum[0];
                __syncthreads();
                if (lane < kExBackRows) {
                    float s = 0.0f;
                    for (int i = 0; i < a.group / 32; ++i) s += part[sub * (a.group / 32) + i][lane];
                    if (live && k0 + lane < a.topk) put_any(a.dweights, a.weight_type, pick0 + k0 + lane, s);
                }
                __syncthreads();
            } else if (first_of_row && live && k0 + row < a.topk) {
                put_any(a.dweights, a.weight_type, pick0 + k0 + row, sum[0]);
            }
        }
    }
}

// ------------------------------------------------------------------ host

int type_bytes(int type) { return type == kF32 ? 4 : 2; }
bool valid_type(int type) { return type == kBf16 || type == kF16 || type == kF32; }

// Widest vector (bytes, at most 16) that divides the row, the strides and the addresses of a call.
int vector_bytes(std::initializer_list<unsigned long long> places) {
    unsigned long long all = 16;
    for (unsigned long long p : places) all |= p;
    return static_cast<int>(all & (~all + 1));  // lowest set bit, at most 16
}
unsigned long long place_of(const void *p) { return reinterpret_cast<uintptr_t>(p); }
// Whether every address (NULL too) is a multiple of an element's bytes: a kernel that took another would fault.
bool aligned_to(int bytes, std::initializer_list<const void *> addresses) {
    for (const void *p : addresses)
        if (place_of(p) % bytes != 0) return false;
    return true;
}
constexpr const char *kMisaligned = "arrays of the expert sort and return must be aligned to their elements";

// Threads that share a token: a power of two near its vectors, from 8 to a whole CTA.
int group_of(int nvec) {
    int g = 8;
    while (g < kExThreads && g < nvec) g <<= 1;
    return g;
}

template <typename Args>
void launch(void (*kernel)(Args), int grid, cudaStream_t stream, bool dependent, const Args &args, const char *name) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kExThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    check_cuda(cudaLaunchKernelEx(&cfg, kernel, args), name);
}

template <int B>
void launch_sort(SortArgs &a, int device, cudaStream_t s) {
    a.group = group_of(a.row_bytes / B);
    if (a.picks <= kExSmallPicks) {
        launch(expert_sort_small_kernel<B>, a.tokens + 1, s, false, a, "expert_sort_small_kernel");
        return;
    }
    const size_t smem = sizeof(int) * (kRankWarps + 2) * (a.experts + 1);
    static std::atomic<uint64_t> done{0};
    allow_shared_memory(expert_rank_kernel, sizeof(int) * (kRankWarps + 2) * (kExMaxExperts + 1), done, device,
                        "cudaFuncSetAttribute(expert_rank_kernel)");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kRankCtas);
    cfg.blockDim = dim3(kRankThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kRankCtas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    check_cuda(cudaLaunchKernelEx(&cfg, expert_rank_kernel, a), "expert_rank_kernel");
    const int per_cta = kExThreads / a.group;
    launch(expert_copy_kernel<B>, (a.tokens + per_cta - 1) / per_cta, s, true, a, "expert_copy_kernel");
}

template <int B>
void launch_unnamed_rows(const ReturnArgs &a, cudaStream_t s) {
    // A cluster for every 8,192 picks, up to 16: more than one only pay where rows are zeroed (both kernels at 4,096 x 8
    // rows of 128 bytes: 5.8 us with one, 7.0 with five, 7.4 with 16; a tenth of the picks dropped 34, 16.7 and 14.1 us).
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kUnnamedCluster * std::min(1 + a.tokens * a.topk / 8192, 16));
    cfg.blockDim = dim3(kUnnamedThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kUnnamedCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    check_cuda(cudaLaunchKernelEx(&cfg, expert_unnamed_rows_kernel<B>, a), "expert_unnamed_rows_kernel");
}

template <int TYPE, int B>
void launch_return(ReturnArgs &a, bool backward, cudaStream_t s) {
    a.group = group_of(a.row_bytes / B);
    // The weights' gradient ends in a sum over the threads of a token: one warp a token, once
    // tokens give every SM 16 of them and rows are no longer than 16 vectors a lane (4,096 tokens with eight BF16 rows
    // of 2,048: 55 us, 59 us with a CTA a token).
    if (backward && a.tokens >= 2368 && a.row_bytes / B <= 512) a.group = std::min(a.group, 32);
    const int per_cta = kExThreads / a.group, grid = (a.tokens + per_cta - 1) / per_cta;
    if (backward) {
        if (a.drows) launch_unnamed_rows<B>(a, s);
        launch(expert_return_backward_kernel<TYPE, B>, grid, s, a.drows != nullptr, a, "expert_return_backward_kernel");
    } else {
        launch(expert_return_kernel<TYPE, B>, grid, s, false, a, "expert_return_kernel");
    }
}

// `vec` is an element at least: the entry points refuse addresses off their elements.
template <int TYPE>
void dispatch_return(ReturnArgs &a, int vec, bool backward, cudaStream_t s) {
    if (vec == 16) launch_return<TYPE, 16>(a, backward, s);
    else if (vec == 8) launch_return<TYPE, 8>(a, backward, s);
    else if (TYPE == kF32 || vec == 4) launch_return<TYPE, 4>(a, backward, s);
    else if constexpr (TYPE != kF32) launch_return<TYPE, 2>(a, backward, s);
}

void run_return(ReturnArgs &a, int type, int vec, bool backward, cudaStream_t s) {
    if (type == kBf16) dispatch_return<kBf16>(a, vec, backward, s);
    else if (type == kF16) dispatch_return<kF16>(a, vec, backward, s);
    else dispatch_return<kF32>(a, vec, backward, s);
}

bool valid_sizes(int type, int tokens, int topk, int hidden) {
    return valid_type(type) && tokens > 0 && topk > 0 && topk <= kExMaxTopk && hidden > 0 && hidden <= (1 << 24) &&
           static_cast<long long>(tokens) * topk < INT_MAX - 16384;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" NVFP4_API nvfp4_status nvfp4_expert_sort(nvfp4_runtime *runtime, const void *x, int type, int64_t x_stride,
                                                    int tokens, int hidden, const void *ids, int ids_bytes,
                                                    int64_t ids_stride, int topk, int experts, void *rows,
                                                    int32_t *perm, int32_t *inverse, int32_t *offsets, void *stream) {
    if (!runtime || !x || !ids || !rows || !perm || !inverse || !offsets || !valid_sizes(type, tokens, topk, hidden) ||
        (ids_bytes != 4 && ids_bytes != 8) || ids_stride < 0 || x_stride < 0)
        return fail_invalid("invalid expert sort arguments");
    if (experts < 1 || experts > kExMaxExperts) return fail_invalid("the expert sort supports 1 to 1024 experts");
    if (!aligned_to(type_bytes(type), {x, rows}) || !aligned_to(ids_bytes, {ids}) ||
        !aligned_to(4, {perm, inverse, offsets}))
        return fail_invalid(kMisaligned);
    try {
        const device_scope scope(runtime);
        check_on_device(runtime, {x, ids, rows}, "expert sort");
        SortArgs a{};
        a.x = static_cast<const uint8_t *>(x);
        a.rows = static_cast<uint8_t *>(rows);
        a.ids = ids;
        a.perm = perm;
        a.inverse = inverse;
        a.offsets = offsets;
        a.x_stride = x_stride * type_bytes(type);
        a.ids_stride = ids_stride;
        a.ids_wide = ids_bytes == 8;
        a.tokens = tokens;
        a.topk = topk;
        a.experts = experts;
        a.picks = tokens * topk;
        a.row_bytes = hidden * type_bytes(type);
        a.per_warp = ((a.picks + kRankCtas * kRankWarps - 1) / (kRankCtas * kRankWarps) + 31) / 32 * 32;
        const int vec = vector_bytes({place_of(x), place_of(rows), static_cast<unsigned long long>(a.x_stride),
                                      static_cast<unsigned long long>(a.row_bytes)});
        std::lock_guard<std::mutex> lock(runtime->queue_mutex);
        runtime->direct_call(static_cast<cudaStream_t>(stream), [&](cudaStream_t os) {
            runtime->profiled_kernel("expert_sort", os, [&](cudaStream_t s) {
                if (vec == 16) launch_sort<16>(a, runtime->device, s);
                else if (vec == 8) launch_sort<8>(a, runtime->device, s);
                else if (vec == 4) launch_sort<4>(a, runtime->device, s);
                else launch_sort<2>(a, runtime->device, s);
            });
        });
        clear_last_error();
        return NVFP4_STATUS_OK;
    } catch (const std::exception &error) {
        return fail_exception(error);
    }
}

extern "C" NVFP4_API nvfp4_status nvfp4_expert_return(nvfp4_runtime *runtime, const void *rows, int type,
                                                      int64_t rows_stride, const int32_t *inverse,
                                                      const void *weights, int weights_type, const void *residual,
                                                      int64_t residual_stride, int tokens, int topk, int hidden,
                                                      void *out, int64_t out_stride, void *stream) {
    if (!runtime || !rows || !inverse || !out || !valid_sizes(type, tokens, topk, hidden) ||
        (weights && !valid_type(weights_type)) || rows_stride < 0 || residual_stride < 0 || out_stride < hidden)
        return fail_invalid("invalid expert return arguments");
    if (!aligned_to(type_bytes(type), {rows, residual, out}) || !aligned_to(4, {inverse}) ||
        (weights && !aligned_to(type_bytes(weights_type), {weights})))
        return fail_invalid(kMisaligned);
    const long long row = static_cast<long long>(hidden) * type_bytes(type), picks = static_cast<long long>(tokens) * topk;
    const row_span to{out, tokens, row, out_stride * type_bytes(type)};
    if (spans_overlap({rows, picks, row, rows_stride * type_bytes(type)}, to))
        return fail_invalid("expert return: out must not overlap the rows");
    if (!(residual == out && (residual_stride == out_stride || tokens == 1)) &&
        spans_overlap({residual, tokens, row, residual_stride * type_bytes(type)}, to))
        return fail_invalid("expert return: the residual is out itself or does not overlap it");
    try {
        const device_scope scope(runtime);
        check_on_device(runtime, {rows, out}, "expert return");
        const int e = type_bytes(type);
        ReturnArgs a{};
        a.rows = static_cast<const uint8_t *>(rows);
        a.residual = static_cast<const uint8_t *>(residual);
        a.inverse = inverse;
        a.weights = weights;
        a.weight_type = weights_type;
        a.out = static_cast<uint8_t *>(out);
        a.rows_stride = rows_stride * e;
        a.residual_stride = residual_stride * e;
        a.out_stride = out_stride * e;
        a.tokens = tokens;
        a.topk = topk;
        a.row_bytes = hidden * e;
        const int vec = vector_bytes({place_of(rows), place_of(out), place_of(residual),
                                      static_cast<unsigned long long>(a.rows_stride),
                                      static_cast<unsigned long long>(residual ? a.residual_stride : 0),
                                      static_cast<unsigned long long>(a.out_stride),
                                      static_cast<unsigned long long>(a.row_bytes)});
        std::lock_guard<std::mutex> lock(runtime->queue_mutex);
        runtime->direct_call(static_cast<cudaStream_t>(stream), [&](cudaStream_t os) {
            runtime->profiled_kernel("expert_return", os,
                                     [&](cudaStream_t s) { run_return(a, type, vec, false, s); });
        });
        clear_last_error();
        return NVFP4_STATUS_OK;
    } catch (const std::exception &error) {
        return fail_exception(error);
    }
}

extern "C" NVFP4_API nvfp4_status nvfp4_expert_return_backward(
    nvfp4_runtime *runtime, const void *dout, int type, int64_t dout_stride, const void *rows, int64_t rows_stride,
    const int32_t *inverse, const int32_t *offsets, const void *weights, int weights_type, int tokens, int topk,
    int hidden, int experts, void *drows, void *dweights, void *stream) {
    if (!runtime || !dout || !inverse || (!drows && !dweights) || (drows && (!offsets || experts < 1)) ||
        (dweights && !rows) || !valid_sizes(type, tokens, topk, hidden) ||
        ((weights || dweights) && !valid_type(weights_type)) || dout_stride < 0 || rows_stride < 0)
        return fail_invalid("invalid expert return gradient arguments");
    if (!aligned_to(type_bytes(type), {dout, rows, drows}) || !aligned_to(4, {inverse, offsets}) ||
        ((weights || dweights) && !aligned_to(type_bytes(weights_type), {weights, dweights})))
        return fail_invalid(kMisaligned);
    try {
        const device_scope scope(runtime);
        check_on_device(runtime, {dout, drows ? drows : dweights}, "expert return gradient");
        const int e = type_bytes(type);
        ReturnArgs a{};
        a.dout = static_cast<const uint8_t *>(dout);
        a.rows = static_cast<const uint8_t *>(rows);
        a.inverse = inverse;
        a.offsets = offsets;
        a.weights = weights;
        a.weight_type = weights_type;
        a.dweights = dweights;
        a.drows = static_cast<uint8_t *>(drows);
        a.dout_stride = dout_stride * e;
        a.rows_stride = rows_stride * e;
        a.tokens = tokens;
        a.topk = topk;
        a.experts = experts;
        a.row_bytes = hidden * e;
        const int vec = vector_bytes({place_of(dout), dweights ? place_of(rows) : 0, place_of(drows),
                                      static_cast<unsigned long long>(a.dout_stride),
                                      static_cast<unsigned long long>(dweights ? a.rows_stride : 0),
                                      static_cast<unsigned long long>(a.row_bytes)});
        std::lock_guard<std::mutex> lock(runtime->queue_mutex);
        runtime->direct_call(static_cast<cudaStream_t>(stream), [&](cudaStream_t os) {
            runtime->profiled_kernel("expert_return_backward", os,
                                     [&](cudaStream_t s) { run_return(a, type, vec, true, s); });
        });
        clear_last_error();
        return NVFP4_STATUS_OK;
    } catch (const std::exception &error) {
        return fail_exception(error);
    }
}
