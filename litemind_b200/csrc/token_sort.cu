// token_sort.cu -- tokens sorted by expert and back, with the routing weights, and the
// gradients of both (lm_moe_sort_plan, lm_moe_sort_rows, lm_moe_unsort_rows,
// lm_moe_unsort_rows_backward).
//
// The plan is a stable counting sort of the (token, slot) pairs by expert: pair p goes to row
//   at[p] = pairs of smaller experts + earlier pairs of the same expert,
// and pairs whose expert is outside [0, experts) get -1 (dropped).  Nothing is ordered by
// atomics, so the same input always gives the same rows.
#include "moe_internal.h"
#include "elem.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <cstdio>

namespace lm {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanMaxExperts = 1024;
constexpr int kPlanCluster = 8;
constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

// This CTA's `v[i]` (shared memory) as seen by the cluster's CTA `rank`.
__device__ __forceinline__ int ld_cluster(const int* v, uint32_t rank) {
    int r;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(r) : "r"(mapa_shared(smem_u32(v), rank)) : "memory");
    return r;
}

// The lanes of the warp that hold the same x: a vote for each bit.  (With __match_any_sync each
// pass took half as long again.)
__device__ __forceinline__ unsigned same_lanes(unsigned x, int bits) {
    unsigned m = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool set = x >> b & 1u;
        const unsigned v = __ballot_sync(0xffffffffu, set);
        m &= set ? v : ~v;
    }
    return m;
}

// One cluster.  Each warp takes a contiguous run of pairs, counts them per expert in its own
// histogram and notes each pair's place there; a scan over (expert, CTA, warp) turns the counts into
// first rows, which are added to the places.  The CTAs read one another's totals through distributed
// shared memory, so that no workspace is needed and two plans at once share nothing.
__global__ void __launch_bounds__(kPlanThreads)
    sort_plan_kernel(const int32_t* __restrict__ idx, int pairs, int experts, int32_t* __restrict__ offsets, int32_t* __restrict__ at) {
    extern __shared__ int hist[];  // [warp][expert], then this CTA's totals [expert]
    __shared__ int scan[kPlanWarps];
    int* totals = hist + kPlanWarps * experts;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = static_cast<int>(cluster_ctarank()), ctas = static_cast<int>(gridDim.x);
    for (int i = threadIdx.x; i < kPlanWarps * experts; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    const int groups = (pairs + 31) / 32, runs = ctas * kPlanWarps, run = rank * kPlanWarps + warp;
    const int each = groups / runs, more = groups % runs;  // the first `more` runs take one group of 32 pairs more
    const int p0 = (run * each + min(run, more)) * 32, p1 = min(pairs, p0 + (each + (run < more)) * 32);
    int* mine = hist + warp * experts;
    const int bits = 32 - __clz(experts);
    const unsigned none = static_cast<unsigned>(experts);  // a dropped pair's expert
    // Counts the run and leaves in `at` each pair's place among its expert's pairs of this run.
    unsigned next = p0 + lane < p1 ? static_cast<unsigned>(idx[p0 + lane]) : none;
    for (int p = p0 + lane; p - lane < p1; p += 32) {
        const unsigned x = min(next, none);
        next = p + 32 < p1 ? static_cast<unsigned>(idx[p + 32]) : none;
        const unsigned same = same_lanes(x, bits);
        const unsigned below = same & ((1u << lane) - 1u);
        int place = -1;
        if (x != none) place = mine[x] + __popc(below);
        __syncwarp();
        if (x != none && below == 0) mine[x] = place + __popc(same);
        __syncwarp();
        if (p < p1) at[p] = place;
    }
    __syncthreads();
    // Thread e: its expert's total here and in the other CTAs, the exclusive scan over experts, and
    // then the first row of each of this CTA's warps.
    const int e = threadIdx.x;
    int here = 0;
    if (e < experts) {
        for (int w = 0; w < kPlanWarps; ++w) here += hist[w * experts + e];
        totals[e] = here;
    }
    int before = 0, total = here;
    if (ctas > 1) {
        __syncwarp();  // the barrier's instructions are a converged warp's; experts may end inside one
        cluster_sync();
        if (e < experts) {
            total = 0;
            for (int c = 0; c < ctas; ++c) {
                const int t = ld_cluster(&totals[e], static_cast<uint32_t>(c));
                if (c < rank) before += t;
                total += t;
            }
        }
        __syncwarp();
        cluster_sync();  // a CTA may not end while another reads its totals
    }
    int incl = total;
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int v = scan[lane];
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += o;
        }
        scan[lane] = v;
    }
    __syncthreads();
    int first = incl - total + (warp > 0 ? scan[warp - 1] : 0);
    if (e < experts) {
        if (rank == 0) {
            offsets[e] = first;
            if (e == experts - 1) offsets[experts] = first + total;
        }
        first += before;
        for (int w = 0; w < kPlanWarps; ++w) {
            const int c = hist[w * experts + e];
            hist[w * experts + e] = first;
            first += c;
        }
    }
    __syncthreads();
#pragma unroll 4
    for (int p = p0 + lane; p < p1; p += 32) {
        const unsigned x = static_cast<unsigned>(idx[p]);
        if (x < none) at[p] += mine[x];
    }
}

// A warp takes 32 x kUnits units of a token's row: it reads them once, all loads in flight, and
// writes them to each of the pairs' rows.
template <class U>
__global__ void __launch_bounds__(kRowThreads)
    sort_rows_kernel(const uint8_t* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ at, int64_t tokens, int k, int64_t units, int parts,
                     uint8_t* __restrict__ rows, int64_t rows_stride, int64_t n_rows) {
    constexpr int kUnits = 4;
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5), t = w / parts;
    if (t >= tokens) return;
    const int64_t u0 = (w - t * parts) * (32 * kUnits) + lane;
    const U* src = reinterpret_cast<const U*>(x + t * x_stride);
    U v[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
        if (u0 + 32 * i < units) v[i] = src[u0 + 32 * i];
    for (int j0 = 0; j0 < k; j0 += 32) {
        const int mine = j0 + lane < k ? at[t * k + j0 + lane] : -1;
        for (int j = 0; j < min(32, k - j0); ++j) {
            const int r = __shfl_sync(0xffffffffu, mine, j);
            if (r < 0 || r >= n_rows) continue;
            U* dst = reinterpret_cast<U*>(rows + r * rows_stride);
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
                if (u0 + 32 * i < units) dst[u0 + 32 * i] = v[i];
        }
    }
}

// ── back, and the gradients ──────────────────────────────────────────────
// V consecutive elements of a row: 8 for rows of whole 16-byte words, else 1.
template <int DT, int V>
struct Part {
    Raw8<DT> r;
    __device__ __forceinline__ void load(const typename Elem<DT>::T* p) { r.load(p); }
    __device__ __forceinline__ void widen(float (&v)[V]) const { r.widen(v); }
    static __device__ __forceinline__ void store(typename Elem<DT>::T* p, const float (&v)[V]) { store8<DT>(p, v); }
};
template <int DT>
struct Part<DT, 1> {
    typename Elem<DT>::T e;
    __device__ __forceinline__ void load(const typename Elem<DT>::T* p) { e = *p; }
    __device__ __forceinline__ void widen(float (&v)[1]) const { v[0] = Elem<DT>::widen(e); }
    static __device__ __forceinline__ void store(typename Elem<DT>::T* p, const float (&v)[1]) { *p = Elem<DT>::narrow(v[0]); }
};

constexpr int kSlots = 4;  // rows whose loads are in flight together
// and stretches of 32 V columns of each.  The way back holds two of 16-bit values in 80 registers; its
// gradient spills 68 to 88 bytes for them and is faster all the same for many tokens (8192 tokens, top 6,
// 2048 bf16 columns: 81 us, one stretch without spills 92; 128 tokens: 5.3 and 3.9).
template <int DT, int V>
constexpr int kStretches = V == 1 ? 4 : DT == LM_DTYPE_F32 ? 1 : 2;

// The next up to kSlots slots of a token that have a row: bits of `left`, in order.  A lane holds
// the row and weight of slot j0 + lane.
struct NextSlots {
    int row[kSlots], slot[kSlots];
    float weight[kSlots];
    __device__ __forceinline__ void take(unsigned& left, int my_row, float my_weight) {
#pragma unroll
        for (int q = 0; q < kSlots; ++q) {
            slot[q] = left != 0 ? __ffs(left) - 1 : -1;
            left &= left - 1;
            row[q] = __shfl_sync(0xffffffffu, my_row, slot[q] & 31);
            weight[q] = __shfl_sync(0xffffffffu, my_weight, slot[q] & 31);
        }
    }
};

// A warp takes kStretches x 32 V columns of a token: y = the sum over its slots in order, in f32,
// rounded once.
template <int DT, int DY, int V>
__global__ void __launch_bounds__(kRowThreads, 3)
    unsort_rows_kernel(const typename Elem<DT>::T* __restrict__ rows, int64_t n_rows, const int32_t* __restrict__ at,
                       const float* __restrict__ weights, int64_t tokens, int k, int64_t cols, int parts, typename Elem<DY>::T* __restrict__ y,
                       int accumulate) {
    constexpr int U = kStretches<DT, V>;
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5), t = w / parts;
    if (t >= tokens) return;
    const int64_t c = ((w - t * parts) * (32 * U) + lane) * V;
    float s[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) s[u][i] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += 32) {
        int my_row = j0 + lane < k ? at[t * k + j0 + lane] : -1;
        if (my_row >= n_rows) my_row = -1;
        const float my_weight = weights != nullptr && j0 + lane < k ? weights[t * k + j0 + lane] : 1.0f;
        for (unsigned left = __ballot_sync(0xffffffffu, my_row >= 0); left != 0;) {
            NextSlots next;
            next.take(left, my_row, my_weight);
            Part<DT, V> v[kSlots][U];
#pragma unroll
            for (int q = 0; q < kSlots; ++q)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (next.slot[q] >= 0 && c + u * 32 * V < cols) v[q][u].load(rows + next.row[q] * cols + c + u * 32 * V);
#pragma unroll
            for (int q = 0; q < kSlots; ++q) {
                if (next.slot[q] < 0) break;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float f[V];
                    v[q][u].widen(f);
#pragma unroll
                    for (int i = 0; i < V; ++i) s[u][i] = fmaf(next.weight[q], f[i], s[u][i]);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (c + u * 32 * V >= cols) break;
        typename Elem<DY>::T* dst = y + t * cols + c + u * 32 * V;
        if (accumulate) {
            Part<DY, V> old;
            float f[V];
            old.load(dst);
            old.widen(f);
#pragma unroll
            for (int i = 0; i < V; ++i) s[u][i] += f[i];
        }
        Part<DY, V>::store(dst, s[u]);
    }
}

// grad_rows[at] = w grad_y, grad_weights = <grad_y, rows[at]> (0 for a dropped pair).  W warps of a
// CTA take a token, its columns in turns, and add their dot products in order at the end.  grad_y has
// the rows' type or, as the output it belongs to, f32.
template <int DT, int DG, int V, int W>
__global__ void __launch_bounds__(kRowThreads, 3)
    unsort_rows_backward_kernel(const typename Elem<DG>::T* __restrict__ grad_y, const typename Elem<DT>::T* rows, int64_t n_rows,
                                const int32_t* __restrict__ at, const float* __restrict__ weights, int64_t tokens, int k, int64_t cols,
                                typename Elem<DT>::T* grad_rows, float* __restrict__ grad_weights) {
    constexpr int U = kStretches<DG, V>;
    __shared__ float red[kRowWarps][LM_SORT_MAX_TOP_K];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kRowWarps / W) + warp / W;
    if (t < tokens) {
        for (int j0 = 0; j0 < k; j0 += 32) {
            int my_row = j0 + lane < k ? at[t * k + j0 + lane] : -1;
            if (my_row >= n_rows) my_row = -1;
            const float my_weight = j0 + lane < k ? weights[t * k + j0 + lane] : 0.0f;
            red[warp][j0 + lane] = 0.0f;
            __syncwarp();
            for (unsigned left = __ballot_sync(0xffffffffu, my_row >= 0); left != 0;) {
                NextSlots next;
                next.take(left, my_row, my_weight);
                float dot[kSlots];
#pragma unroll
                for (int q = 0; q < kSlots; ++q) dot[q] = 0.0f;
                for (int64_t c = (warp % W * 32 * U + lane) * V; c < cols; c += W * 32 * U * V) {
                    Part<DG, V> g[U];
                    Part<DT, V> v[kSlots][U];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + u * 32 * V < cols) g[u].load(grad_y + t * cols + c + u * 32 * V);
#pragma unroll
                    for (int q = 0; q < kSlots; ++q)
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (next.slot[q] >= 0 && c + u * 32 * V < cols) v[q][u].load(rows + next.row[q] * cols + c + u * 32 * V);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (c + u * 32 * V >= cols) break;
                        float gf[V];
                        g[u].widen(gf);
#pragma unroll
                        for (int q = 0; q < kSlots; ++q) {
                            if (next.slot[q] < 0) break;
                            float f[V], out[V];
                            v[q][u].widen(f);
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                dot[q] = fmaf(gf[i], f[i], dot[q]);
                                out[i] = next.weight[q] * gf[i];
                            }
                            Part<DT, V>::store(grad_rows + next.row[q] * cols + c + u * 32 * V, out);
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < kSlots; ++q) {
                    if (next.slot[q] < 0) break;
                    for (int off = 16; off > 0; off >>= 1) dot[q] += __shfl_xor_sync(0xffffffffu, dot[q], off);
                    if (lane == 0) red[warp][j0 + next.slot[q]] = dot[q];
                }
            }
        }
    }
    __syncthreads();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (kRowWarps / W);
    for (int i = threadIdx.x; i < kRowWarps / W * k; i += kRowThreads) {
        const int token = i / k, j = i - token * k;
        if (t0 + token >= tokens) break;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += red[token * W + w][j];
        grad_weights[(t0 + token) * k + j] = s;
    }
}

// A launch of one warp for each (token, part of its row).
template <class F>
lm_status with_parts(int64_t tokens, int64_t parts, F&& f) {
    const int64_t blocks = (tokens * parts + kRowWarps - 1) / kRowWarps;
    if (parts > INT32_MAX || blocks > INT32_MAX) return context_free_fail(LM_ERR_UNSUPPORTED, "rows of more than 2^44 bytes in all");
    f(static_cast<unsigned>(blocks), static_cast<int>(parts));
    return context_free_finish(cudaGetLastError());
}

// Rows that an int32 `at` can name.
int64_t touched(int64_t n_rows) { return std::min<int64_t>(n_rows, INT32_MAX); }
bool sizes_ok(int64_t tokens, int32_t k) {
    return tokens >= 0 && k > 0 && k <= LM_SORT_MAX_TOP_K && tokens <= (INT32_MAX - 1024) / k;  // 32-bit pair numbers, with room to step past the last
}

// The rows' gradient and the weights'; `who` names the entry in messages.
lm_status unsort_backward(const char* who, const void* grad_y, int32_t grad_y_dtype, const void* rows, int32_t dtype, int64_t n_rows, const int32_t* at,
                          const float* weights, int64_t tokens, int32_t top_k, int64_t cols, void* grad_rows, float* grad_weights, void* stream) {
    const auto refuse = [&](const char* why) {
        char message[192];
        std::snprintf(message, sizeof message, "%s: %s", who, why);
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, message);
    };
    if (!is_float_type(dtype)) return refuse("tensors are f32, bf16 or f16");
    if (!sizes_ok(tokens, top_k) || n_rows < 0 || cols < 0 || cols > LM_MX_MAX_COLS)
        return refuse("a size out of range");
    if (tokens == 0) return LM_OK;
    if (at == nullptr || weights == nullptr || grad_weights == nullptr || (cols > 0 && grad_y == nullptr) || (cols > 0 && n_rows > 0 && (rows == nullptr || grad_rows == nullptr)) ||
        !aligned(grad_y, elem_size(grad_y_dtype)) || !aligned(rows, elem_size(dtype)) || !aligned(grad_rows, elem_size(dtype)) || !aligned(at, 4) || !aligned(weights, 4) ||
        !aligned(grad_weights, 4))
        return refuse("a null or misaligned pointer");
    const int64_t row_bytes = cols * elem_size(dtype), rows_bytes = touched(n_rows) * row_bytes, grad_y_bytes = tokens * cols * elem_size(grad_y_dtype);
    if (overlap({grad_y, grad_y_bytes}, {grad_rows, rows_bytes}) || (grad_rows != rows && overlap({rows, rows_bytes}, {grad_rows, rows_bytes})))
        return refuse("grad_rows overlaps grad_y or part of rows");
    const Span to(grad_rows, rows_bytes), dots(grad_weights, tokens * top_k * 4), plan(at, tokens * top_k * 4), scale(weights, tokens * top_k * 4);
    if (overlap(to, plan) || overlap(to, scale) || overlap(to, dots) || overlap(dots, plan) || overlap(dots, scale) || overlap(dots, {rows, rows_bytes}) ||
        overlap(dots, {grad_y, grad_y_bytes}))
        return refuse("grad_rows and grad_weights overlap, or overlap at, weights, rows or grad_y");
    const bool vec = cols % 8 == 0 && aligned(grad_y, 16) && aligned(rows, 16) && aligned(grad_rows, 16);
    with_dtype(dtype, [&](auto dt) {
        with_bool(vec, [&](auto v) {
            constexpr int DT = decltype(dt)::value, V = decltype(v)::value ? 8 : 1;
            using T = typename Elem<DT>::T;
            const auto go = [&](auto dg, auto warps) {
                constexpr int DG = decltype(dg)::value, W = decltype(warps)::value, per = kRowWarps / W;
                unsort_rows_backward_kernel<DT, DG, V, W><<<static_cast<unsigned>((tokens + per - 1) / per), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    static_cast<const typename Elem<DG>::T*>(grad_y), static_cast<const T*>(rows), n_rows, at, weights, tokens, top_k, cols, static_cast<T*>(grad_rows),
                    grad_weights);
            };
            // As many warps a token as its row has stretches for them (2048 bf16 columns, 16384 tokens:
            // one warp 89 us, two 87, four 93, eight, half of them idle, 127; 1 token: 8.3, 5.6, 4.2).
            const auto fit = [&](auto dg) {
                constexpr int64_t piece = 32 * V * kStretches<decltype(dg)::value, V>;
                const int64_t pieces = (cols + piece - 1) / piece;
                if (pieces <= 1) go(dg, std::integral_constant<int, 1>{});
                else if (pieces <= 2) go(dg, std::integral_constant<int, 2>{});
                else if (pieces <= 4) go(dg, std::integral_constant<int, 4>{});
                else go(dg, std::integral_constant<int, 8>{});
            };
            if (grad_y_dtype == LM_DTYPE_F32) fit(std::integral_constant<int, LM_DTYPE_F32>{});
            else fit(dt);
        });
    });
    return context_free_finish(cudaGetLastError());
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" {

lm_status lm_moe_sort_plan(const int32_t* topk_idx, int64_t tokens, int32_t top_k, int32_t experts, int32_t* offsets, int32_t* at,
                           void* stream) {
    if (!sizes_ok(tokens, top_k) || experts <= 0 || experts > kPlanMaxExperts)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_plan: tokens x top_k beyond 2^31, top_k beyond 64 or experts beyond 1024");
    if (offsets == nullptr || !aligned(offsets, 4) || (tokens > 0 && (topk_idx == nullptr || at == nullptr || !aligned(topk_idx, 4) || !aligned(at, 4))))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_plan: a null or misaligned pointer");
    const int64_t pairs = tokens * top_k;
    const Span idx(topk_idx, pairs * 4), places(at, pairs * 4), starts(offsets, (int64_t{experts} + 1) * 4);
    if (overlap(idx, places) || overlap(idx, starts) || overlap(places, starts))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_plan: topk_idx, offsets and at overlap");
    // A cluster's launch and its two barriers cost 1.4 us more than one CTA, which takes 0.7 us for each
    // 1000 pairs (8000 pairs: one CTA 8.5 us, two 7.2, four 5.9, eight 5.2; 98304: 67 and 12.4).
    const int ctas = pairs <= 2048 ? 1 : kPlanCluster;
    const int smem = (kPlanWarps + 1) * experts * 4;
    if (smem > 40 * 1024)
        if (const cudaError_t e = cudaFuncSetAttribute(sort_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kPlanWarps + 1) * kPlanMaxExperts * 4);
            e != cudaSuccess)
            return context_free_finish(e);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = static_cast<unsigned>(ctas);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    return context_free_finish(cudaLaunchKernelEx(&cfg, sort_plan_kernel, topk_idx, static_cast<int>(pairs), static_cast<int>(experts), offsets, at));
}

lm_status lm_moe_sort_rows(const void* x, int64_t x_stride, const int32_t* at, int64_t tokens, int32_t top_k, int64_t row_bytes, void* rows,
                           int64_t rows_stride, int64_t n_rows, void* stream) {
    if (!sizes_ok(tokens, top_k) || row_bytes < 0 || row_bytes > (int64_t(1) << 31) || n_rows < 0 || x_stride < row_bytes || rows_stride < row_bytes)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_rows: a size or stride out of range");
    if (tokens == 0 || row_bytes == 0 || n_rows == 0) return LM_OK;
    if (x == nullptr || at == nullptr || rows == nullptr || !aligned(at, 4))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_rows: a null or misaligned pointer");
    const Span to(rows, touched(n_rows), rows_stride, row_bytes);
    if (overlap(to, {x, tokens, x_stride, row_bytes}) || overlap(to, {at, tokens * top_k * 4}))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_rows: rows overlaps x or at");
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) | static_cast<uintptr_t>(x_stride) |
                          static_cast<uintptr_t>(rows_stride) | static_cast<uintptr_t>(row_bytes);
    const auto go = [&](auto unit) {
        using U = decltype(unit);
        const int64_t units = row_bytes / static_cast<int64_t>(sizeof(U));
        return with_parts(tokens, (units + 127) / 128, [&](unsigned grid, int parts) {
            sort_rows_kernel<U><<<grid, kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint8_t*>(x), x_stride, at, tokens, top_k, units, parts,
                                                                                             static_cast<uint8_t*>(rows), rows_stride, n_rows);
        });
    };
    if (all % 16 == 0) return go(uint4{});
    if (all % 4 == 0) return go(uint32_t{});
    if (all % 2 == 0) return go(uint16_t{});
    return go(uint8_t{});
}

lm_status lm_moe_unsort_rows(const void* rows, int32_t dtype, int64_t n_rows, const int32_t* at, const float* weights, int64_t tokens, int32_t top_k,
                             int64_t cols, void* y, int32_t y_dtype, int32_t accumulate, void* stream) {
    if (!is_float_type(dtype) || (y_dtype != dtype && y_dtype != LM_DTYPE_F32))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows: rows are f32, bf16 or f16, y the same or f32");
    if (!sizes_ok(tokens, top_k) || n_rows < 0 || cols < 0 || cols > LM_MX_MAX_COLS)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows: a size out of range");
    if (tokens == 0 || cols == 0) return LM_OK;
    if ((rows == nullptr && n_rows > 0) || at == nullptr || y == nullptr || !aligned(rows, elem_size(dtype)) || !aligned(y, elem_size(y_dtype)) || !aligned(at, 4) ||
        !aligned(weights, 4))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows: a null or misaligned pointer");
    const Span to(y, tokens * cols * elem_size(y_dtype));
    if (overlap(to, {rows, touched(n_rows) * cols * elem_size(dtype)}) || overlap(to, {at, tokens * top_k * 4}) || overlap(to, {weights, tokens * top_k * 4}))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows: y overlaps rows, at or weights");
    const bool vec = cols % 8 == 0 && aligned(rows, 16) && aligned(y, 16);
    lm_status st = LM_OK;
    with_dtype(dtype, [&](auto dt) {
        with_bool(vec, [&](auto v) {
            constexpr int DT = decltype(dt)::value, V = decltype(v)::value ? 8 : 1;
            constexpr int64_t each = 32 * V * kStretches<DT, V>;
            const auto go = [&](auto dy) {
                constexpr int DY = decltype(dy)::value;
                st = with_parts(tokens, (cols + each - 1) / each, [&](unsigned grid, int parts) {
                    unsort_rows_kernel<DT, DY, V><<<grid, kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                        static_cast<const typename Elem<DT>::T*>(rows), n_rows, at, weights, tokens, top_k, cols, parts, static_cast<typename Elem<DY>::T*>(y),
                        accumulate != 0);
                });
            };
            if (y_dtype == LM_DTYPE_F32) go(std::integral_constant<int, LM_DTYPE_F32>{});
            else go(dt);
        });
    });
    return st;
}

lm_status lm_moe_unsort_rows_backward(const void* grad_y, const void* rows, int32_t dtype, int64_t n_rows, const int32_t* at, const float* weights,
                                      int64_t tokens, int32_t top_k, int64_t cols, void* grad_rows, float* grad_weights, void* stream) {
    return unsort_backward("lm_moe_unsort_rows_backward", grad_y, dtype, rows, dtype, n_rows, at, weights, tokens, top_k, cols, grad_rows, grad_weights, stream);
}

lm_status lm_moe_unsort_rows_backward_f32(const float* grad_y, const void* rows, int32_t dtype, int64_t n_rows, const int32_t* at, const float* weights,
                                          int64_t tokens, int32_t top_k, int64_t cols, void* grad_rows, float* grad_weights, void* stream) {
    return unsort_backward("lm_moe_unsort_rows_backward_f32", grad_y, LM_DTYPE_F32, rows, dtype, n_rows, at, weights, tokens, top_k, cols, grad_rows, grad_weights, stream);
}

}  // extern "C"
