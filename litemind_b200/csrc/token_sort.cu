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

#include <algorithm>

namespace lm {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanMaxExperts = 1024;

// One CTA.  Each warp takes a contiguous run of pairs and counts them per expert in its own
// histogram; a scan over (expert, warp) turns the counts into first rows; a second pass over the
// run hands the rows out in order.
__global__ void __launch_bounds__(kPlanThreads)
    sort_plan_kernel(const int32_t* __restrict__ idx, int64_t pairs, int experts, int32_t* __restrict__ offsets,
                     int32_t* __restrict__ at) {
    extern __shared__ int hist[];  // [warp][expert]
    __shared__ int scan[kPlanWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < kPlanWarps * experts; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    const int64_t groups = (pairs + 31) / 32;
    const int64_t g0 = groups * warp / kPlanWarps, g1 = groups * (warp + 1) / kPlanWarps;
    int* mine = hist + warp * experts;
    for (int64_t g = g0; g < g1; ++g) {
        const int64_t p = g * 32 + lane;
        const int e = p < pairs ? idx[p] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && e < experts && __ffs(same) - 1 == lane) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // Thread e: its expert's total, then the exclusive scan over experts, then each warp's first row.
    int total = 0;
    const int e = threadIdx.x;
    if (e < experts)
        for (int w = 0; w < kPlanWarps; ++w) total += hist[w * experts + e];
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
        offsets[e] = first;
        if (e == experts - 1) offsets[experts] = first + total;
        for (int w = 0; w < kPlanWarps; ++w) {
            const int c = hist[w * experts + e];
            hist[w * experts + e] = first;
            first += c;
        }
    }
    __syncthreads();
    for (int64_t g = g0; g < g1; ++g) {
        const int64_t p = g * 32 + lane;
        const int x = p < pairs ? idx[p] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, x);
        const bool live = x >= 0 && x < experts;
        const int row = live ? mine[x] + __popc(same & ((1u << lane) - 1u)) : -1;
        __syncwarp();
        if (live && __ffs(same) - 1 == lane) mine[x] += __popc(same);
        __syncwarp();
        if (p < pairs) at[p] = row;
    }
}

// A CTA a token: its row is read once and written to each of its pairs' rows.
template <class U>
__global__ void __launch_bounds__(256)
    sort_rows_kernel(const uint8_t* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ at, int k, int64_t units,
                     uint8_t* __restrict__ rows, int64_t rows_stride, int64_t n_rows) {
    const int64_t t = blockIdx.x;
    for (int64_t u = threadIdx.x; u < units; u += 256) {
        const U v = reinterpret_cast<const U*>(x + t * x_stride)[u];
        for (int j = 0; j < k; ++j) {
            const int r = at[t * k + j];
            if (r >= 0 && r < n_rows) reinterpret_cast<U*>(rows + r * rows_stride)[u] = v;
        }
    }
}

// A CTA a token: y = sum over slots in order, in f32, rounded once.
template <int DT, int DY>
__global__ void __launch_bounds__(256)
    unsort_rows_kernel(const typename Elem<DT>::T* __restrict__ rows, int64_t n_rows, const int32_t* __restrict__ at,
                       const float* __restrict__ weights, int k, int64_t cols, typename Elem<DY>::T* __restrict__ y, bool accumulate) {
    const int64_t t = blockIdx.x;
    for (int64_t c = threadIdx.x; c < cols; c += 256) {
        float s = 0.0f;
        for (int j = 0; j < k; ++j) {
            const int r = at[t * k + j];
            if (r >= 0 && r < n_rows) {
                const float v = Elem<DT>::widen(rows[r * cols + c]);
                s = weights != nullptr ? fmaf(weights[t * k + j], v, s) : s + v;
            }
        }
        if (accumulate) s += Elem<DY>::widen(y[t * cols + c]);
        y[t * cols + c] = Elem<DY>::narrow(s);
    }
}

// A CTA a token: grad_rows[at] = w grad_y, grad_weights = <grad_y, rows[at]> (0 for a dropped pair).
template <int DT>
__global__ void __launch_bounds__(256)
    unsort_rows_backward_kernel(const typename Elem<DT>::T* __restrict__ grad_y, const typename Elem<DT>::T* rows,
                                int64_t n_rows, const int32_t* __restrict__ at, const float* __restrict__ weights, int k, int64_t cols,
                                typename Elem<DT>::T* grad_rows, float* __restrict__ grad_weights) {
    __shared__ float red[8];
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int j = 0; j < k; ++j) {
        const int r = at[t * k + j];
        const bool live = r >= 0 && r < n_rows;
        const float w = weights[t * k + j];
        float s = 0.0f;
        if (live) {
            for (int64_t c = threadIdx.x; c < cols; c += 256) {
                const float g = Elem<DT>::widen(grad_y[t * cols + c]);
                s = fmaf(g, Elem<DT>::widen(rows[r * cols + c]), s);
                grad_rows[r * cols + c] = Elem<DT>::narrow(w * g);
            }
        }
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            float a = 0.0f;
            for (int i = 0; i < 8; ++i) a += red[i];
            grad_weights[t * k + j] = a;
        }
        __syncthreads();
    }
}

bool sizes_ok(int64_t tokens, int32_t k) {
    return tokens >= 0 && k > 0 && k <= LM_SORT_MAX_TOP_K && tokens <= INT32_MAX / k;
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
    const int smem = kPlanWarps * experts * 4;
    if (smem > 48 * 1024)
        if (const cudaError_t e = cudaFuncSetAttribute(sort_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanWarps * kPlanMaxExperts * 4);
            e != cudaSuccess)
            return context_free_finish(e);
    sort_plan_kernel<<<1, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(topk_idx, tokens * top_k, experts, offsets, at);
    return context_free_finish(cudaGetLastError());
}

lm_status lm_moe_sort_rows(const void* x, int64_t x_stride, const int32_t* at, int64_t tokens, int32_t top_k, int64_t row_bytes, void* rows,
                           int64_t rows_stride, int64_t n_rows, void* stream) {
    if (!sizes_ok(tokens, top_k) || row_bytes < 0 || row_bytes > (int64_t(1) << 31) || n_rows < 0 || x_stride < row_bytes || rows_stride < row_bytes)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_rows: a size or stride out of range");
    if (tokens == 0 || row_bytes == 0 || n_rows == 0) return LM_OK;
    if (x == nullptr || at == nullptr || rows == nullptr || !aligned(at, 4))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_sort_rows: a null or misaligned pointer");
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) | static_cast<uintptr_t>(x_stride) |
                          static_cast<uintptr_t>(rows_stride) | static_cast<uintptr_t>(row_bytes);
    const auto go = [&](auto unit) {
        using U = decltype(unit);
        sort_rows_kernel<U><<<static_cast<unsigned>(tokens), 256, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const uint8_t*>(x), x_stride, at, top_k, row_bytes / static_cast<int64_t>(sizeof(U)), static_cast<uint8_t*>(rows), rows_stride,
            n_rows);
    };
    if (all % 16 == 0) go(uint4{});
    else if (all % 4 == 0) go(uint32_t{});
    else if (all % 2 == 0) go(uint16_t{});
    else go(uint8_t{});
    return context_free_finish(cudaGetLastError());
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
    with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const auto go = [&](auto dy) {
            constexpr int DY = decltype(dy)::value;
            unsort_rows_kernel<DT, DY><<<static_cast<unsigned>(tokens), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                static_cast<const typename Elem<DT>::T*>(rows), n_rows, at, weights, top_k, cols, static_cast<typename Elem<DY>::T*>(y), accumulate != 0);
        };
        if (y_dtype == LM_DTYPE_F32) go(std::integral_constant<int, LM_DTYPE_F32>{});
        else go(dt);
    });
    return context_free_finish(cudaGetLastError());
}

lm_status lm_moe_unsort_rows_backward(const void* grad_y, const void* rows, int32_t dtype, int64_t n_rows, const int32_t* at, const float* weights,
                                      int64_t tokens, int32_t top_k, int64_t cols, void* grad_rows, float* grad_weights, void* stream) {
    if (!is_float_type(dtype)) return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows_backward: tensors are f32, bf16 or f16");
    if (!sizes_ok(tokens, top_k) || n_rows < 0 || cols < 0 || cols > LM_MX_MAX_COLS)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows_backward: a size out of range");
    if (tokens == 0) return LM_OK;
    if (at == nullptr || weights == nullptr || grad_weights == nullptr || (cols > 0 && grad_y == nullptr) || (cols > 0 && n_rows > 0 && (rows == nullptr || grad_rows == nullptr)) ||
        !aligned(grad_y, elem_size(dtype)) || !aligned(rows, elem_size(dtype)) || !aligned(grad_rows, elem_size(dtype)) || !aligned(at, 4) || !aligned(weights, 4) ||
        !aligned(grad_weights, 4))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_moe_unsort_rows_backward: a null or misaligned pointer");
    with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        using T = typename Elem<DT>::T;
        unsort_rows_backward_kernel<DT><<<static_cast<unsigned>(tokens), 256, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(grad_y), static_cast<const T*>(rows), n_rows, at, weights, top_k, cols, static_cast<T*>(grad_rows), grad_weights);
    });
    return context_free_finish(cudaGetLastError());
}

}  // extern "C"
