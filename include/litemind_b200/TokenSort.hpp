// TokenSort.hpp -- tokens sorted by expert and back with the routing weights, and the gradients of
// both: thin C++ forms of lm_moe_sort_* (litemind_moe.h) on device memory.  Each call returns the
// lm_status of the launch.  The reference handles one token at a time and needs none
// (src/DeepSeekRunner.cpp:273-285).
#pragma once

#include <cstddef>
#include <cstdint>

#include "litemind_moe.h"

namespace litemind::b200 {

/** Where each (token, slot) pair's row is among the rows sorted by expert; device memory of the caller. */
struct SortPlan {
    int32_t* offsets{nullptr};  ///< experts + 1
    int32_t* at{nullptr};       ///< tokens x top_k, -1 for a dropped pair
    std::size_t tokens{0};
    int32_t top_k{0};
    int32_t experts{0};

    /** Fills offsets and at from the routing's indices (device, tokens x top_k). */
    lm_status build(const int32_t* topk_idx, void* stream = nullptr) const {
        return lm_moe_sort_plan(topk_idx, static_cast<int64_t>(tokens), top_k, experts, offsets, at, stream);
    }
    /** rows[at[t, j]] = x[t], rows of row_bytes bytes each. */
    lm_status sort(const void* x, std::size_t row_bytes, void* rows, std::size_t n_rows, void* stream = nullptr) const {
        return sort(x, row_bytes, row_bytes, rows, row_bytes, n_rows, stream);
    }
    /** The same with rows of x and of the result x_stride and rows_stride bytes apart. */
    lm_status sort(const void* x, std::size_t x_stride, std::size_t row_bytes, void* rows, std::size_t rows_stride, std::size_t n_rows,
                   void* stream = nullptr) const {
        return lm_moe_sort_rows(x, static_cast<int64_t>(x_stride), at, static_cast<int64_t>(tokens), top_k,
                                static_cast<int64_t>(row_bytes), rows, static_cast<int64_t>(rows_stride), static_cast<int64_t>(n_rows),
                                stream);
    }
    /** y[t] (+)= the sum over j of weights[t, j] * rows[at[t, j]]; without weights the gradient of sort. */
    lm_status unsort(const void* rows, int32_t dtype, std::size_t n_rows, const float* weights, std::size_t cols, void* y,
                     int32_t y_dtype, bool accumulate = false, void* stream = nullptr) const {
        return lm_moe_unsort_rows(rows, dtype, static_cast<int64_t>(n_rows), at, weights, static_cast<int64_t>(tokens), top_k,
                                  static_cast<int64_t>(cols), y, y_dtype, accumulate ? 1 : 0, stream);
    }
    /** The gradient of unsort with weights. */
    lm_status unsort_backward(const void* grad_y, const void* rows, int32_t dtype, std::size_t n_rows, const float* weights,
                              std::size_t cols, void* grad_rows, float* grad_weights, void* stream = nullptr) const {
        return lm_moe_unsort_rows_backward(grad_y, rows, dtype, static_cast<int64_t>(n_rows), at, weights,
                                           static_cast<int64_t>(tokens), top_k, static_cast<int64_t>(cols), grad_rows, grad_weights,
                                           stream);
    }
    /** The same with grad_y in f32 whatever the type of the rows: the gradient of unsort with an f32 y. */
    lm_status unsort_backward_f32(const float* grad_y, const void* rows, int32_t dtype, std::size_t n_rows, const float* weights,
                                  std::size_t cols, void* grad_rows, float* grad_weights, void* stream = nullptr) const {
        return lm_moe_unsort_rows_backward_f32(grad_y, rows, dtype, static_cast<int64_t>(n_rows), at, weights,
                                               static_cast<int64_t>(tokens), top_k, static_cast<int64_t>(cols), grad_rows,
                                               grad_weights, stream);
    }
};

}  // namespace litemind::b200
