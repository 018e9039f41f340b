// Mx.hpp -- microscaled (MX) matrices on device memory: 4-bit weights and 8- or 4-bit activations
// with a power-of-two scale for each 32 columns, and their grouped product.
//
// Thin C++ forms of lm_mx_* (litemind_moe.h, which describes the layout).  As in Gemm.hpp the
// pointers are device memory and each call returns the lm_status of the launch.  The reference has no
// counterpart: its weights are bf16 (include/Gemm.hpp:23-72).
#pragma once

#include <cstddef>
#include <cstdint>

#include "litemind_moe.h"

namespace litemind::b200::mx {

/** A matrix [rows, cols], or a stack of them row after row, in device memory that the caller owns. */
struct Matrix {
    std::uint8_t* data{nullptr};    ///< rows x data_pitch(format, cols) bytes, on a 32-byte boundary
    std::uint8_t* scales{nullptr};  ///< rows x scale_pitch(cols) bytes, on a 16-byte boundary
    std::size_t rows{0};
    std::size_t cols{0};
    int32_t format{LM_MX_E2M1};
};

/** Bytes of one row of codes / of scales. */
inline std::size_t data_pitch(int32_t format, std::size_t cols) {
    return static_cast<std::size_t>(lm_mx_data_pitch(format, static_cast<int64_t>(cols)));
}
inline std::size_t scale_pitch(std::size_t cols) { return static_cast<std::size_t>(lm_mx_scale_pitch(static_cast<int64_t>(cols))); }

/** values [rows, cols] (LM_DTYPE_F32, _BF16 or _F16, row_stride elements apart) to MX. */
inline lm_status quantize(const void* values, int32_t dtype, std::size_t row_stride, const Matrix& out, void* stream = nullptr) {
    return lm_mx_quantize(values, dtype, static_cast<int64_t>(out.rows), static_cast<int64_t>(out.cols),
                          static_cast<int64_t>(row_stride), out.format, out.data, out.scales, stream);
}

/** The values that a matrix stands for. */
inline lm_status dequantize(const Matrix& in, void* values, int32_t dtype, std::size_t row_stride, void* stream = nullptr) {
    return lm_mx_dequantize(in.data, in.scales, in.format, static_cast<int64_t>(in.rows), static_cast<int64_t>(in.cols), values,
                            dtype, static_cast<int64_t>(row_stride), stream);
}

/**
 * out[r, :] = W_g x[r, :] for the rows r of each group: w holds `groups` matrices of w.rows / groups
 * rows in LM_MX_E2M1, offsets (device, groups + 1) the groups' rows of x; null with one group.
 */
inline lm_status matmul(const Matrix& x, const Matrix& w, std::size_t groups, const int32_t* offsets, void* out, int32_t out_dtype,
                        std::size_t out_stride, void* stream = nullptr) {
    if (w.format != LM_MX_E2M1 || w.cols != x.cols || groups == 0 || groups > LM_MX_MAX_GROUPS || w.rows % groups != 0)
        return LM_ERR_INVALID_ARGUMENT;
    return lm_mx_matmul(x.data, x.scales, x.format, static_cast<int64_t>(x.rows), w.data, w.scales, static_cast<int32_t>(groups),
                        static_cast<int64_t>(w.rows / groups), static_cast<int64_t>(x.cols), offsets, out, out_dtype,
                        static_cast<int64_t>(out_stride), stream);
}

}  // namespace litemind::b200::mx
