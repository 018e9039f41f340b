// mx_ops.cu -- microscaled (MX) rows made and read back, and the residual's addition and RMS
// norm that end in them (lm_mx_quantize, lm_mx_dequantize, lm_gemm_add_rms_norm_mx).
//
// All three move each value once and compute a few operations on it: HBM bounds them for large
// inputs and the launch for small ones.
#include "moe_internal.h"
#include "mx_block.cuh"

#include <algorithm>

namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int kSegCols = 256;  // columns a warp takes at a time: 8 a lane, 8 blocks of 32

// A warp takes one segment of a row: 256 columns, 8 scale bytes.  `segs` covers the padded
// scales, so the last segments of a row may hold scale padding only.
template <int DT, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const typename Elem<DT>::T* __restrict__ values, int64_t rows, int64_t cols, int64_t row_stride,
                       int segs, uint8_t* __restrict__ data, int64_t data_pitch, uint8_t* __restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const int64_t total = rows * segs;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); w < total; w += step) {
        const int64_t row = w / segs;
        const int seg = static_cast<int>(w - row * segs);
        const int64_t col = static_cast<int64_t>(seg) * kSegCols + lane * 8;
        const typename Elem<DT>::T* p = values + row * row_stride + col;
        float v[8];
        if (VEC && col + 8 <= cols) {
            load8<DT>(p, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? Elem<DT>::widen(p[i]) : 0.0f;
        }
        const uint32_t byte = mx_scale_byte<FMT>(v);
        const uint2 codes = mx_encode8<FMT>(v, byte);
        constexpr int kBytes = FMT == LM_MX_E2M1 ? 4 : 8;
        const int64_t at = static_cast<int64_t>(seg) * (32 * kBytes) + lane * kBytes;
        if (at < data_pitch) {
            if constexpr (FMT == LM_MX_E2M1) *reinterpret_cast<uint32_t*>(data + row * data_pitch + at) = codes.x;
            else *reinterpret_cast<uint2*>(data + row * data_pitch + at) = codes;
        }
        const uint32_t word = mx_gather_scales(byte, lane);
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + w * 8 + (lane >> 4) * 4) = word;
    }
}

template <int DT, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t* __restrict__ data, int64_t data_pitch, const uint8_t* __restrict__ scales,
                         int64_t scale_pitch, int64_t rows, int64_t cols, int segs, typename Elem<DT>::T* __restrict__ values,
                         int64_t row_stride) {
    const int lane = threadIdx.x & 31;
    const int64_t total = rows * segs;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); w < total; w += step) {
        const int64_t row = w / segs;
        const int seg = static_cast<int>(w - row * segs);
        const int64_t col = static_cast<int64_t>(seg) * kSegCols + lane * 8;
        if (col >= cols) continue;
        constexpr int kBytes = FMT == LM_MX_E2M1 ? 4 : 8;
        const uint8_t* src = data + row * data_pitch + col * kBytes / 8;
        uint2 codes = make_uint2(0u, 0u);
        if constexpr (FMT == LM_MX_E2M1) codes.x = *reinterpret_cast<const uint32_t*>(src);
        else codes = *reinterpret_cast<const uint2*>(src);
        float v[8];
        mx_decode8<FMT>(codes, scales[row * scale_pitch + col / kMxBlock], v);
        typename Elem<DT>::T* p = values + row * row_stride + col;
        if (VEC && col + 8 <= cols) {
            store8<DT>(p, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < cols) p[i] = Elem<DT>::narrow(v[i]);
        }
    }
}

// One CTA a row.  Thread t holds columns 8 t .. 8 t + 7 of each stretch of 8 * kThreads columns.
// The sum is stored in the residual's type and normalised as stored; its squares are summed in
// f64, as lm_gemm_rms_norm does.
template <int DT, int DD, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    add_rms_norm_mx_kernel(const typename Elem<DT>::T* hidden, const typename Elem<DD>::T* delta,
                           const float* __restrict__ weight, int64_t cols, float eps, typename Elem<DT>::T* sum,
                           __nv_bfloat16* __restrict__ out_bf16, uint8_t* __restrict__ data, int64_t data_pitch,
                           uint8_t* __restrict__ scales, int64_t scale_pitch) {
    __shared__ double red[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * cols;
    double s = 0.0;
    for (int64_t col = threadIdx.x * 8; col < cols; col += kThreads * 8) {
        for (int i = 0; i < 8; ++i) {
            if (col + i < cols) {
                float v = Elem<DT>::widen(hidden[base + col + i]);
                if (delta != nullptr) v += Elem<DD>::widen(delta[base + col + i]);
                const typename Elem<DT>::T stored = Elem<DT>::narrow(v);
                sum[base + col + i] = stored;
                const double d = Elem<DT>::widen(stored);
                s = fma(d, d, s);
            }
        }
    }
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) s += red[i];
    const float inverse = static_cast<float>(1.0 / sqrt(s / static_cast<double>(cols) + static_cast<double>(eps)));
    for (int64_t col = threadIdx.x * 8; col < scale_pitch * kMxBlock; col += kThreads * 8) {
        float v[8];
        for (int i = 0; i < 8; ++i) {
            v[i] = 0.0f;
            if (col + i < cols) {
                v[i] = Elem<DT>::widen(sum[base + col + i]) * inverse * weight[col + i];
                if (out_bf16 != nullptr) out_bf16[base + col + i] = __float2bfloat16_rn(v[i]);
            }
        }
        const uint32_t byte = mx_scale_byte<FMT>(v);
        const uint2 codes = mx_encode8<FMT>(v, byte);
        constexpr int kBytes = FMT == LM_MX_E2M1 ? 4 : 8;
        const int64_t at = col / 8 * kBytes;
        uint8_t* dst = data + static_cast<int64_t>(blockIdx.x) * data_pitch + at;
        if (at < data_pitch) {
            if constexpr (FMT == LM_MX_E2M1) *reinterpret_cast<uint32_t*>(dst) = codes.x;
            else *reinterpret_cast<uint2*>(dst) = codes;
        }
        if ((lane & 3) == 0) scales[static_cast<int64_t>(blockIdx.x) * scale_pitch + col / kMxBlock] = static_cast<uint8_t>(byte);
    }
}

bool is_mx_format(int32_t format) { return format == LM_MX_E2M1 || format == LM_MX_E4M3; }

unsigned grid_for(int64_t segments) {
    const int64_t warps = kThreads / 32;
    return static_cast<unsigned>(std::min<int64_t>((segments + warps - 1) / warps, 148 * 8 * 4));
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" {

int64_t lm_mx_data_pitch(int32_t format, int64_t cols) {
    return is_mx_format(format) && cols >= 0 && cols <= LM_MX_MAX_COLS ? mx_data_pitch(format, cols) : 0;
}
int64_t lm_mx_scale_pitch(int64_t cols) { return cols >= 0 && cols <= LM_MX_MAX_COLS ? mx_scale_pitch(cols) : 0; }

lm_status lm_mx_quantize(const void* values, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride, int32_t format,
                         uint8_t* data, uint8_t* scales, void* stream) {
    if (!is_float_type(dtype) || !is_mx_format(format))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_quantize: values are f32, bf16 or f16, the format is E2M1 or E4M3");
    if (rows < 0 || cols < 0 || rows > LM_MX_MAX_ROWS || cols > LM_MX_MAX_COLS || row_stride < cols)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_quantize: rows, cols or row_stride out of range");
    if (rows == 0 || cols == 0) return LM_OK;
    if (values == nullptr || data == nullptr || scales == nullptr || !aligned(values, elem_size(dtype)) || !aligned(data, 32) || !aligned(scales, 16))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_quantize: data must be 32-byte aligned and scales 16-byte aligned");
    const int segs = static_cast<int>(mx_scale_pitch(cols) / 8);
    const bool vec = aligned(values, 16) && row_stride * elem_size(dtype) % 16 == 0;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    with_dtype(dtype, [&](auto dt) {
        with_format(format, [&](auto fmt) {
            with_bool(vec, [&](auto v) {
                using T = typename Elem<decltype(dt)::value>::T;
                mx_quantize_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(v)::value>
                    <<<grid_for(rows * segs), kThreads, 0, s>>>(static_cast<const T*>(values), rows, cols, row_stride, segs, data,
                                                                mx_data_pitch(format, cols), scales);
            });
        });
    });
    return context_free_finish(cudaGetLastError());
}

lm_status lm_mx_dequantize(const uint8_t* data, const uint8_t* scales, int32_t format, int64_t rows, int64_t cols, void* values,
                           int32_t dtype, int64_t row_stride, void* stream) {
    if (!is_float_type(dtype) || !is_mx_format(format))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_dequantize: values are f32, bf16 or f16, the format is E2M1 or E4M3");
    if (rows < 0 || cols < 0 || rows > LM_MX_MAX_ROWS || cols > LM_MX_MAX_COLS || row_stride < cols)
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_dequantize: rows, cols or row_stride out of range");
    if (rows == 0 || cols == 0) return LM_OK;
    if (values == nullptr || data == nullptr || scales == nullptr || !aligned(values, elem_size(dtype)) || !aligned(data, 32) || !aligned(scales, 16))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_dequantize: data must be 32-byte aligned and scales 16-byte aligned");
    const int segs = static_cast<int>((cols + kSegCols - 1) / kSegCols);
    const bool vec = aligned(values, 16) && row_stride * elem_size(dtype) % 16 == 0;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    with_dtype(dtype, [&](auto dt) {
        with_format(format, [&](auto fmt) {
            with_bool(vec, [&](auto v) {
                using T = typename Elem<decltype(dt)::value>::T;
                mx_dequantize_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(v)::value>
                    <<<grid_for(rows * segs), kThreads, 0, s>>>(data, mx_data_pitch(format, cols), scales, mx_scale_pitch(cols), rows,
                                                                cols, segs, static_cast<T*>(values), row_stride);
            });
        });
    });
    return context_free_finish(cudaGetLastError());
}

lm_status lm_gemm_add_rms_norm_mx(const void* hidden, int32_t dtype, const void* delta, int32_t delta_dtype, const float* weight,
                                  int64_t rows, int64_t count, float epsilon, void* sum, uint16_t* out_bf16, int32_t format,
                                  uint8_t* data, uint8_t* scales, void* stream) {
    const auto residual_type = [](int32_t t) { return t == LM_DTYPE_F32 || t == LM_DTYPE_BF16; };
    if (!residual_type(dtype) || (delta != nullptr && !residual_type(delta_dtype)) || !is_mx_format(format))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_gemm_add_rms_norm_mx: hidden and delta are f32 or bf16, the format is E2M1 or E4M3");
    if (rows < 0 || count < 0 || rows > LM_MX_MAX_ROWS || count > LM_MX_MAX_COLS || !(epsilon >= 0.0f))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_gemm_add_rms_norm_mx: rows, count or epsilon out of range");
    if (rows == 0 || count == 0) return LM_OK;
    if (hidden == nullptr || weight == nullptr || sum == nullptr || data == nullptr || scales == nullptr || !aligned(hidden, elem_size(dtype)) ||
        !aligned(sum, elem_size(dtype)) || (delta != nullptr && !aligned(delta, elem_size(delta_dtype))) || !aligned(weight, 4) ||
        !aligned(out_bf16, 2) || !aligned(data, 32) || !aligned(scales, 16))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_gemm_add_rms_norm_mx: a null pointer, or data not 32-byte or scales not 16-byte aligned");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (delta == nullptr) delta_dtype = dtype;
    with_bool(dtype == LM_DTYPE_F32, [&](auto hf) {
        with_bool(delta_dtype == LM_DTYPE_F32, [&](auto df) {
            with_format(format, [&](auto fmt) {
                constexpr int DT = decltype(hf)::value ? LM_DTYPE_F32 : LM_DTYPE_BF16;
                constexpr int DD = decltype(df)::value ? LM_DTYPE_F32 : LM_DTYPE_BF16;
                add_rms_norm_mx_kernel<DT, DD, decltype(fmt)::value, false><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(
                    static_cast<const typename Elem<DT>::T*>(hidden), static_cast<const typename Elem<DD>::T*>(delta), weight, count,
                    epsilon, static_cast<typename Elem<DT>::T*>(sum), reinterpret_cast<__nv_bfloat16*>(out_bf16), data,
                    mx_data_pitch(format, count), scales, mx_scale_pitch(count));
            });
        });
    });
    return context_free_finish(cudaGetLastError());
}

}  // extern "C"
