// mx_ops.cu -- microscaled (MX) rows made and read back, and the residual's addition and RMS
// norm that end in them (lm_mx_quantize, lm_mx_dequantize, lm_gemm_add_rms_norm_mx).
//
// All three move each value once and compute a few operations on it: HBM bounds them for large
// inputs and the launch for small ones.
#include "moe_internal.h"
#include "mx_block.cuh"

#include <cstdint>

namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSegCols = 256;  // columns a warp takes at a time: 8 a lane, 8 blocks of 32
constexpr int kFlight = 4;     // segments a warp has in flight

// Segments of all rows, laid end to end; a warp takes kFlight of them, kWarps apart, at a time.
// I is the type of a segment's number: 32 bits where they fit, since a 64-bit division for each
// segment costs as much as its conversion.
template <class I>
__device__ __forceinline__ I first_segment() {
    return static_cast<I>(blockIdx.x) * (kWarps * kFlight) + (threadIdx.x >> 5);
}

// Eight values from column `col` on; zeros past the row's end.
template <int DT, bool VEC>
__device__ __forceinline__ void load_cols(const typename Elem<DT>::T* row, int64_t col, int64_t cols, float (&v)[8]) {
    if (VEC && col + 8 <= cols) {
        load8<DT>(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? Elem<DT>::widen(row[col + i]) : 0.0f;
    }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store_cols(typename Elem<DT>::T* row, int64_t col, int64_t cols, const float (&v)[8]) {
    if (VEC && col + 8 <= cols) {
        store8<DT>(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) row[col + i] = Elem<DT>::narrow(v[i]);
    }
}

// A lane's eight codes at column `col` of a row of codes; nothing past its padding.
template <int FMT>
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t col, int64_t data_pitch, uint2 codes) {
    constexpr int kBytes = FMT == LM_MX_E2M1 ? 4 : 8;
    const int64_t at = col / 8 * kBytes;
    if (at >= data_pitch) return;
    if constexpr (FMT == LM_MX_E2M1) *reinterpret_cast<uint32_t*>(row + at) = codes.x;
    else *reinterpret_cast<uint2*>(row + at) = codes;
}

// A warp takes a segment of a row: 256 columns, 8 scale bytes.  `segs` covers the padded scales,
// so the last segments of a row may hold scale padding only.
template <int DT, int FMT, bool VEC, class I>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const typename Elem<DT>::T* __restrict__ values, I total, int64_t cols, int64_t row_stride, int segs,
                       uint8_t* __restrict__ data, int64_t data_pitch, uint8_t* __restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const I w0 = first_segment<I>();
    float v[kFlight][8];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        const I w = w0 + f * kWarps, row = w / segs;
        const int64_t col = static_cast<int64_t>(w - row * segs) * kSegCols + lane * 8;
        load_cols<DT, VEC>(values + row * row_stride, col, w < total ? cols : 0, v[f]);
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        const I w = w0 + f * kWarps, row = w / segs;
        if (w >= total) break;
        const int64_t col = static_cast<int64_t>(w - row * segs) * kSegCols + lane * 8;
        const uint32_t byte = mx_scale_byte<FMT>(v[f]);
        store_codes<FMT>(data + row * data_pitch, col, data_pitch, mx_encode8<FMT>(v[f], byte));
        const uint32_t word = mx_gather_scales(byte, lane);
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + static_cast<int64_t>(w) * 8 + (lane >> 4) * 4) = word;
    }
}

template <int DT, int FMT, bool VEC, class I>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t* __restrict__ data, int64_t data_pitch, const uint8_t* __restrict__ scales, int64_t scale_pitch, I total,
                         int64_t cols, int segs, typename Elem<DT>::T* __restrict__ values, int64_t row_stride) {
    const int lane = threadIdx.x & 31;
    const I w0 = first_segment<I>();
    uint2 codes[kFlight];
    uint32_t byte[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        const I w = w0 + f * kWarps, row = w / segs;
        const int64_t col = static_cast<int64_t>(w - row * segs) * kSegCols + lane * 8;
        codes[f] = make_uint2(0u, 0u);
        byte[f] = 0;
        if (w < total && col < cols) {
            const uint8_t* src = data + row * data_pitch + col * (FMT == LM_MX_E2M1 ? 4 : 8) / 8;
            if constexpr (FMT == LM_MX_E2M1) codes[f].x = *reinterpret_cast<const uint32_t*>(src);
            else codes[f] = *reinterpret_cast<const uint2*>(src);
            byte[f] = scales[row * scale_pitch + col / kMxBlock];
        }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        const I w = w0 + f * kWarps, row = w / segs;
        if (w >= total) break;
        const int64_t col = static_cast<int64_t>(w - row * segs) * kSegCols + lane * 8;
        float v[8];
        mx_decode8<FMT>(codes[f], byte[f], v);
        store_cols<DT, VEC>(values + row * row_stride, col, cols, v);
    }
}

// The sum's eight values at `col`, rounded to the residual's type and stored, and their squares' sum.
template <int DT, bool VEC>
__device__ __forceinline__ double add_store(const typename Elem<DT>::T* hidden, const void* delta, bool delta_f32, int64_t col, int64_t cols,
                                           typename Elem<DT>::T* sum, float (&v)[8]) {
    load_cols<DT, VEC>(hidden, col, cols, v);
    if (delta != nullptr) {
        float d[8];
        if (delta_f32) load_cols<LM_DTYPE_F32, VEC>(static_cast<const float*>(delta), col, cols, d);
        else load_cols<LM_DTYPE_BF16, VEC>(static_cast<const __nv_bfloat16*>(delta), col, cols, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += d[i];
    }
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = Elem<DT>::widen(Elem<DT>::narrow(v[i]));
        s = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), s);
    }
    store_cols<DT, VEC>(sum, col, cols, v);
    return s;
}

// The norm's eight values at `col` to their bf16 copy, codes and scale byte.
template <bool VEC>
__device__ __forceinline__ void put_norm(float (&v)[8], float inverse, const float* weight, int64_t col, int64_t cols, __nv_bfloat16* out_bf16,
                                         int format, uint8_t* data, int64_t data_pitch, uint8_t* scales) {
    float g[8];
    load_cols<LM_DTYPE_F32, VEC>(weight, col, cols, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? v[i] * inverse * g[i] : 0.0f;
    if (out_bf16 != nullptr) store_cols<LM_DTYPE_BF16, VEC>(out_bf16, col, cols, v);
    uint32_t byte;
    if (format == LM_MX_E2M1) {
        byte = mx_scale_byte<LM_MX_E2M1>(v);
        store_codes<LM_MX_E2M1>(data, col, data_pitch, mx_encode8<LM_MX_E2M1>(v, byte));
    } else {
        byte = mx_scale_byte<LM_MX_E4M3>(v);
        store_codes<LM_MX_E4M3>(data, col, data_pitch, mx_encode8<LM_MX_E4M3>(v, byte));
    }
    if ((threadIdx.x & 3) == 0) scales[col / kMxBlock] = static_cast<uint8_t>(byte);
}

// The sum of s over the `T` threads of a row.
template <int T>
__device__ __forceinline__ double row_sum(double s, double* red) {
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if constexpr (T > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
        __syncthreads();
        s = 0.0;
        for (int i = 0; i < T / 32; ++i) s += red[i];
    }
    return s;
}

// T threads a row, eight columns each of every stretch of 8 T.  With CHUNKS > 0 that many
// stretches stay in registers between the sum and the norm; CHUNKS = 0 reads the stored sum again
// (each thread its own stores).  The sum is normalised as stored, its squares
// added in f64 as lm_gemm_rms_norm adds them.
template <int DT, bool VEC, int T, int CHUNKS>
__global__ void __launch_bounds__(kThreads)
    add_rms_norm_mx_kernel(const typename Elem<DT>::T* hidden, const void* delta, int delta_f32, const float* __restrict__ weight, int64_t rows,
                           int64_t cols, float eps, typename Elem<DT>::T* sum, __nv_bfloat16* __restrict__ out_bf16, int format,
                           uint8_t* __restrict__ data, int64_t data_pitch, uint8_t* __restrict__ scales, int64_t scale_pitch) {
    __shared__ double red[kWarps];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / T) + threadIdx.x / T;
    if (row >= rows) return;
    const int64_t first = threadIdx.x % T * 8, end = scale_pitch * kMxBlock;
    hidden += row * cols, sum += row * cols, data += row * data_pitch, scales += row * scale_pitch;
    if (delta != nullptr) delta = static_cast<const uint8_t*>(delta) + row * cols * (delta_f32 ? 4 : 2);
    if (out_bf16 != nullptr) out_bf16 += row * cols;
    double s = 0.0;
    if constexpr (CHUNKS > 0) {
        float v[CHUNKS][8];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) s += add_store<DT, VEC>(hidden, delta, delta_f32 != 0, first + c * T * 8, cols, sum, v[c]);
        const float inverse = static_cast<float>(1.0 / sqrt(row_sum<T>(s, red) / static_cast<double>(cols) + static_cast<double>(eps)));
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (first + c * T * 8 < end) put_norm<VEC>(v[c], inverse, weight, first + c * T * 8, cols, out_bf16, format, data, data_pitch, scales);
    } else {
        float v[8];
        for (int64_t col = first; col < cols; col += T * 8) s += add_store<DT, VEC>(hidden, delta, delta_f32 != 0, col, cols, sum, v);
        const float inverse = static_cast<float>(1.0 / sqrt(row_sum<T>(s, red) / static_cast<double>(cols) + static_cast<double>(eps)));
        for (int64_t col = first; col < end; col += T * 8) {
            load_cols<DT, VEC>(sum, col, cols, v);
            put_norm<VEC>(v, inverse, weight, col, cols, out_bf16, format, data, data_pitch, scales);
        }
    }
}

bool is_mx_format(int32_t format) { return format == LM_MX_E2M1 || format == LM_MX_E4M3; }

// Calls f with the segments' number in the type that holds it, and the grid for them.
template <class F>
lm_status with_segments(int64_t segments, F&& f) {
    const int64_t each = kWarps * kFlight, blocks = (segments + each - 1) / each;
    if (blocks > INT32_MAX) return context_free_fail(LM_ERR_UNSUPPORTED, "an MX matrix of more than 2^44 columns in all");
    if (segments <= INT32_MAX - each) f(static_cast<uint32_t>(segments), static_cast<unsigned>(blocks));
    else f(segments, static_cast<unsigned>(blocks));
    return context_free_finish(cudaGetLastError());
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
    return with_segments(rows * segs, [&](auto total, unsigned grid) {
        with_dtype(dtype, [&](auto dt) {
            with_format(format, [&](auto fmt) {
                with_bool(vec, [&](auto v) {
                    using T = typename Elem<decltype(dt)::value>::T;
                    mx_quantize_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(v)::value><<<grid, kThreads, 0, s>>>(
                        static_cast<const T*>(values), total, cols, row_stride, segs, data, mx_data_pitch(format, cols), scales);
                });
            });
        });
    });
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
    return with_segments(rows * segs, [&](auto total, unsigned grid) {
        with_dtype(dtype, [&](auto dt) {
            with_format(format, [&](auto fmt) {
                with_bool(vec, [&](auto v) {
                    using T = typename Elem<decltype(dt)::value>::T;
                    mx_dequantize_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(v)::value><<<grid, kThreads, 0, s>>>(
                        data, mx_data_pitch(format, cols), scales, mx_scale_pitch(cols), total, cols, segs, static_cast<T*>(values), row_stride);
                });
            });
        });
    });
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
    // Rows of a whole number of 16-byte words, all starting on one: eight columns a load.
    const bool vec = count % 8 == 0 && aligned(hidden, 16) && aligned(sum, 16) && aligned(delta, 16) && aligned(out_bf16, 16) && aligned(weight, 16);
    const int64_t wide = mx_scale_pitch(count) * kMxBlock;
    // A warp a row while its registers hold the row and there are enough rows to fill the GPU (16384
    // rows of 2048 bf16: MEASURE); else a CTA a row, for the latency of few rows and for wide ones.
    const bool warp_rows = wide <= 2048 && rows >= 148 * 4 * kWarps;
    with_bool(dtype == LM_DTYPE_F32, [&](auto hf) {
        with_bool(vec, [&](auto v) {
            constexpr int DT = decltype(hf)::value ? LM_DTYPE_F32 : LM_DTYPE_BF16;
            constexpr bool VEC = decltype(v)::value;
            using T = typename Elem<DT>::T;
            const auto go = [&](auto threads, auto chunks) {
                constexpr int per = kThreads / decltype(threads)::value;
                add_rms_norm_mx_kernel<DT, VEC, decltype(threads)::value, decltype(chunks)::value><<<static_cast<unsigned>((rows + per - 1) / per), kThreads, 0, s>>>(
                    static_cast<const T*>(hidden), delta, delta_dtype == LM_DTYPE_F32, weight, rows, count, epsilon, static_cast<T*>(sum),
                    reinterpret_cast<__nv_bfloat16*>(out_bf16), format, data, mx_data_pitch(format, count), scales, mx_scale_pitch(count));
            };
            if (warp_rows) go(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
            else if (wide <= 2048) go(std::integral_constant<int, kThreads>{}, std::integral_constant<int, 1>{});
            else if (wide <= 8192) go(std::integral_constant<int, kThreads>{}, std::integral_constant<int, 4>{});
            else go(std::integral_constant<int, kThreads>{}, std::integral_constant<int, 0>{});
        });
    });
    return context_free_finish(cudaGetLastError());
}

}  // extern "C"
