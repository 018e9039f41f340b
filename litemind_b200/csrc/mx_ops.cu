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

// A warp takes kFlight segments of one row: block (x, y) holds rows kWarps x .. and segments
// kFlight y .. of each, so that no index needs a division (divisions cost as much as the conversion).
__device__ __forceinline__ int64_t warp_row() { return static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); }
__device__ __forceinline__ int64_t first_col() { return static_cast<int64_t>(blockIdx.y) * (kFlight * kSegCols) + (threadIdx.x & 31) * 8; }

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
__device__ __forceinline__ Raw8<DT> load_raw(const typename Elem<DT>::T* row, int64_t col, int64_t cols) {
    Raw8<DT> r;
    if (VEC && col + 8 <= cols) {
        r.load(row + col);
    } else {
        typename Elem<DT>::T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = col + i < cols ? row[col + i] : Elem<DT>::narrow(0.0f);
        memcpy(r.w, e, sizeof e);
    }
    return r;
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

// Each segment has 8 scale bytes; the last ones of a row may be padding only.
template <int DT, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const typename Elem<DT>::T* __restrict__ values, int64_t rows, int64_t cols, int64_t row_stride, uint8_t* __restrict__ data,
                       int64_t data_pitch, uint8_t* __restrict__ scales, int64_t scale_pitch) {
    const int lane = threadIdx.x & 31;
    const int64_t row = warp_row(), col0 = first_col();
    if (row >= rows) return;
    values += row * row_stride, data += row * data_pitch, scales += row * scale_pitch;
    Raw8<DT> raw[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) raw[f] = load_raw<DT, VEC>(values, col0 + f * kSegCols, cols);
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        const int64_t col = col0 + f * kSegCols;
        if (col >= scale_pitch * kMxBlock) break;  // the same for a whole warp: pitches are multiples of 8 bytes
        const uint32_t byte = mx_scale_byte<FMT>(raw[f]);
        float v[8];
        raw[f].widen(v);
        store_codes<FMT>(data, col, data_pitch, mx_encode8<FMT>(v, byte));
        const uint32_t word = mx_gather_scales(byte, lane);
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + col / kMxBlock) = word;
    }
}

template <int DT, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t* __restrict__ data, int64_t data_pitch, const uint8_t* __restrict__ scales, int64_t scale_pitch, int64_t rows,
                         int64_t cols, typename Elem<DT>::T* __restrict__ values, int64_t row_stride) {
    const int64_t row = warp_row(), col0 = first_col();
    if (row >= rows) return;
    values += row * row_stride;
    if constexpr (!VEC) {
        // Rows that do not start on whole words: lane i takes column i of each block, so that stores
        // run along the row (8192 x 2047 to bf16 took 51 us with eight neighbouring columns a lane).
        const int lane = threadIdx.x & 31;
        data += row * data_pitch, scales += row * scale_pitch;
        const int64_t col1 = min(cols, static_cast<int64_t>(blockIdx.y + 1) * (kFlight * kSegCols));
#pragma unroll 8
        for (int64_t col = static_cast<int64_t>(blockIdx.y) * (kFlight * kSegCols) + lane; col < col1; col += kMxBlock) {
            uint32_t code = FMT == LM_MX_E2M1 ? data[col / 2] : data[col];
            if (FMT == LM_MX_E2M1 && (col & 1)) code >>= 4;
            float v[8];
            mx_decode8<FMT>(make_uint2(code, 0u), scales[col / kMxBlock], v);
            values[col] = Elem<DT>::narrow(v[0]);
        }
        return;
    }
    data += row * data_pitch + col0 * (FMT == LM_MX_E2M1 ? 4 : 8) / 8, scales += row * scale_pitch + col0 / kMxBlock;
    uint2 codes[kFlight];
    uint32_t byte[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        codes[f] = make_uint2(0u, 0u);
        byte[f] = 0;
        if (col0 + f * kSegCols < cols) {
            if constexpr (FMT == LM_MX_E2M1) codes[f].x = *reinterpret_cast<const uint32_t*>(data + f * (kSegCols / 2));
            else codes[f] = *reinterpret_cast<const uint2*>(data + f * kSegCols);
            byte[f] = scales[f * (kSegCols / kMxBlock)];
        }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        if (col0 + f * kSegCols >= cols) break;
        float v[8];
        mx_decode8<FMT>(codes[f], byte[f], v);
        store_cols<DT, VEC>(values, col0 + f * kSegCols, cols, v);
    }
}

// Eight columns of the residual and of its update as they lie in memory, so that the loads of both
// and of every stretch are in flight together: whatever converts the first of them waits for it.
template <int DT>
struct Pair8 {
    Raw8<DT> hidden;
    Raw8<LM_DTYPE_F32> delta;  // bf16: in the first half
};
template <int DT, bool VEC, int N>
__device__ __forceinline__ void load_pairs(const typename Elem<DT>::T* hidden, const void* delta, bool delta_f32, int64_t col, int64_t step, int64_t cols,
                                           Pair8<DT> (&p)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) p[c].hidden = load_raw<DT, VEC>(hidden, col + c * step, cols);
    if (delta == nullptr) return;
    if (delta_f32) {
#pragma unroll
        for (int c = 0; c < N; ++c) p[c].delta = load_raw<LM_DTYPE_F32, VEC>(static_cast<const float*>(delta), col + c * step, cols);
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const Raw8<LM_DTYPE_BF16> d = load_raw<LM_DTYPE_BF16, VEC>(static_cast<const __nv_bfloat16*>(delta), col + c * step, cols);
            memcpy(p[c].delta.w, d.w, sizeof d.w);
        }
    }
}
// Their sum, rounded to the residual's type and stored, in v; returns the sum of its squares.
template <int DT, bool VEC>
__device__ __forceinline__ double add_store(const Pair8<DT>& p, bool add, bool delta_f32, float (&v)[8], int64_t col, int64_t cols,
                                            typename Elem<DT>::T* sum) {
    double s = 0.0;
    p.hidden.widen(v);
    if (add) {
        float d[8];
        if (delta_f32) {
            p.delta.widen(d);
        } else {
            Raw8<LM_DTYPE_BF16> half;
            memcpy(half.w, p.delta.w, sizeof half.w);
            half.widen(d);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += d[i];
    }
    Raw8<DT> r;  // rounded once, for the store and the norm
    r.narrow(v);
    r.widen(v);
    if (VEC && col + 8 <= cols) r.store(sum + col);
    else store_cols<DT, false>(sum, col, cols, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), s);
    return s;
}

// The norm's eight values at `col` to their bf16 copy, codes and scale byte.
template <bool VEC>
__device__ __forceinline__ void put_norm(float (&v)[8], float inverse, const float* weight, int64_t col, int64_t cols, __nv_bfloat16* out_bf16,
                                         int format, uint8_t* data, int64_t data_pitch, uint8_t* scales) {
    float g[8];
    load_cols<LM_DTYPE_F32, VEC>(weight, col, cols, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inverse * g[i];
    if (VEC ? col >= cols : col + 8 > cols) {  // an infinite inverse leaves NaN past the row's end
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (VEC || col + i >= cols) v[i] = 0.0f;
    }
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

// The inverse root of the CTA's mean square: its first warp's work, 15% of the instructions of a row
// of 2048 when every thread did it.  Rounded to f32: it overflows below a root mean square of 2^-127, with
// epsilon 0 only (a second factor for such rows cost the others 1% or more).
template <int T>
__device__ __forceinline__ float block_inverse(double s, double inv_cols, double eps) {
    __shared__ double red[32];
    __shared__ float inverse;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (lane == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = lane < T / 32 ? red[lane] : 0.0;
#pragma unroll
        for (int off = T / 64 > 8 ? 16 : T / 64 > 4 ? 8 : 4; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        if (lane == 0) inverse = static_cast<float>(rsqrt(s * inv_cols + eps));
    }
    __syncthreads();
    return inverse;
}

// A CTA of T threads a row, eight columns a thread of every stretch of 8 T.  With CHUNKS > 0 that
// many stretches are loaded before anything is converted or stored (sum may be hidden or delta, so
// the compiler cannot), and stay in registers between the sum and the norm; CHUNKS = 0 reads the
// stored sum again (each thread its own stores).  The sum is normalised as stored, its squares added
// in f64 as lm_gemm_rms_norm adds them.  bf16 rows: 16384 x 2048 in 44 us, 5.4 TB/s, of which
// instructions take most (issue slots 77% busy at 49 us; with loads converted one after another two
// stretches took 56 us, with 48 registers a thread 47); f32 rows: 65 us, HBM's rate.
template <int DT, bool VEC, int T, int CHUNKS>
__global__ void __launch_bounds__(T, VEC && CHUNKS != 1 ? 1536 / T : 1)
    add_rms_norm_mx_kernel(const typename Elem<DT>::T* hidden, const void* delta, int delta_f32, const float* __restrict__ weight, int64_t cols,
                           double inv_cols, double eps, typename Elem<DT>::T* sum, __nv_bfloat16* __restrict__ out_bf16, int format,
                           uint8_t* __restrict__ data, int64_t data_pitch, uint8_t* __restrict__ scales, int64_t scale_pitch) {
    const int64_t row = blockIdx.x, first = threadIdx.x * 8, end = scale_pitch * kMxBlock;
    hidden += row * cols, sum += row * cols, data += row * data_pitch, scales += row * scale_pitch;
    if (delta != nullptr) delta = static_cast<const uint8_t*>(delta) + row * cols * (delta_f32 ? 4 : 2);
    if (out_bf16 != nullptr) out_bf16 += row * cols;
    double s = 0.0;
    if constexpr (CHUNKS > 0) {
        Pair8<DT> p[CHUNKS];
        float v[CHUNKS][8];
        load_pairs<DT, VEC>(hidden, delta, delta_f32 != 0, first, T * 8, cols, p);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) s += add_store<DT, VEC>(p[c], delta != nullptr, delta_f32 != 0, v[c], first + c * T * 8, cols, sum);
        const float inverse = block_inverse<T>(s, inv_cols, eps);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (first + c * T * 8 < end) put_norm<VEC>(v[c], inverse, weight, first + c * T * 8, cols, out_bf16, format, data, data_pitch, scales);
    } else {
        float v[8];
        for (int64_t col = first; col < cols; col += T * 8) {
            Pair8<DT> p[1];
            load_pairs<DT, VEC>(hidden, delta, delta_f32 != 0, col, 0, cols, p);
            s += add_store<DT, VEC>(p[0], delta != nullptr, delta_f32 != 0, v, col, cols, sum);
        }
        const float inverse = block_inverse<T>(s, inv_cols, eps);
        for (int64_t col = first; col < end; col += T * 8) {
            load_cols<DT, VEC>(sum, col, cols, v);
            put_norm<VEC>(v, inverse, weight, col, cols, out_bf16, format, data, data_pitch, scales);
        }
    }
}

bool is_mx_format(int32_t format) { return format == LM_MX_E2M1 || format == LM_MX_E4M3; }

// Blocks of kWarps rows by kFlight segments.
dim3 grid_for(int64_t rows, int64_t cols) {
    return dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps), static_cast<unsigned>((cols + kFlight * kSegCols - 1) / (kFlight * kSegCols)));
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
    const Span from(values, rows, row_stride * elem_size(dtype), cols * elem_size(dtype)), codes(data, rows * mx_data_pitch(format, cols)),
        bytes(scales, rows * mx_scale_pitch(cols));
    if (overlap(codes, from) || overlap(bytes, from) || overlap(codes, bytes))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_quantize: values, data and scales overlap");
    const bool vec = aligned(values, 16) && row_stride * elem_size(dtype) % 16 == 0;
    const dim3 grid = grid_for(rows, mx_scale_pitch(cols) * kMxBlock);
    with_dtype(dtype, [&](auto dt) {
        with_format(format, [&](auto fmt) {
            with_bool(vec, [&](auto v) {
                using T = typename Elem<decltype(dt)::value>::T;
                mx_quantize_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    static_cast<const T*>(values), rows, cols, row_stride, data, mx_data_pitch(format, cols), scales, mx_scale_pitch(cols));
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
    const Span to(values, rows, row_stride * elem_size(dtype), cols * elem_size(dtype));
    if (overlap(to, {data, rows * mx_data_pitch(format, cols)}) || overlap(to, {scales, rows * mx_scale_pitch(cols)}))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_dequantize: values overlaps data or scales");
    const bool vec = aligned(values, 16) && row_stride * elem_size(dtype) % 16 == 0;
    const dim3 grid = grid_for(rows, cols);
    with_dtype(dtype, [&](auto dt) {
        with_format(format, [&](auto fmt) {
            with_bool(vec, [&](auto v) {
                using T = typename Elem<decltype(dt)::value>::T;
                mx_dequantize_kernel<decltype(dt)::value, decltype(fmt)::value, decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    data, mx_data_pitch(format, cols), scales, mx_scale_pitch(cols), rows, cols, static_cast<T*>(values), row_stride);
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
    const Span total(sum, rows * count * elem_size(dtype)), plain(out_bf16, rows * count * 2), codes(data, rows * mx_data_pitch(format, count)),
        bytes_of_scales(scales, rows * mx_scale_pitch(count)), gain(weight, count * 4);
    for (const Span* out : {&plain, &codes, &bytes_of_scales})
        if (overlap(*out, {hidden, rows * count * elem_size(dtype)}) || overlap(*out, {delta, rows * count * elem_size(delta_dtype)}) || overlap(*out, gain) || overlap(*out, total))
            return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_gemm_add_rms_norm_mx: out_bf16, data or scales overlaps an input or sum");
    if (overlap(plain, codes) || overlap(plain, bytes_of_scales) || overlap(codes, bytes_of_scales) || overlap(total, gain))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_gemm_add_rms_norm_mx: out_bf16, data and scales overlap, or sum overlaps weight");
    // Each thread stores the sum over the values it loaded and nobody else's.
    const int64_t bytes = rows * count * elem_size(dtype), delta_bytes = rows * count * elem_size(delta_dtype);
    if ((sum != hidden && overlap({sum, bytes}, {hidden, bytes})) || ((sum != delta || delta_dtype != dtype) && overlap({sum, bytes}, {delta, delta_bytes})))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_gemm_add_rms_norm_mx: sum overlaps a part of hidden or delta, or a delta of another type");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Rows of a whole number of 16-byte words, all starting on one: eight columns a load.
    const bool vec = count % 8 == 0 && aligned(hidden, 16) && aligned(sum, 16) && aligned(delta, 16) && aligned(out_bf16, 16) && aligned(weight, 16);
    const int64_t wide = mx_scale_pitch(count) * kMxBlock;
    with_bool(dtype == LM_DTYPE_F32, [&](auto hf) {
        with_bool(vec, [&](auto v) {
            constexpr int DT = decltype(hf)::value ? LM_DTYPE_F32 : LM_DTYPE_BF16;
            constexpr bool VEC = decltype(v)::value;
            using T = typename Elem<DT>::T;
            const auto go = [&](auto threads, auto chunks) {
                constexpr int N = decltype(threads)::value;
                add_rms_norm_mx_kernel<DT, VEC, N, decltype(chunks)::value><<<static_cast<unsigned>(rows), N, 0, s>>>(
                    static_cast<const T*>(hidden), delta, delta_dtype == LM_DTYPE_F32, weight, count, 1.0 / static_cast<double>(count), epsilon, static_cast<T*>(sum),
                    reinterpret_cast<__nv_bfloat16*>(out_bf16), format, data, mx_data_pitch(format, count), scales, mx_scale_pitch(count));
            };
            // T threads for every eight of the widest row of a class (bf16 rows of 1024 took 31 us with 128
            // threads and 49 with 256, 20000 rows).  bf16 rows that fill the GPU three times over, which
            // instructions bound, take two stretches a thread (us, two and one: 16384 x 2048 44 and 49, 4096 x
            // 8192 49 and 56, 4000 x 2048 12.8 and 13.3); fewer rows, where latency counts, and f32 rows,
            // which HBM bounds, take one (2000 x 2048 7.2 and 6.5, 8192 x 8192 f32 136 and 132).  Wider
            // rows read their sum again (2048 x 16384: 63, held in registers 80; 20 to 32 bytes spilled).
            // Below a class's top the CTA's last threads idle: rows of 2560 bf16 columns go at 68% of the
            // rate of 2048, of 5120 at 86% of 4096's (f32: 89 and 88%).
            const bool many = rows * wide > int64_t(3) * 148 * 2048 * 8;
            const auto fit = [&](auto stretches) {
                constexpr int C = decltype(stretches)::value;
                if (wide <= 1024) go(std::integral_constant<int, 128 / C>{}, stretches);
                else if (wide <= 2048) go(std::integral_constant<int, 256 / C>{}, stretches);
                else if (wide <= 4096) go(std::integral_constant<int, 512 / C>{}, stretches);
                else if (wide <= 6144) go(std::integral_constant<int, 768 / C>{}, stretches);
                else go(std::integral_constant<int, 1024 / C>{}, stretches);
            };
            if (wide > 8192) {
                if (many) go(std::integral_constant<int, 512>{}, std::integral_constant<int, 0>{});
                else go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 0>{});
            } else if constexpr (DT == LM_DTYPE_BF16) {
                if (many) fit(std::integral_constant<int, 2>{});
                else fit(std::integral_constant<int, 1>{});
            } else {
                fit(std::integral_constant<int, 1>{});
            }
        });
    });
    return context_free_finish(cudaGetLastError());
}

}  // extern "C"
