// elem.cuh -- f32, bf16 and f16 elements behind an LM_DTYPE_* constant, and what the entry points
// over them share: argument checks and the choice of an instantiation.
#pragma once

#include <cstdint>
#include <cstring>
#include <numeric>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "litemind_moe.h"

namespace lm {

// ── element types ─────────────────────────────────────────────────────────
template <int DT>
struct Elem;
template <>
struct Elem<LM_DTYPE_F32> {
    using T = float;
    static __device__ __forceinline__ float widen(float v) { return v; }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <>
struct Elem<LM_DTYPE_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<LM_DTYPE_F16> {
    using T = __half;
    static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
};

// Eight consecutive elements from / to a 16-byte aligned address.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* p, float (&v)[8]) {
    if constexpr (DT == LM_DTYPE_F32) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typename Elem<DT>::T e[2];
            memcpy(e, &w[i], 4);
            v[2 * i] = Elem<DT>::widen(e[0]);
            v[2 * i + 1] = Elem<DT>::widen(e[1]);
        }
    }
}
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::T* p, const float (&v)[8]) {
    if constexpr (DT == LM_DTYPE_F32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const typename Elem<DT>::T e[2] = {Elem<DT>::narrow(v[2 * i]), Elem<DT>::narrow(v[2 * i + 1])};
            memcpy(&w[i], e, 4);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Eight elements as they lie in memory: half the registers of their f32 values for 16-bit types
// while loads are in flight.
template <int DT>
struct Raw8 {
    alignas(16) uint32_t w[2 * sizeof(typename Elem<DT>::T)];
    __device__ __forceinline__ void load(const typename Elem<DT>::T* p) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) {
            const uint4 q = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
        }
    }
    __device__ __forceinline__ void narrow(const float (&v)[8]) { store8<DT>(reinterpret_cast<typename Elem<DT>::T*>(w), v); }
    __device__ __forceinline__ void store(typename Elem<DT>::T* p) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        typename Elem<DT>::T e[8];
        memcpy(e, w, sizeof e);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<DT>::widen(e[i]);
    }
};

// ── entry points ─────────────────────────────────────────────────────────
inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
// Rows of `width` bytes, `stride` bytes apart; a null pointer has none.
struct Span {
    const void* p;
    int64_t rows, stride, width;
    Span(const void* start, int64_t bytes) : Span(start, 1, bytes, bytes) {}
    Span(const void* start, int64_t n, int64_t step, int64_t bytes)
        : p(start), rows(n == 1 || step == bytes ? 1 : n), stride(step), width(n == 1 || step == bytes ? n * bytes : bytes) {}
};
// Whether two of them share a byte.  Columns side by side in one buffer do not: rows are compared
// modulo the strides' common step, which is exact for equal strides and for a single row, and for
// others may call rows shared that only come near one another.
inline bool overlap(const Span& a, const Span& b) {
    if (a.p == nullptr || b.p == nullptr || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
    using Wide = unsigned __int128;  // strides are the caller's
    const auto end = [](const Span& s) { return Wide(reinterpret_cast<uintptr_t>(s.p)) + Wide(s.rows - 1) * Wide(s.stride) + Wide(s.width); };
    const Wide x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    if (end(a) <= y || end(b) <= x) return false;
    if (a.rows == 1 && b.rows == 1) return true;
    const int64_t step = a.rows == 1 ? b.stride : b.rows == 1 ? a.stride : std::gcd(a.stride, b.stride);
    const int64_t ahead = static_cast<int64_t>(y >= x ? (y - x) % Wide(step) : (Wide(step) - (x - y) % Wide(step)) % Wide(step));
    return ahead < a.width || step - ahead < b.width;
}
inline int64_t elem_size(int32_t dtype) { return dtype == LM_DTYPE_F32 ? 4 : 2; }
inline bool is_float_type(int32_t dtype) { return dtype == LM_DTYPE_F32 || dtype == LM_DTYPE_BF16 || dtype == LM_DTYPE_F16; }

// Each calls f with the choice as a compile-time constant.
template <class F>
void with_dtype(int32_t dtype, F&& f) {
    if (dtype == LM_DTYPE_F32) f(std::integral_constant<int, LM_DTYPE_F32>{});
    else if (dtype == LM_DTYPE_BF16) f(std::integral_constant<int, LM_DTYPE_BF16>{});
    else f(std::integral_constant<int, LM_DTYPE_F16>{});
}
template <class F>
void with_format(int32_t format, F&& f) {
    if (format == LM_MX_E2M1) f(std::integral_constant<int, LM_MX_E2M1>{});
    else f(std::integral_constant<int, LM_MX_E4M3>{});
}
template <class F>
void with_bool(bool b, F&& f) {
    if (b) f(std::true_type{});
    else f(std::false_type{});
}

}  // namespace lm
