// mx_block.cuh -- microscaled (MX) rows: their layout and the encoding of one block.
//
// A row of `cols` values is stored as
//   codes   E4M3: one byte a value; E2M1: two values a byte, the even column in the low half;
//           zero codes up to a multiple of 128 columns
//   scales  one E8M0 byte (2^(byte - 127)) for each block of 32 columns; zero bytes up to a
//           multiple of 16, so that a row's scales move as 16-byte words
// The scale of a block is the largest power of two that keeps its largest magnitude below twice
// the format's largest power of two: biased exponent of max|v| minus emax (2 for E2M1, 8 for
// E4M3).  A code is v / scale rounded to nearest even and clamped to the largest finite value.
// Scaling by a power of two is exact, so that rounding is the only one.  A block that holds a NaN
// or an infinity has no such scale: its byte is 255 (NaN) and its codes are 0.
#pragma once

#include "elem.cuh"

namespace lm {

constexpr int kMxBlock = 32;
constexpr int kMxTileCols = 128;  // codes are padded to this many columns (a TMA box's width)

inline int64_t mx_padded_cols(int64_t cols) { return (cols + kMxTileCols - 1) / kMxTileCols * kMxTileCols; }
inline int64_t mx_data_pitch(int format, int64_t cols) {
    return format == LM_MX_E2M1 ? mx_padded_cols(cols) / 2 : mx_padded_cols(cols);
}
inline int64_t mx_scale_pitch(int64_t cols) { return (cols + 511) / 512 * 16; }

// ── one block, eight values in each of four neighbouring lanes ───────────
template <int FMT>
constexpr int kMxEmax = FMT == LM_MX_E2M1 ? 2 : 8;

// The scale byte of a block whose largest magnitude has these f32 bits.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    return static_cast<uint32_t>(max(static_cast<int>(top >> 23) - kMxEmax<FMT>, 0));
}
// The scale byte of the block that lanes 4i..4i+3 of this warp hold (all 32 lanes call it).
// Magnitudes order as their bits do, infinities and NaN above all.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(const float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    return mx_scale_of<FMT>(top);
}
// The same from the elements as they lie: 16-bit types two at a time.
template <int FMT, int DT>
__device__ __forceinline__ uint32_t mx_scale_byte(const Raw8<DT>& r) {
    if constexpr (DT == LM_DTYPE_F32) {
        float v[8];
        r.widen(v);
        return mx_scale_byte<FMT>(v);
    } else {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __vmaxu2(top, r.w[i] & 0x7fff7fffu);
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = max(top & 0xffffu, top >> 16);
        if constexpr (DT == LM_DTYPE_BF16) return mx_scale_of<FMT>(top << 16);
        else return mx_scale_of<FMT>(__float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top)))));
    }
}

// This lane's eight codes: 32 bits of E2M1, or 64 of E4M3 in (x, y).
template <int FMT>
__device__ __forceinline__ uint2 mx_encode8(const float (&v)[8], uint32_t scale_byte) {
    if (scale_byte == 255u) return make_uint2(0u, 0u);
    const float inv = __uint_as_float((254u - scale_byte) << 23);  // 2^(127 - byte); byte <= 252
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = v[i] * inv;
    uint2 r = make_uint2(0u, 0u);
    if constexpr (FMT == LM_MX_E2M1) {
        asm("{\n .reg .b8 a, b, c, d;\n"
            " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
            " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
            " mov.b32 %0, {a, b, c, d};\n}\n"
            : "=r"(r.x)
            : "f"(s[0]), "f"(s[1]), "f"(s[2]), "f"(s[3]), "f"(s[4]), "f"(s[5]), "f"(s[6]), "f"(s[7]));
    } else {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(h[i]) : "f"(s[2 * i]), "f"(s[2 * i + 1]));
        r.x = h[0] | (static_cast<uint32_t>(h[1]) << 16);
        r.y = h[2] | (static_cast<uint32_t>(h[3]) << 16);
    }
    return r;
}

// The eight values of such codes.  f16 holds every E2M1 and E4M3 value exactly.
template <int FMT>
__device__ __forceinline__ void mx_decode8(uint2 codes, uint32_t scale_byte, float (&v)[8]) {
    const float scale = __uint_as_float(scale_byte == 255u ? 0x7fc00000u : scale_byte == 0u ? 0x00400000u : scale_byte << 23);
    uint32_t h[4];
    if constexpr (FMT == LM_MX_E2M1) {
        asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
            " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
            " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(codes.x));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t pair = static_cast<uint16_t>((i < 2 ? codes.x : codes.y) >> (16 * (i & 1)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[i]) : "h"(pair));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 p;
        memcpy(&p, &h[i], 4);
        v[2 * i] = __low2float(p) * scale;
        v[2 * i + 1] = __high2float(p) * scale;
    }
}

// Lanes 4i of a warp hold the byte of block i: lane 0 gets blocks 0-3 and lane 16 blocks 4-7 as a word.
__device__ __forceinline__ uint32_t mx_gather_scales(uint32_t scale_byte, int lane) {
    uint32_t w = scale_byte << (8 * ((lane >> 2) & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    w |= __shfl_xor_sync(0xffffffffu, w, 8);
    return w;
}

}  // namespace lm
