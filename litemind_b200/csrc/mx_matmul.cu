// mx_matmul.cu -- grouped products of microscaled (MX) matrices (lm_mx_matmul).
//
// out[r, n] = sum over k of X[r, k] W_g[n, k]: X in E4M3 or E2M1, W in E2M1, f32 sums.  A CTA
// decodes 64 x 64 tiles of X and W_g into shared memory as f32, 32 columns (one scale) at a time,
// and each thread keeps a 4 x 4 part of the output tile in registers.
#include "moe_internal.h"
#include "mx_block.cuh"

namespace lm {
namespace {

constexpr int kTile = 64;
constexpr int kThreads = 256;

template <int XF, int DT>
__global__ void __launch_bounds__(kThreads)
    mx_matmul_kernel(const uint8_t* __restrict__ x, int64_t x_pitch, const uint8_t* __restrict__ x_scales, int64_t rows,
                     const uint8_t* __restrict__ w, int64_t w_pitch, const uint8_t* __restrict__ w_scales, int64_t scale_pitch,
                     int groups, int64_t n, int64_t k, const int32_t* __restrict__ offsets, typename Elem<DT>::T* __restrict__ out,
                     int64_t out_stride) {
    __shared__ float sx[kTile][kMxBlock + 1], sw[kTile][kMxBlock + 1];
    __shared__ int64_t s_row0, s_row1;
    __shared__ int s_group;
    if (threadIdx.x == 0) {
        // The row tile's group: groups' tiles follow one another.
        int64_t tile = blockIdx.y, at = 0;
        s_group = -1;
        for (int g = 0; g < groups; ++g) {
            const int64_t zero = 0;
            const int64_t lo = max(at, offsets == nullptr ? zero : min(static_cast<int64_t>(offsets[g]), rows));
            const int64_t hi = max(lo, offsets == nullptr ? rows : min(static_cast<int64_t>(offsets[g + 1]), rows));
            at = hi;
            const int64_t tiles = (hi - lo + kTile - 1) / kTile;
            if (tile < tiles) {
                s_group = g;
                s_row0 = lo + tile * kTile;
                s_row1 = min(hi, s_row0 + kTile);
                break;
            }
            tile -= tiles;
        }
    }
    __syncthreads();
    if (s_group < 0) return;
    const int64_t row0 = s_row0, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int nr = static_cast<int>(s_row1 - row0);
    const int64_t w0 = static_cast<int64_t>(s_group) * n + n0;
    const int r = threadIdx.x >> 2, c8 = (threadIdx.x & 3) * 8;  // this thread's row and columns of each operand tile
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += kMxBlock) {
        float v[8] = {};
        if (r < nr) {
            const uint8_t* p = x + (row0 + r) * x_pitch + (k0 + c8) * (XF == LM_MX_E2M1 ? 4 : 8) / 8;
            uint2 codes = make_uint2(*reinterpret_cast<const uint32_t*>(p), 0u);
            if constexpr (XF == LM_MX_E4M3) codes = *reinterpret_cast<const uint2*>(p);
            mx_decode8<XF>(codes, x_scales[(row0 + r) * scale_pitch + k0 / kMxBlock], v);
        }
        for (int i = 0; i < 8; ++i) {
            sx[r][c8 + i] = v[i];
            v[i] = 0.0f;
        }
        if (n0 + r < n) {
            const uint2 codes = make_uint2(*reinterpret_cast<const uint32_t*>(w + (w0 + r) * w_pitch + (k0 + c8) / 2), 0u);
            mx_decode8<LM_MX_E2M1>(codes, w_scales[(w0 + r) * scale_pitch + k0 / kMxBlock], v);
        }
        for (int i = 0; i < 8; ++i) sw[r][c8 + i] = v[i];
        __syncthreads();
        for (int kk = 0; kk < kMxBlock; ++kk) {
            float a[4], b[4];
            for (int i = 0; i < 4; ++i) a[i] = sx[ty * 4 + i][kk], b[i] = sw[tx * 4 + i][kk];
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (ty * 4 + i < nr && n0 + tx * 4 + j < n)
                out[(row0 + ty * 4 + i) * out_stride + n0 + tx * 4 + j] = Elem<DT>::narrow(acc[i][j]);
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" {

lm_status lm_mx_matmul(const uint8_t* x, const uint8_t* x_scales, int32_t x_format, int64_t rows, const uint8_t* w, const uint8_t* w_scales,
                       int32_t groups, int64_t n, int64_t k, const int32_t* offsets, void* out, int32_t out_dtype, int64_t out_stride,
                       void* stream) {
    if ((x_format != LM_MX_E2M1 && x_format != LM_MX_E4M3) || !is_float_type(out_dtype))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_matmul: x is E2M1 or E4M3, out is f32, bf16 or f16");
    if (rows < 0 || rows > LM_MX_MAX_ROWS - 1024 || groups < 1 || groups > LM_MX_MAX_GROUPS || n < 0 || n > INT32_MAX / groups || k < 1 || k > LM_MX_MAX_COLS ||
        out_stride < n || (groups > 1 && offsets == nullptr))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_matmul: a size out of range, or groups without offsets");
    if (rows == 0 || n == 0) return LM_OK;
    if (out == nullptr || !aligned(out, elem_size(out_dtype)) || !aligned(offsets, 4) || x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr ||
        !aligned(x, 32) || !aligned(x_scales, 16) || !aligned(w, 32) || !aligned(w_scales, 16))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_matmul: a null pointer, or data not 32-byte or scales not 16-byte aligned");
    const int64_t tiles = (rows + kTile - 1) / kTile + groups - 1;
    if (tiles > 65535) return context_free_fail(LM_ERR_UNSUPPORTED, "lm_mx_matmul: too many rows");
    const dim3 grid(static_cast<unsigned>((n + kTile - 1) / kTile), static_cast<unsigned>(tiles));
    with_format(x_format, [&](auto xf) {
        with_dtype(out_dtype, [&](auto dt) {
            mx_matmul_kernel<decltype(xf)::value, decltype(dt)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                x, mx_data_pitch(x_format, k), x_scales, rows, w, mx_data_pitch(LM_MX_E2M1, k), w_scales, mx_scale_pitch(k), groups, n, k, offsets,
                static_cast<typename Elem<decltype(dt)::value>::T*>(out), out_stride);
        });
    });
    return context_free_finish(cudaGetLastError());
}

}  // extern "C"
