// mx_matmul.cu -- grouped products of microscaled (MX) matrices (lm_mx_matmul) on the block-scaled
// tcgen05 tensor cores.
//
//   D[128 rows of W_g, BN rows of X] = W_g X^T,   out[r, n] = D[n, r]
//
// The weights are the MMA's M side, so that a few rows of X cost a narrow N instead of a padded M.
// One persistent CTA an SM walks the tiles (group, BN rows of X, 128 rows of W).  Its warps:
//   0      TMA producer: a ring of stages of 128 columns.  4-bit codes travel packed (half a byte a
//          column from HBM and L2) and are spread by the TMA into the MMA's padded form.
//   1      MMA issuer: four block-scaled MMAs of 32 columns a stage, one scale byte each
//   4-7    scales, straight from their rows to TMEM (no shared memory): a lane loads 16 bytes of a
//          row, the scales of four stages; each warp writes its own quadrant's copy
//   8-11   epilogue: TMEM to registers to out, rounded once; double buffered against the MMA
// Every wait is bounded (ptx.cuh): a pipeline that stalls records a status for lm_mx_sync.
#include "moe_internal.h"
#include "mx_block.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace lm {
namespace {

constexpr int kBlockM = 128;
constexpr int kStageCols = 128;     // columns of a stage: one 128-byte row of the swizzled tiles
constexpr int kSfStages = 4;        // stages of one scale group: 16 scale bytes a row
constexpr int kThreads = 384;
constexpr int kSms = 148;
constexpr int kATileBytes = kBlockM * kStageCols;

template <int BN>
struct Cfg {
    static constexpr int kBTileBytes = BN * kStageCols;
    static constexpr int kStageBytes = kATileBytes + kBTileBytes;
    static constexpr int kFit = 212 * 1024 / kStageBytes;
    static constexpr int kStages = kFit > 12 ? 12 : kFit;
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes;
    static constexpr int kAccs = BN <= 128 ? 2 : 1;                // accumulators in TMEM
    static constexpr int kSfbCols = BN <= 128 ? 4 : BN / 32;       // TMEM columns of a stage's X scales
    static constexpr int kSfCols = kSfStages * (4 + kSfbCols);     // TMEM columns of a scale group
    static constexpr int kSfGroups = std::min(8, (512 - kAccs * BN) / kSfCols);
    static_assert(BN % 16 == 0 && BN >= 16 && BN <= 256, "N of an M = 128 MMA");
    static_assert(kStages >= 3 && kSfGroups >= 2, "rings");
};

struct Args {
    const uint8_t* x_scales;
    const uint8_t* w_scales;
    const int32_t* offsets;  // or null: one group of all rows
    void* out;
    int64_t out_stride;
    int64_t scale_pitch;
    int64_t w_rows;  // groups * n
    int rows, groups, n;
    int k_stages;
    int x_four_bit;
    int out_dtype;
    int* status;
};

__device__ int g_status;  // the first device-side error since the last lm_mx_sync

// Where group g's rows start (cut[g]) and its first column tile (tiles[g]); one warp.  Offsets are
// clamped to the rows and to ascending order, so no value of theirs leads outside the matrices.
template <int BN>
__device__ void cut_groups(const Args& a, int* cut, int* tiles) {
    const int lane = threadIdx.x & 31;
    if (a.offsets == nullptr) {
        if (lane == 0) {
            cut[0] = 0, cut[1] = a.rows;
            tiles[0] = 0, tiles[1] = (a.rows + BN - 1) / BN;
        }
        return;
    }
    int last = min(max(a.offsets[0], 0), a.rows), sum = 0;
    if (lane == 0) cut[0] = last, tiles[0] = 0;
    int next = lane < a.groups ? a.offsets[lane + 1] : 0;
    for (int g0 = 0; g0 < a.groups; g0 += 32) {
        int c = min(next, a.rows);
        if (g0 + 32 + lane < a.groups) next = a.offsets[g0 + 32 + lane + 1];
        c = max(c, last);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, c, d);
            if (lane >= d) c = max(c, o);
        }
        int before = __shfl_up_sync(0xffffffffu, c, 1);
        if (lane == 0) before = last;
        const bool live = g0 + lane < a.groups;
        int t = live ? (c - before + BN - 1) / BN : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, t, d);
            if (lane >= d) t += o;
        }
        if (live) cut[g0 + lane + 1] = c, tiles[g0 + lane + 1] = sum + t;
        sum += __shfl_sync(0xffffffffu, t, 31);
        last = __shfl_sync(0xffffffffu, c, min(31, a.groups - 1 - g0));
    }
}

struct Tile {
    int group, row0, rows;  // rows of X: row0 .. row0 + rows - 1
    int n0;                 // first row of W_g
};

template <int BN>
__device__ __forceinline__ Tile tile_at(const Args& a, const int* cut, const int* tiles, int t, int m_blocks) {
    const int ct = t / m_blocks;
    int lo = 0, hi = a.groups;  // tiles[lo] <= ct < tiles[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tiles[mid] <= ct) lo = mid; else hi = mid;
    }
    Tile r;
    r.group = lo;
    r.row0 = cut[lo] + (ct - tiles[lo]) * BN;
    r.rows = min(BN, cut[lo + 1] - r.row0);
    r.n0 = (t - ct * m_blocks) * kBlockM;
    return r;
}

template <int DT>
__device__ __forceinline__ void store_columns(void* out, int64_t at, int64_t stride, int cols, const uint32_t (&v)[16]) {
    typename Elem<DT>::T* p = static_cast<typename Elem<DT>::T*>(out) + at;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < cols) p[i * stride] = Elem<DT>::narrow(__uint_as_float(v[i]));
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
    mx_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Args a) {
    using C = Cfg<BN>;
    constexpr int S = C::kStages, G = C::kSfGroups;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int s_cut[LM_MX_MAX_GROUPS + 1], s_tiles[LM_MX_MAX_GROUPS + 1];
    __shared__ uint64_t full[S], empty[S], sf_full[G], sf_empty[G], tmem_full[C::kAccs], tmem_empty[C::kAccs], drain;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t* smem_a = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_b = smem_a + S * kATileBytes;
    volatile int* abort_flag = &s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_x);
        for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < G; ++i) mbar_init(&sf_full[i], 4), mbar_init(&sf_empty[i], 1);
        for (int i = 0; i < C::kAccs; ++i) mbar_init(&tmem_full[i], 1), mbar_init(&tmem_empty[i], 4);
        mbar_init(&drain, 1);
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    if (warp == 2) cut_groups<BN>(a, s_cut, s_tiles);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t tmem_sf = tmem + C::kAccs * BN;
    const int m_blocks = (a.n + kBlockM - 1) / kBlockM;
    const int total = s_tiles[a.groups] * m_blocks;

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t bytes = kATileBytes / 2 + (a.x_four_bit ? C::kBTileBytes / 2 : C::kBTileBytes);
            int stage = 0;
            uint32_t phase = 0, issued = 0, issued_phase = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
                const Tile tile = tile_at<BN>(a, s_cut, s_tiles, t, m_blocks);
                const int w_row = tile.group * a.n + tile.n0;
                for (int s = 0; s < a.k_stages; ++s) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, a.status, kDevTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&full[stage], bytes);
                    tma_load_2d(smem_a + stage * kATileBytes, &map_w, &full[stage], s * kStageCols, w_row);
                    tma_load_2d(smem_b + stage * C::kBTileBytes, &map_x, &full[stage], s * kStageCols, tile.row0);
                    issued |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == S) stage = 0, phase ^= 1u;
                }
            }
            if (!ok)  // copies in flight land before the CTA's shared memory is given up
                for (int i = 0; i < S; ++i)
                    if (issued & (1u << i)) mbar_wait_drain(&full[i], (issued_phase >> i) & 1u, 100000000ull);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, sg = 0, acc = 0;
            uint32_t phase = 0, sf_phase = 0, acc_phase = 0;
            bool ok = true, any = false;
            const uint32_t b_format = a.x_four_bit ? kUmmaE2M1 : kUmmaE4M3;
            for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
                if (!mbar_wait(&tmem_empty[acc], acc_phase ^ 1u, abort_flag, a.status, kDevTimeoutMma)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc * BN;
                for (int s = 0; s < a.k_stages; ++s) {
                    const int sub = s & (kSfStages - 1);
                    if (sub == 0 && !mbar_wait(&sf_full[sg], sf_phase, abort_flag, a.status, kDevTimeoutMma)) {
                        ok = false;
                        break;
                    }
                    if (!mbar_wait(&full[stage], phase, abort_flag, a.status, kDevTimeoutMma)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t da = umma_desc_sw128(smem_u32(smem_a + stage * kATileBytes));
                    const uint64_t db = umma_desc_sw128(smem_u32(smem_b + stage * C::kBTileBytes));
                    const uint32_t sfa = tmem_sf + sg * C::kSfCols + sub * 4;
                    const uint32_t sfb = tmem_sf + sg * C::kSfCols + 4 * kSfStages + sub * C::kSfbCols;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)  // 32 columns are 32 bytes, 2 in the descriptor's units
                        umma_mx(d, da + 2 * kk, db + 2 * kk, umma_idesc_mx(kUmmaE2M1, b_format, kBlockM, BN, kk), sfa, sfb,
                                s != 0 || kk != 0);
                    any = true;
                    umma_commit(&empty[stage]);
                    if (++stage == S) stage = 0, phase ^= 1u;
                    if (sub == kSfStages - 1 || s == a.k_stages - 1) {
                        umma_commit(&sf_empty[sg]);
                        if (++sg == G) sg = 0, sf_phase ^= 1u;
                    }
                }
                if (!ok) break;
                umma_commit(&tmem_full[acc]);
                if (++acc == C::kAccs) acc = 0, acc_phase ^= 1u;
            }
            if (!ok && any) {  // the MMAs issued so far end before TMEM is released
                umma_commit(&drain);
                mbar_wait_drain(&drain, 0, 100000000ull);
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const uint32_t quad = static_cast<uint32_t>(warp & 3) * 32u << 16;
        constexpr int kXRows = (BN + 31) / 32;
        const int sf_groups = (a.k_stages + kSfStages - 1) / kSfStages;
        int sg = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
            const Tile tile = tile_at<BN>(a, s_cut, s_tiles, t, m_blocks);
            const int64_t w_row = static_cast<int64_t>(tile.group) * a.n + tile.n0 + lane;
            const uint8_t* wp = a.w_scales + w_row * a.scale_pitch;
            const uint8_t* xp = a.x_scales + (static_cast<int64_t>(tile.row0) + lane) * a.scale_pitch;
            for (int q = 0; ok && q < sf_groups; ++q) {
                uint4 w[4], x[kXRows];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    w[c] = w_row + 32 * c < a.w_rows ? __ldg(reinterpret_cast<const uint4*>(wp + 32 * c * a.scale_pitch + 16 * q))
                                                     : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < kXRows; ++c)
                    x[c] = tile.row0 + lane + 32 * c < a.rows ? __ldg(reinterpret_cast<const uint4*>(xp + 32 * c * a.scale_pitch + 16 * q))
                                                              : make_uint4(0, 0, 0, 0);
                // lane 0 polls: the warp goes on together
                int go = 1;
                if (lane == 0) go = mbar_wait(&sf_empty[sg], phase ^ 1u, abort_flag, a.status, kDevTimeoutProducer);
                ok = __shfl_sync(0xffffffffu, go, 0) != 0;
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = tmem_sf + quad + sg * C::kSfCols;
                uint32_t r[16];
#pragma unroll
                for (int c = 0; c < 4; ++c) r[c] = w[c].x, r[4 + c] = w[c].y, r[8 + c] = w[c].z, r[12 + c] = w[c].w;
                tmem_st16(at, r);
#pragma unroll
                for (int h = 0; h < C::kSfbCols / 4; ++h) {  // 16 words: X rows in fours, or two stages of eight
                    uint32_t u[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int word = h * 16 + i, sub = word / C::kSfbCols, c = word % C::kSfbCols;
                        u[i] = 0;
                        if (c < kXRows) u[i] = sub == 0 ? x[c].x : sub == 1 ? x[c].y : sub == 2 ? x[c].z : x[c].w;
                    }
                    tmem_st16(at + 16 + 16 * h, u);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sf_full[sg]);
                if (++sg == G) sg = 0, phase ^= 1u;
            }
        }
    } else if (warp >= 8) {
        const int quad = warp & 3;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x) {
            const Tile tile = tile_at<BN>(a, s_cut, s_tiles, t, m_blocks);
            int go = 1;
            if (lane == 0) go = mbar_wait(&tmem_full[acc], acc_phase, abort_flag, a.status, kDevTimeoutEpilogue);
            if (__shfl_sync(0xffffffffu, go, 0) == 0) break;
            tc_fence_after();
            const int n = tile.n0 + quad * 32 + lane;
            const uint32_t src = tmem + acc * BN + (static_cast<uint32_t>(quad * 32) << 16);
            for (int c0 = 0; c0 < tile.rows; c0 += 16) {
                uint32_t v[16];
                tmem_ld16(src + c0, v);
                tmem_ld_wait();
                if (n < a.n) {
                    const int64_t at = (static_cast<int64_t>(tile.row0) + c0) * a.out_stride + n;
                    const int cols = tile.rows - c0;
                    if (a.out_dtype == LM_DTYPE_F32) store_columns<LM_DTYPE_F32>(a.out, at, a.out_stride, cols, v);
                    else if (a.out_dtype == LM_DTYPE_BF16) store_columns<LM_DTYPE_BF16>(a.out, at, a.out_stride, cols, v);
                    else store_columns<LM_DTYPE_F16>(a.out, at, a.out_stride, cols, v);
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_empty[acc]);
            if (++acc == C::kAccs) acc = 0, acc_phase ^= 1u;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

template <int BN>
lm_status launch(const CUtensorMap& map_w, const uint8_t* x, int64_t rows, int64_t cols, Args a, int64_t tiles, cudaStream_t stream) {
    using C = Cfg<BN>;
    CUtensorMap map_x;
    std::string error;
    if (!encode_tensor_map_mx(&map_x, x, a.x_four_bit != 0, static_cast<uint64_t>(rows), static_cast<uint64_t>(cols), BN, error))
        return context_free_fail(LM_ERR_CUDA, error.c_str());
    if (const cudaError_t e = cudaFuncSetAttribute(mx_matmul_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes); e != cudaSuccess)
        return context_free_finish(e);
    mx_matmul_kernel<BN><<<static_cast<unsigned>(std::min<int64_t>(tiles, kSms)), kThreads, C::kSmemBytes, stream>>>(map_w, map_x, a);
    return context_free_finish(cudaGetLastError());
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
    if (rows < 0 || rows > LM_MX_MAX_ROWS - 1024 || groups < 1 || groups > LM_MX_MAX_GROUPS || n < 0 || n > (INT32_MAX - 1024) / groups || k < 1 ||
        k > LM_MX_MAX_COLS || out_stride < n || (groups > 1 && offsets == nullptr))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_matmul: a size out of range, or groups without offsets");
    if (rows == 0 || n == 0) return LM_OK;
    if (out == nullptr || !aligned(out, elem_size(out_dtype)) || !aligned(offsets, 4) || x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr ||
        !aligned(x, 32) || !aligned(x_scales, 16) || !aligned(w, 32) || !aligned(w_scales, 16))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_matmul: a null pointer, or data not 32-byte or scales not 16-byte aligned");
    // The tile's width: the average rows of a group, so that a group is one tile where that is cheap.
    const int64_t each = (rows + groups - 1) / groups;
    const int bn = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
    const int64_t m_blocks = (n + kBlockM - 1) / kBlockM;
    const int64_t column_tiles = (rows + bn - 1) / bn + std::min<int64_t>(groups, rows) - 1;  // at most
    if (column_tiles * m_blocks > INT32_MAX - kSms) return context_free_fail(LM_ERR_UNSUPPORTED, "lm_mx_matmul: more than 2^31 tiles");
    Args a{};
    a.x_scales = x_scales;
    a.w_scales = w_scales;
    a.offsets = offsets;
    a.out = out;
    a.out_stride = out_stride;
    a.scale_pitch = mx_scale_pitch(k);
    a.w_rows = groups * n;
    a.rows = static_cast<int>(rows);
    a.groups = groups;
    a.n = static_cast<int>(n);
    a.k_stages = static_cast<int>(mx_padded_cols(k) / kStageCols);
    a.x_four_bit = x_format == LM_MX_E2M1;
    a.out_dtype = out_dtype;
    void* status = nullptr;
    if (const cudaError_t e = cudaGetSymbolAddress(&status, g_status); e != cudaSuccess) return context_free_finish(e);
    a.status = static_cast<int*>(status);
    const int64_t cols = mx_padded_cols(k);
    CUtensorMap map_w;
    std::string error;
    if (!encode_tensor_map_mx(&map_w, w, true, static_cast<uint64_t>(a.w_rows), static_cast<uint64_t>(cols), kBlockM, error))
        return context_free_fail(LM_ERR_CUDA, error.c_str());
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t tiles = column_tiles * m_blocks;
    switch (bn) {
        case 16: return launch<16>(map_w, x, rows, cols, a, tiles, s);
        case 32: return launch<32>(map_w, x, rows, cols, a, tiles, s);
        case 64: return launch<64>(map_w, x, rows, cols, a, tiles, s);
        default: return launch<128>(map_w, x, rows, cols, a, tiles, s);
    }
}

lm_status lm_mx_sync(void* stream) {
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int code = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&code, g_status, sizeof code, 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return context_free_finish(e);
    if (code == 0) return LM_OK;
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_status, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return context_free_finish(e);
    return context_free_fail(LM_ERR_DEVICE_TIMEOUT, "lm_mx_sync: a product gave up waiting; its results are invalid");
}

}  // extern "C"
