// mx_matmul.cu -- grouped products of microscaled (MX) matrices (lm_mx_matmul) on the block-scaled
// tcgen05 tensor cores.
//
//   D[128 rows of W_g, BN rows of X] = W_g X^T,   out[r, n] = D[n, r]
//
// The weights are the MMA's M side, so that a few rows of X cost a narrow N instead of a padded M.
// One persistent CTA an SM walks the tiles (group, BN rows of X, 128 rows of W).  Its warps:
//   0      TMA producer: a ring of stages of 256 columns.  4-bit codes travel packed (half a byte a
//          column from HBM and L2) and are spread by the TMA into the MMA's padded form.
//   1      MMA issuer: eight block-scaled MMAs of 32 columns a stage
//   2      scale producer: 32 bytes of each row, the scales of 1024 columns, to shared memory by TMA,
//          up to three such chunks ahead
//   4-7    scales from shared memory to TMEM, each warp to its own quadrant
//   8-11   epilogue: TMEM to registers to out, rounded once; double buffered against the MMA
// A stage costs the issuer about 400 cycles of waits, descriptors and commits whatever its width,
// and four MMAs take 200 (N = 16) to 256 (N = 128): hence eight of them a stage.
// Every wait is bounded (ptx.cuh): a pipeline that stalls records a status for lm_ops_sync.
#include "moe_internal.h"
#include "mx_block.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace lm {
namespace {

constexpr int kBlockM = 128;
constexpr int kBoxCols = 128;       // columns of a TMA box: one 128-byte row of the swizzled tiles
constexpr int kStageBoxes = 2;
constexpr int kChunkBoxes = 8;      // a chunk of scales: 32 bytes a row
constexpr int kChunkBytes = 32;
constexpr int kChunks = 3;
constexpr int kThreads = 384;
constexpr int kSms = 148;
constexpr int kABoxBytes = kBlockM * kBoxCols;

template <int BN>
struct Cfg {
    static constexpr int kBBoxBytes = BN * kBoxCols;
    static constexpr int kStageBytes = kStageBoxes * (kABoxBytes + kBBoxBytes);
    static constexpr int kScaleBytes = (kBlockM + BN) * kChunkBytes;
    static constexpr int kFit = (216 * 1024 - kChunks * kScaleBytes) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kChunks * kScaleBytes;
    static constexpr int kSfCols = kChunkBoxes * (4 + 4);  // TMEM columns of a chunk: per box 4 of W's scales, 4 of X's
    static constexpr int kSfGroups = (512 - 2 * BN) / kSfCols;
    static_assert(BN % 16 == 0 && BN >= 16 && BN <= 128, "N of an M = 128 MMA, two accumulators");
    static_assert(kStages >= 3 && kSfGroups >= 2, "rings");
};

struct Args {
    const int32_t* offsets;  // or null: one group of all rows
    void* out;
    int64_t out_stride;
    int rows, groups, n;
    int k_boxes;
    int x_four_bit;
    int out_dtype;
    int* status;
};

__device__ int g_status;  // the first device-side error since the last lm_ops_sync

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
    mx_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_xs, const Args a) {
    using C = Cfg<BN>;
    constexpr int S = C::kStages, G = C::kSfGroups;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int s_cut[LM_MX_MAX_GROUPS + 1], s_tiles[LM_MX_MAX_GROUPS + 1];
    __shared__ uint64_t full[S], empty[S], chunk_full[kChunks], chunk_empty[kChunks], sf_full[G], sf_empty[G], tmem_full[2], tmem_empty[2], drain;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t* smem_a = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_b = smem_a + S * kStageBoxes * kABoxBytes;
    uint8_t* smem_s = smem_b + S * kStageBoxes * C::kBBoxBytes;  // chunks: 128 rows of W's scales, then BN of X's
    volatile int* abort_flag = &s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_ws);
        tma_prefetch_desc(&map_xs);
        for (int i = 0; i < S; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < kChunks; ++i) mbar_init(&chunk_full[i], 1), mbar_init(&chunk_empty[i], 4);
        for (int i = 0; i < G; ++i) mbar_init(&sf_full[i], 4), mbar_init(&sf_empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&tmem_full[i], 1), mbar_init(&tmem_empty[i], 4);
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
    const uint32_t tmem_sf = tmem + 2 * BN;
    const int m_blocks = (a.n + kBlockM - 1) / kBlockM;
    const int total = s_tiles[a.groups] * m_blocks;

    // In the issuing warps all lanes walk the loop and an elected one issues, so that descriptors and
    // addresses stay in uniform registers (under `if (lane == 0)` a stage took twice as long).
    if (warp == 0) {
        const uint32_t box_bytes = kABoxBytes / 2 + (a.x_four_bit ? C::kBBoxBytes / 2 : C::kBBoxBytes);
        int stage = 0;
        uint32_t phase = 0, issued = 0, issued_phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
            const Tile tile = tile_at<BN>(a, s_cut, s_tiles, t, m_blocks);
            const int w_row = tile.group * a.n + tile.n0;
            for (int b = 0; b < a.k_boxes; b += kStageBoxes) {
                ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, abort_flag, a.status, kDevTimeoutProducer));
                if (!ok) break;
                if (elect_one()) {
                    const int boxes = min(kStageBoxes, a.k_boxes - b);
                    mbar_arrive_expect_tx(&full[stage], boxes * box_bytes);
                    for (int i = 0; i < boxes; ++i) {
                        tma_load_2d(smem_a + (stage * kStageBoxes + i) * kABoxBytes, &map_w, &full[stage], (b + i) * kBoxCols, w_row);
                        tma_load_2d(smem_b + (stage * kStageBoxes + i) * C::kBBoxBytes, &map_x, &full[stage], (b + i) * kBoxCols, tile.row0);
                    }
                }
                __syncwarp();
                issued |= 1u << stage;
                issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == S) stage = 0, phase ^= 1u;
            }
        }
        if (!ok)  // copies in flight land before the CTA's shared memory is given up
            for (int i = 0; i < S; ++i)
                if (issued & (1u << i)) mbar_wait_drain(&full[i], (issued_phase >> i) & 1u, 100000000ull);
    } else if (warp == 1) {
        int stage = 0, sg = 0, acc = 0;
        uint32_t phase = 0, sf_phase = 0, acc_phase = 0;
        bool ok = true, any = false, seen = false;
        const uint32_t format = (a.x_four_bit ? kUmmaE2M1 : kUmmaE4M3) << 10;
        const uint64_t desc_a = umma_desc_sw128(smem_u32(smem_a)), desc_b = umma_desc_sw128(smem_u32(smem_b));
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
            ok = __all_sync(0xffffffffu, mbar_wait(&tmem_empty[acc], acc_phase ^ 1u, abort_flag, a.status, kDevTimeoutMma));
            const uint32_t d = tmem + acc * BN;
            for (int b = 0; ok && b < a.k_boxes; b += kStageBoxes) {
                if (b % kChunkBoxes == 0) ok = mbar_wait(&sf_full[sg], sf_phase, abort_flag, a.status, kDevTimeoutMma);
                if (!seen) ok = ok && mbar_wait(&full[stage], phase, abort_flag, a.status, kDevTimeoutMma);
                if (b % kChunkBoxes == 0 || !seen) ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const int next = stage + 1 == S ? 0 : stage + 1;
                // A look at the next stage while the tensor cores still work: even the wait for a
                // complete barrier costs as much as an MMA.
                const bool look = mbar_test(&full[next], phase ^ (next == 0));
                const bool last = b + kStageBoxes >= a.k_boxes;
                const bool sf_end = last || (b + kStageBoxes) % kChunkBoxes == 0;
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < kStageBoxes; ++i) {
                        if (b + i < a.k_boxes) {
                            const uint64_t da = desc_a + static_cast<uint32_t>((stage * kStageBoxes + i) * (kABoxBytes >> 4));
                            const uint64_t db = desc_b + static_cast<uint32_t>((stage * kStageBoxes + i) * (C::kBBoxBytes >> 4));
                            const uint32_t sf = tmem_sf + sg * C::kSfCols + (b % kChunkBoxes + i) * 8;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)  // 32 columns are 32 bytes, 2 in the descriptor's units
                                umma_mx(d, da + 2 * kk, db + 2 * kk, umma_idesc_mx(kUmmaE2M1, 0, kBlockM, BN, kk) | format, sf, sf + 4,
                                        b != 0 || i != 0 || kk != 0);
                        }
                    }
                    umma_commit(&empty[stage]);
                    if (sf_end) umma_commit(&sf_empty[sg]);
                    if (last) umma_commit(&tmem_full[acc]);
                }
                __syncwarp();
                any = true;
                seen = __all_sync(0xffffffffu, look);
                phase ^= next == 0, stage = next;
                if (sf_end && ++sg == G) sg = 0, sf_phase ^= 1u;
            }
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
        if (!ok && any) {  // the MMAs issued so far end before TMEM is released
            if (elect_one()) umma_commit(&drain);
            __syncwarp();
            mbar_wait_drain(&drain, 0, 100000000ull);
        }
    } else if (warp == 2) {
        int chunk = 0;
        uint32_t phase = 0, issued = 0, issued_phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
            const Tile tile = tile_at<BN>(a, s_cut, s_tiles, t, m_blocks);
            for (int b = 0; b < a.k_boxes; b += kChunkBoxes) {
                ok = __all_sync(0xffffffffu, mbar_wait(&chunk_empty[chunk], phase ^ 1u, abort_flag, a.status, kDevTimeoutProducer));
                if (!ok) break;
                if (elect_one()) {
                    uint8_t* dst = smem_s + chunk * C::kScaleBytes;
                    mbar_arrive_expect_tx(&chunk_full[chunk], C::kScaleBytes);
                    tma_load_2d(dst, &map_ws, &chunk_full[chunk], b / kChunkBoxes * kChunkBytes, tile.group * a.n + tile.n0);
                    tma_load_2d(dst + kBlockM * kChunkBytes, &map_xs, &chunk_full[chunk], b / kChunkBoxes * kChunkBytes, tile.row0);
                }
                __syncwarp();
                issued |= 1u << chunk;
                issued_phase = (issued_phase & ~(1u << chunk)) | (phase << chunk);
                if (++chunk == kChunks) chunk = 0, phase ^= 1u;
            }
        }
        if (!ok)
            for (int i = 0; i < kChunks; ++i)
                if (issued & (1u << i)) mbar_wait_drain(&chunk_full[i], (issued_phase >> i) & 1u, 100000000ull);
    } else if (warp >= 4 && warp < 8) {
        const uint32_t quad = static_cast<uint32_t>(warp & 3) * 32u << 16;
        constexpr int kXRows = (BN + 31) / 32;
        int sg = 0, chunk = 0;
        uint32_t phase = 0, chunk_phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
            for (int b = 0; ok && b < a.k_boxes; b += kChunkBoxes) {
                // Every lane waits for what it reads; a lane that gave up takes its warp along.
                ok = mbar_wait(&chunk_full[chunk], chunk_phase, abort_flag, a.status, kDevTimeoutProducer);
                ok = ok && mbar_wait(&sf_empty[sg], phase ^ 1u, abort_flag, a.status, kDevTimeoutProducer);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint8_t* src = smem_s + chunk * C::kScaleBytes + lane * kChunkBytes;
#pragma unroll
                for (int h = 0; h < 4; ++h) {  // 8 bytes of a row are the scales of two boxes: 16 columns of TMEM
                    uint32_t r[16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint2 w = *reinterpret_cast<const uint2*>(src + 32 * c * kChunkBytes + 8 * h);
                        uint2 x = make_uint2(0u, 0u);
                        if (c < kXRows && (BN >= 32 || lane < BN)) x = *reinterpret_cast<const uint2*>(src + (kBlockM + 32 * c) * kChunkBytes + 8 * h);
                        r[c] = w.x, r[8 + c] = w.y, r[4 + c] = x.x, r[12 + c] = x.y;
                    }
                    tmem_st16(tmem_sf + quad + sg * C::kSfCols + 16 * h, r);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sf_full[sg]);
                    mbar_arrive(&chunk_empty[chunk]);
                }
                if (++sg == G) sg = 0, phase ^= 1u;
                if (++chunk == kChunks) chunk = 0, chunk_phase ^= 1u;
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
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

struct Matrix {
    const uint8_t* codes;
    const uint8_t* scales;
    bool four_bit;
    int64_t rows;
};

template <int BN>
lm_status launch(const Matrix& w, const Matrix& x, int64_t k, const Args& a, int64_t tiles, cudaStream_t stream) {
    using C = Cfg<BN>;
    CUtensorMap map_w, map_x, map_ws, map_xs;
    std::string error;
    const uint64_t cols = static_cast<uint64_t>(mx_padded_cols(k)), pitch = static_cast<uint64_t>(mx_scale_pitch(k));
    const auto encode = [&](const Matrix& m, uint32_t box, CUtensorMap* codes, CUtensorMap* scales) {
        return encode_tensor_map_mx(codes, m.codes, m.four_bit, static_cast<uint64_t>(m.rows), cols, box, error) &&
               encode_tensor_map_mx_scales(scales, m.scales, static_cast<uint64_t>(m.rows), pitch, box, kChunkBytes, error);
    };
    if (!encode(w, kBlockM, &map_w, &map_ws) || !encode(x, BN, &map_x, &map_xs)) return context_free_fail(LM_ERR_CUDA, error.c_str());
    if (const cudaError_t e = cudaFuncSetAttribute(mx_matmul_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes); e != cudaSuccess)
        return context_free_finish(e);
    mx_matmul_kernel<BN><<<static_cast<unsigned>(std::min<int64_t>(tiles, kSms)), kThreads, C::kSmemBytes, stream>>>(map_w, map_x, map_ws, map_xs,
                                                                                                                          a);
    return context_free_finish(cudaGetLastError());
}

}  // namespace

cudaError_t ops_status(int** status) {
    void* p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, g_status);
    *status = static_cast<int*>(p);
    return e;
}

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
    // The tile's width: groups are ragged, so half as much again as the average rows of a group keeps
    // most of them in one tile (a second tile reads the group's weights again).
    const int64_t each = (rows + groups - 1) / groups;
    const int bn = each <= 10 ? 16 : each <= 20 ? 32 : each <= 40 ? 64 : 128;
    const int64_t m_blocks = (n + kBlockM - 1) / kBlockM;
    const int64_t column_tiles = (rows + bn - 1) / bn + std::min<int64_t>(groups, rows) - 1;  // at most
    if (column_tiles * m_blocks > INT32_MAX - kSms) return context_free_fail(LM_ERR_UNSUPPORTED, "lm_mx_matmul: more than 2^31 tiles");
    Args a{};
    a.offsets = offsets;
    a.out = out;
    a.out_stride = out_stride;
    a.rows = static_cast<int>(rows);
    a.groups = groups;
    a.n = static_cast<int>(n);
    a.k_boxes = static_cast<int>(mx_padded_cols(k) / kBoxCols);
    a.x_four_bit = x_format == LM_MX_E2M1;
    a.out_dtype = out_dtype;
    if (const cudaError_t e = ops_status(&a.status); e != cudaSuccess) return context_free_finish(e);
    const Matrix mw{w, w_scales, true, groups * n}, mx{x, x_scales, x_format == LM_MX_E2M1, rows};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t tiles = column_tiles * m_blocks;
    switch (bn) {
        case 16: return launch<16>(mw, mx, k, a, tiles, s);
        case 32: return launch<32>(mw, mx, k, a, tiles, s);
        case 64: return launch<64>(mw, mx, k, a, tiles, s);
        default: return launch<128>(mw, mx, k, a, tiles, s);
    }
}

lm_status lm_ops_sync(void* stream) {
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
    return context_free_fail(LM_ERR_DEVICE_TIMEOUT, "lm_ops_sync: a kernel gave up waiting; its results are invalid");
}

}  // extern "C"
