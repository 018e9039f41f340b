// mx_matmul.cu -- grouped products of microscaled (MX) matrices (lm_mx_matmul) on the block-scaled
// tcgen05 tensor cores.
//
//   D[128 rows of W_g, BN rows of X] = W_g X^T,   out[r, n] = D[n, r]
//
// The weights are the MMA's M side, so that a few rows of X cost a narrow N instead of a padded M.
// One persistent CTA an SM walks the tiles (group, BN rows of X, 128 rows of W); for many rows a
// group, pairs of CTAs walk tiles of 256 rows of W by 128 of X together, each bringing its half of
// both operands (at the full rate of the MMA a CTA of its own asks the L2 for 92 bytes a cycle and one
// of a pair for 62; a prompt's 24576 rows move 54 an SM and cycle, the dense shape below 42).
// E4M3 rows of X take kind::mxf8f6f4, whose 4-bit operand is padded to a byte a code: W's codes
// travel packed and the TMA spreads them in shared memory.  E2M1 rows take kind::mxf4 with both
// operands packed, half the shared memory and half the MMAs (dense 4096 x 10944 x 2048: 53 us, 84
// to 91 with E4M3 rows, by the clock).
// A CTA's warps:
//   0      TMA producer: a ring of stages of two boxes of 128 bytes a row
//   1      MMA issuer (of the pair's first CTA): four block-scaled MMAs a box
//   2      scale producer: the scales of a chunk of boxes, to shared memory by TMA, ahead of the codes
//   4-7    scales from shared memory to TMEM, each warp to its own quadrant
//   8-15   epilogue: TMEM to registers to out, rounded once; two warps a quadrant share the rows of X
// A stage costs the issuer about 400 cycles of waits, descriptors and commits whatever its width,
// and the four MMAs of a box take 200 (N = 16) to 256 (N = 128): hence two boxes a stage.
// Every wait is bounded (ptx.cuh): a pipeline that stalls records a status for lm_ops_sync.  Once all
// warps have stopped, each waits for what it left in flight (copies, MMAs) before shared memory and
// TMEM are given up; a pair does so together, since the second CTA's copies end on the first's barriers.
#include "moe_internal.h"
#include "mx_block.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <utility>

namespace lm {
namespace {

constexpr int kBlockM = 128;
constexpr int kThreads = 512;
constexpr int kSms = 148;
constexpr int kMaxSplit = 4;
constexpr int kBoxRow = 128;  // bytes of a row of a TMA box in shared memory: one swizzled row
constexpr int kABoxBytes = kBlockM * kBoxRow;

template <int BN, bool PAIR, bool FOUR>
struct Cfg {
    static constexpr int kCtas = PAIR ? 2 : 1;
    static constexpr int kBRows = BN / kCtas;  // rows of X that a CTA brings
    static constexpr int kBoxCols = FOUR ? 256 : 128;  // both operands packed, or 8 bits a column in shared memory
    static constexpr int kBBoxBytes = kBRows * kBoxRow;
    static constexpr int kStageBoxes = 2;
    static constexpr int kStageBytes = kStageBoxes * (kABoxBytes + kBBoxBytes);
    // A chunk of scales: 1024 columns, 32 bytes a row, a word for each 128 columns (TMEM: 4 columns of
    // W's words, 4 of X's).  What the two accumulators leave of TMEM holds four chunks or more.
    static constexpr int kChunkBytes = 32, kChunkWords = kChunkBytes / 4, kBoxWords = kBoxCols / 128;
    static constexpr int kChunkBoxes = kChunkWords / kBoxWords, kChunks = 3;
    static constexpr int kSfCols = kChunkWords * 8, kSfGroups = 4;
    static constexpr int kScaleBytes = (kBlockM + BN) * kChunkBytes;
    static constexpr int kStagesFit = (216 * 1024 - kChunks * kScaleBytes) / kStageBytes;
    static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kChunks * kScaleBytes;
    static_assert(BN % 16 == 0 && BN >= 16 && 2 * BN + kSfGroups * kSfCols <= 512 && (!PAIR || BN % 32 == 0), "N of the MMA");
    static_assert(kBBoxBytes % 1024 == 0 || !PAIR, "swizzled tiles start on 1024 bytes");
    // Stages of one round of the issuer: two where a box's MMAs are short and the ring is long.
    static constexpr int kRound = kStages >= 5 && !FOUR ? 2 : 1;
    static_assert(kStages >= 3 && kChunkBoxes % (kRound * kStageBoxes) == 0, "rings");
};

struct Args {
    const int32_t* offsets;  // or null: one group of all rows
    void* out;
    int64_t out_stride;
    int rows, groups, n;
    int x_box, xs_box;  // rows of X and of its scales of a TMA box
    int k_boxes;
    int split;  // CTAs (a cluster) that share a tile's boxes; more than 1: a cluster has one tile
    int out_dtype;
    int out_pairs;  // 16-bit elements n, n + 1 (n even) lie on 4-byte boundaries
    int stall;      // testing only: a LM_STALL_* barrier that expects one arrival more than it gets
    uint64_t wait_limit_ns;
    int* status;
};

__device__ int g_status;       // the first device-side error of the process: which wait ran out
__device__ unsigned g_stalls;  // CTAs that gave up so far; never cleared

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
    int n0;                 // first row of W_g for this CTA
};

template <int BN, bool PAIR, bool FOUR>
__device__ __forceinline__ Tile tile_at(const Args& a, const int* cut, const int* tiles, int t, int m_blocks, int rank) {
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
    r.n0 = (t - ct * m_blocks) * kBlockM * Cfg<BN, PAIR, FOUR>::kCtas + rank * kBlockM;
    return r;
}

// The MMA's N for a tile of `rows` rows of X: no wider than they need.
template <bool PAIR>
__device__ __forceinline__ int mma_n(int rows) {
    return PAIR ? (rows + 31) & ~31 : (rows + 15) & ~15;
}

// Columns v[0 .. 31] of the accumulator (this lane's n) to rows of out from `p` on, `rows` of them.
// 16-bit types: neighbouring lanes swap values, and each stores two n of every second row.
template <int DT>
__device__ __forceinline__ void store_columns(typename Elem<DT>::T* p, int64_t stride, int rows, bool n_ok, bool pairs, const uint32_t (&v)[32]) {
    if constexpr (DT != LM_DTYPE_F32) {
        if (pairs) {
            const int odd = threadIdx.x & 1;
            uint32_t* q = reinterpret_cast<uint32_t*>(p - odd + odd * stride);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
                const typename Elem<DT>::T e[2] = {Elem<DT>::narrow(__uint_as_float(odd ? got : v[j])), Elem<DT>::narrow(__uint_as_float(odd ? v[j + 1] : got))};
                uint32_t w;
                memcpy(&w, e, 4);
                if (j + odd < rows) *q = w;
                q += stride;  // two rows of 16-bit elements
            }
            return;
        }
    }
    if (!n_ok) return;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        if (j < rows) *p = Elem<DT>::narrow(__uint_as_float(v[j]));
        p += stride;
    }
}

template <int BN, bool PAIR, bool FOUR>
__global__ void __launch_bounds__(kThreads, 1)
    mx_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_xs, const Args a) {
    using C = Cfg<BN, PAIR, FOUR>;
    constexpr int S = C::kStages, G = C::kSfGroups, B = C::kStageBoxes;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int s_cut[LM_MX_MAX_GROUPS + 1], s_tiles[LM_MX_MAX_GROUPS + 1];
    // In a pair `full`, `sf_full` and `tmem_empty` are the first CTA's, whose warp 1 issues the MMAs;
    // the MMAs' commits arrive in both CTAs.
    __shared__ uint64_t full[S], empty[S], chunk_full[C::kChunks], chunk_empty[C::kChunks], sf_full[G], sf_empty[G], tmem_full[2], tmem_empty[2], drain;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ uint32_t s_peer_gave_up, s_peer_sent;  // written by the pair's other CTA
    uint8_t* smem_a = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_b = smem_a + S * B * kABoxBytes;
    uint8_t* smem_s = smem_b + S * B * C::kBBoxBytes;  // chunks: 128 rows of W's scales, then BN of X's
    float* partial = reinterpret_cast<float*>(smem_a);  // with a split: the ring is idle when its only tile is done
    volatile int* abort_flag = &s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
    const int split = PAIR ? 1 : a.split, part = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int ctas = C::kCtas * split, first = blockIdx.x / ctas, step = gridDim.x / ctas;
    // This CTA's boxes, from a multiple of 16 bytes of scales on.
    constexpr int kUnit = 4 / C::kBoxWords;
    const int units = (a.k_boxes + kUnit - 1) / kUnit, box0 = units * part / split * kUnit, boxes = min(a.k_boxes, units * (part + 1) / split * kUnit) - box0;

    const auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        return mbar_wait(bar, parity, abort_flag, a.status, code, a.wait_limit_ns);
    };
    const auto wait_both = [&](uint64_t* bar, uint32_t parity, int code) {  // on a barrier that both CTAs of a pair arrive on
        return mbar_wait<PAIR>(bar, parity, abort_flag, a.status, code, a.wait_limit_ns);
    };
    const auto commit = [&](uint64_t* bar) {
        if constexpr (PAIR) umma_commit_both(bar);
        else umma_commit(bar);
    };
    const auto arrive_first = [&](uint64_t* bar) {  // on the first CTA's barrier
        if constexpr (PAIR) mbar_arrive_cluster_tmem(mapa_shared(smem_u32(bar), 0));
        else mbar_arrive(bar);
    };

    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_ws);
        tma_prefetch_desc(&map_xs);
        const auto init = [&](uint64_t* bars, int count, uint32_t arrivals, int stall) {
            for (int i = 0; i < count; ++i) mbar_init(&bars[i], arrivals + (a.stall == stall));
        };
        init(full, S, 1, LM_STALL_FULL), init(empty, S, 1, LM_STALL_EMPTY);
        init(chunk_full, C::kChunks, 1, LM_STALL_CHUNK_FULL), init(chunk_empty, C::kChunks, 4, LM_STALL_CHUNK_EMPTY);
        init(sf_full, G, 4 * C::kCtas, LM_STALL_SCALE_FULL), init(sf_empty, G, 1, LM_STALL_SCALE_EMPTY);
        init(tmem_full, 2, 1, LM_STALL_TMEM_FULL), init(tmem_empty, 2, 8 * C::kCtas, LM_STALL_TMEM_EMPTY);
        mbar_init(&drain, 1);
        s_abort = 0, s_peer_gave_up = 0, s_peer_sent = 0;
        fence_mbar_init();
    }
    __syncwarp();
    if constexpr (PAIR) cluster_sync();  // both CTAs' barriers exist before either signals the other's
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(&s_tmem, 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(&s_tmem, 512);
            tmem_relinquish();
        }
    }
    if (warp == 2) cut_groups<BN>(a, s_cut, s_tiles);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t tmem_sf = tmem + 2 * BN;
    const int m_blocks = (a.n + kBlockM * C::kCtas - 1) / (kBlockM * C::kCtas);
    const int total = s_tiles[a.groups] * m_blocks;

    const uint32_t box_bytes = (FOUR ? kABoxBytes : kABoxBytes / 2) + a.x_box * kBoxRow;  // spread codes count packed
    // What a thread may leave in flight: stages sent (warp 0), chunks sent (warp 2), MMAs (the issuing lane).
    uint32_t sent = 0;
    bool mmas = false;

    // An elected lane issues, so that descriptors and addresses stay in uniform registers (under
    // `if (lane == 0)` a stage took twice as long).
    if (warp == 0) {
        constexpr int kColStep = FOUR ? kBoxRow : C::kBoxCols;  // a box in the map's elements: bytes when packed
        // Narrow tiles are for groups of few rows, whose weights are read once: they leave L2 first
        // (128 tokens over 64 experts: 43.8 -> 41.8 us; with 128 rows a tile it cost 7%).
        const uint64_t once = policy_evict_first();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first; ok && t < total; t += step) {
            const Tile tile = tile_at<BN, PAIR, FOUR>(a, s_cut, s_tiles, t, m_blocks, rank);
            const int w_row = tile.group * a.n + tile.n0;
            const int x_row = tile.row0 + rank * mma_n<PAIR>(tile.rows) / 2;
            for (int b = 0; b < boxes; b += B) {
                ok = __all_sync(0xffffffffu, wait(&empty[stage], phase ^ 1u, kDevTimeoutProducer));
                if (!ok) break;
                if (elect_one()) {
                    const int n_boxes = min(B, boxes - b);
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], C::kCtas * n_boxes * box_bytes);
                    for (int i = 0; i < n_boxes; ++i) {
                        uint8_t *da = smem_a + (stage * B + i) * kABoxBytes, *db = smem_b + (stage * B + i) * C::kBBoxBytes;
                        if constexpr (PAIR) {
                            const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
                            tma_load_2d_pair(da, &map_w, bar, (box0 + b + i) * kColStep, w_row);
                            tma_load_2d_pair(db, &map_x, bar, (box0 + b + i) * kColStep, x_row);
                        } else {
                            if constexpr (BN <= 64) tma_load_2d_hint(da, &map_w, &full[stage], (box0 + b + i) * kColStep, w_row, once);
                            else tma_load_2d(da, &map_w, &full[stage], (box0 + b + i) * kColStep, w_row);
                            tma_load_2d(db, &map_x, &full[stage], (box0 + b + i) * kColStep, x_row);
                        }
                    }
                }
                __syncwarp();
                ++sent;
                if (++stage == S) stage = 0, phase ^= 1u;
            }
        }
    } else if (warp == 1 && rank == 0) {
        // One lane does all of it: the votes and elections of a whole warp cost more than they order
        // (64 experts of 12 rows: 40.1 us, one lane 39.2; 384 rows a group 173 and 162).
        if (elect_one()) {
            int stage = 0, sg = 0, acc = 0;
            uint32_t phase = 0, sf_phase = 0, acc_phase = 0;
            bool ok = true, seen = false, sf_seen = false;
            const uint64_t desc_a = umma_desc_sw128(smem_u32(smem_a)), desc_b = umma_desc_sw128(smem_u32(smem_b));
            constexpr int U = C::kRound;
            const auto after = [](int st, int by) { return st + by >= S ? st + by - S : st + by; };
            for (int t = first; ok && t < total; t += step) {
                int width = BN;  // a pair's MMAs are no wider than the tile's rows need; one CTA's take 50 cycles at least
                if constexpr (PAIR) width = mma_n<PAIR>(tile_at<BN, PAIR, FOUR>(a, s_cut, s_tiles, t, m_blocks, rank).rows);
                const uint32_t shape = static_cast<uint32_t>(width >> 3) << 17;
                ok = wait_both(&tmem_empty[acc], acc_phase ^ 1u, kDevTimeoutMma);
                const uint32_t d = tmem + acc * BN;
                for (int b = 0; ok && b < boxes; b += U * B) {
                    const int stages = min(U, (boxes - b + B - 1) / B);
                    const bool sf_begin = b % C::kChunkBoxes == 0;
                    if ((sf_begin && !sf_seen) || !seen) {
                        ok = !sf_begin || sf_seen || wait_both(&sf_full[sg], sf_phase, kDevTimeoutMma);
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (u < stages) ok = ok && wait(&full[after(stage, u)], phase ^ (stage + u >= S), kDevTimeoutMma);
                        if (!ok) break;
                    }
                    tc_fence_after();
                    const bool last = b + stages * B >= boxes;
                    const bool sf_end = last || (b + stages * B) % C::kChunkBoxes == 0;
                    const int next = after(stage, stages), sg_next = sg + 1 == G ? 0 : sg + 1;
                    const uint32_t next_phase = phase ^ (stage + stages >= S);
                    // A look at the next round while the tensor cores still work: even the wait for a
                    // complete barrier costs as much as an MMA.
                    bool look = true;
#pragma unroll
                    for (int u = 0; u < U; ++u) look = look && mbar_test(&full[after(next, u)], next_phase ^ (next + u >= S));
                    const bool sf_look = sf_end && mbar_test<PAIR>(&sf_full[sg_next], sf_phase ^ (sg_next == 0));
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (u >= stages) break;
                        const int st = after(stage, u);
#pragma unroll
                        for (int i = 0; i < B; ++i) {
                            const int box = u * B + i;
                            if (b + box < boxes) {
                                const uint64_t da = desc_a + static_cast<uint32_t>((st * B + i) * (kABoxBytes >> 4));
                                const uint64_t db = desc_b + static_cast<uint32_t>((st * B + i) * (C::kBBoxBytes >> 4));
                                const uint32_t sf = tmem_sf + sg * C::kSfCols + (b % C::kChunkBoxes + box) * C::kBoxWords * 8;
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk) {  // 32 or 64 columns: 32 bytes, 2 in the descriptors' units
                                    constexpr uint32_t kA = FOUR ? kUmmaPackedE2M1 : kUmmaE2M1, kB = FOUR ? kUmmaPackedE2M1 : kUmmaE4M3;
                                    const uint32_t idesc = umma_idesc_mx(kA, kB, kBlockM * C::kCtas, 0, FOUR ? kk % 2 * 2 : kk) | shape;
                                    const uint32_t word = sf + (FOUR ? kk / 2 * 8 : 0);
                                    umma_mx<PAIR, FOUR>(d, da + 2 * kk, db + 2 * kk, idesc, word, word + 4, b != 0 || box != 0 || kk != 0);
                                }
                            }
                        }
                        commit(&empty[st]);
                    }
                    if (sf_end) commit(&sf_empty[sg]);
                    if (last) commit(&tmem_full[acc]);
                    mmas = true;
                    seen = look;
                    phase = next_phase, stage = next;
                    if (sf_end) sf_seen = sf_look, sf_phase ^= sg_next == 0, sg = sg_next;
                }
                if (++acc == 2) acc = 0, acc_phase ^= 1u;
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        int chunk = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first; ok && t < total; t += step) {
            const Tile tile = tile_at<BN, PAIR, FOUR>(a, s_cut, s_tiles, t, m_blocks, rank);
            for (int b = 0; b < boxes; b += C::kChunkBoxes) {
                ok = __all_sync(0xffffffffu, wait(&chunk_empty[chunk], phase ^ 1u, kDevTimeoutProducer));
                if (!ok) break;
                if (elect_one()) {
                    uint8_t* dst = smem_s + chunk * C::kScaleBytes;
                    mbar_arrive_expect_tx(&chunk_full[chunk], (kBlockM + a.xs_box) * C::kChunkBytes);
                    tma_load_2d(dst, &map_ws, &chunk_full[chunk], (box0 + b) * C::kBoxWords * 4, tile.group * a.n + tile.n0);
                    tma_load_2d(dst + kBlockM * C::kChunkBytes, &map_xs, &chunk_full[chunk], (box0 + b) * C::kBoxWords * 4, tile.row0);
                }
                __syncwarp();
                ++sent;
                if (++chunk == C::kChunks) chunk = 0, phase ^= 1u;
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const uint32_t quad = static_cast<uint32_t>(warp & 3) * 32u << 16;
        constexpr int kXRows = (BN + 31) / 32;
        int sg = 0, chunk = 0;
        uint32_t phase = 0, chunk_phase = 0;
        bool ok = true;
        for (int t = first; ok && t < total; t += step) {
            for (int b = 0; b < boxes; b += C::kChunkBoxes) {
                // Every lane waits for what it reads; a lane that gave up takes its warp along.
                ok = wait(&chunk_full[chunk], chunk_phase, kDevTimeoutProducer);
                ok = __all_sync(0xffffffffu, ok && wait(&sf_empty[sg], phase ^ 1u, kDevTimeoutProducer));
                if (!ok) break;
                tc_fence_after();
                // 16 bytes of a row, its scales of 512 columns, at a time; the TMA's 32-byte swizzle swaps
                // the halves of every second four rows, so that eight lanes reach all banks (with plain
                // rows a chunk took 900 to 2000 cycles, the longest step of most products).
                const uint8_t* src = smem_s + chunk * C::kScaleBytes + lane * C::kChunkBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t* at = src + 16 * (h ^ (lane >> 2 & 1));
                    uint4 w[4], x[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        w[c] = *reinterpret_cast<const uint4*>(at + 32 * c * C::kChunkBytes);
                        x[c] = make_uint4(0u, 0u, 0u, 0u);
                        if (c < kXRows && (BN >= 32 || lane < BN)) x[c] = *reinterpret_cast<const uint4*>(at + (kBlockM + 32 * c) * C::kChunkBytes);
                    }
                    uint32_t r[16];
                    const uint32_t to = tmem_sf + quad + sg * C::kSfCols + 32 * h;
#pragma unroll
                    for (int c = 0; c < 4; ++c) r[c] = w[c].x, r[4 + c] = x[c].x, r[8 + c] = w[c].y, r[12 + c] = x[c].y;
                    tmem_st16(to, r);
#pragma unroll
                    for (int c = 0; c < 4; ++c) r[c] = w[c].z, r[4 + c] = x[c].z, r[8 + c] = w[c].w, r[12 + c] = x[c].w;
                    tmem_st16(to + 16, r);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    arrive_first(&sf_full[sg]);
                    mbar_arrive(&chunk_empty[chunk]);
                }
                if (++sg == G) sg = 0, phase ^= 1u;
                if (++chunk == C::kChunks) chunk = 0, chunk_phase ^= 1u;
            }
        }
    } else if (warp >= 8) {
        const int quad = warp & 3, half = (warp - 8) >> 2;
        constexpr int kHalf = BN >= 64 ? BN / 2 : BN;  // a warp's rows of X; few: the first four warps take all
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = first; t < total; t += step) {
            const Tile tile = tile_at<BN, PAIR, FOUR>(a, s_cut, s_tiles, t, m_blocks, rank);
            int go = 1;
            if (lane == 0) go = wait(&tmem_full[acc], acc_phase, kDevTimeoutEpilogue);
            if (__shfl_sync(0xffffffffu, go, 0) == 0) break;
            tc_fence_after();
            const int n_warp = tile.n0 + quad * 32, n = n_warp + lane;
            const uint32_t src = tmem + acc * BN + (static_cast<uint32_t>(quad * 32) << 16);
            const bool pairs = a.out_pairs != 0 && n_warp + 32 <= a.n;
            const int c_first = half * kHalf, c_end = min(tile.rows, c_first + kHalf);
            for (int c0 = c_first; c0 < c_end; c0 += 32) {
                uint32_t v[32];
                tmem_ld16(src + c0, *reinterpret_cast<uint32_t(*)[16]>(v));
                if constexpr (kHalf >= 32) tmem_ld16(src + c0 + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
                tmem_ld_wait();
                if (split > 1) {  // this part's sums, for the cluster to add
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c0 + j < c_end) partial[(c0 + j) * kBlockM + quad * 32 + lane] = __uint_as_float(v[j]);
                    continue;
                }
                const int64_t at = (static_cast<int64_t>(tile.row0) + c0) * a.out_stride + n;
                const int rows = c_end - c0;
                if (a.out_dtype == LM_DTYPE_F32) store_columns<LM_DTYPE_F32>(static_cast<float*>(a.out) + at, a.out_stride, rows, n < a.n, pairs, v);
                else if (a.out_dtype == LM_DTYPE_BF16) store_columns<LM_DTYPE_BF16>(static_cast<__nv_bfloat16*>(a.out) + at, a.out_stride, rows, n < a.n, pairs, v);
                else store_columns<LM_DTYPE_F16>(static_cast<__half*>(a.out) + at, a.out_stride, rows, n < a.n, pairs, v);
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_first(&tmem_empty[acc]);
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
    }
    if constexpr (!PAIR) {
        if (split > 1) {
            // The parts' sums, added in the parts' order, each CTA its share of the tile's elements.
            __syncthreads();
            cluster_sync();
            if (first < total) {
                const Tile tile = tile_at<BN, PAIR, FOUR>(a, s_cut, s_tiles, first, m_blocks, rank);
                for (int i = part * kThreads + threadIdx.x; i < tile.rows * kBlockM; i += split * kThreads) {
                    float sum = 0.0f, v[kMaxSplit];
#pragma unroll
                    for (int p = 0; p < kMaxSplit; ++p)
                        if (p < split) v[p] = ld_cluster_f32(mapa_shared(smem_u32(partial + i), p));
#pragma unroll
                    for (int p = 0; p < kMaxSplit; ++p)
                        if (p < split) sum += v[p];
                    const int n = tile.n0 + i % kBlockM;
                    const int64_t at = (static_cast<int64_t>(tile.row0) + i / kBlockM) * a.out_stride + n;
                    if (n < a.n) {
                        if (a.out_dtype == LM_DTYPE_F32) static_cast<float*>(a.out)[at] = sum;
                        else if (a.out_dtype == LM_DTYPE_BF16) static_cast<__nv_bfloat16*>(a.out)[at] = Elem<LM_DTYPE_BF16>::narrow(sum);
                        else static_cast<__half*>(a.out)[at] = Elem<LM_DTYPE_F16>::narrow(sum);
                    }
                }
            }
            __syncwarp();
            cluster_sync();  // no CTA leaves while another reads its sums
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    bool gave_up = s_abort != 0;
    if constexpr (PAIR) {
        if (gave_up && threadIdx.x == 0) st_cluster_u32(mapa_shared(smem_u32(&s_peer_gave_up), rank ^ 1), 1);
        __syncwarp();
        cluster_sync();  // neither CTA leaves while the other may signal it or use its memory
        gave_up = gave_up || s_peer_gave_up != 0;
    }
    if (gave_up) {  // all warps, of both CTAs of a pair, have stopped
        if (threadIdx.x == 0) atomicAdd(&g_stalls, 1u);
        constexpr uint64_t limit = 100000000;  // 0.1 s, whatever the pipeline's own limit: copies in flight take microseconds
        // The copies of the last round of a ring; those of earlier rounds have been consumed.
        const auto land = [&](uint64_t* bars, uint32_t ring, uint32_t count) {
            for (uint32_t j = count > ring ? count - ring : 0; j < count; ++j) mbar_wait_drain(&bars[j % ring], j / ring & 1u, limit);
        };
        uint32_t all = sent;
        if constexpr (PAIR) {
            if (rank == 1 && threadIdx.x == 0) st_cluster_u32(mapa_shared(smem_u32(&s_peer_sent), 0), sent);
            __syncwarp();
            cluster_sync();
            // Stages that the second CTA sent and the first never announced: half of their bytes.
            if (rank == 0 && threadIdx.x == 0) {
                const uint32_t per_tile = (boxes + B - 1) / B;
                for (uint32_t j = sent; j < s_peer_sent; ++j)
                    mbar_arrive_expect_tx(&full[j % S], min(B, boxes - static_cast<int>(j % per_tile) * B) * box_bytes);
            }
            __syncwarp();
            all = max(sent, s_peer_sent);
        }
        if (warp == 0 && rank == 0) land(full, S, all);
        if (warp == 2) land(chunk_full, C::kChunks, sent);
        if (mmas) {
            if constexpr (PAIR) umma_commit_pair(mapa_shared(smem_u32(&drain), 0));
            else umma_commit(&drain);
            mbar_wait_drain(&drain, 0, limit);
        }
        __syncwarp();
        tc_fence_before();
        __syncthreads();
        if constexpr (PAIR) cluster_sync();
    }
    tc_fence_after();
    if (warp == 1) {
        if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

struct Matrix {
    const uint8_t* codes;
    const uint8_t* scales;
    int64_t rows;
};

template <int BN, bool PAIR, bool FOUR>
lm_status launch(const Matrix& w, const Matrix& x, int64_t k, Args a, int64_t tiles, cudaStream_t stream) {
    using C = Cfg<BN, PAIR, FOUR>;
    // No box is higher than X: rows past a map's end cost the TMA more than rows that are there (151552
    // rows of W by 2048 columns, tiles of 32 rows: 48 us with one row of X in a box of 32).  What a lower
    // box leaves in shared memory reaches columns of the accumulator that nobody reads.
    a.x_box = static_cast<int>(std::min<int64_t>(C::kBRows, x.rows));
    a.xs_box = static_cast<int>(std::min<int64_t>(BN, x.rows));
    CUtensorMap map_w, map_x, map_ws, map_xs;
    const uint64_t cols = static_cast<uint64_t>(mx_padded_cols(k)), pitch = static_cast<uint64_t>(mx_scale_pitch(k));
    const auto encode = [&](const Matrix& m, uint32_t box, uint32_t scale_box, CUtensorMap* codes, CUtensorMap* scales) {
        const bool spread = !FOUR && codes == &map_w;
        return encode_tensor_map_mx(codes, m.codes, spread, static_cast<uint64_t>(m.rows), FOUR ? cols / 2 : cols, box) &&
               encode_tensor_map_mx_scales(scales, m.scales, static_cast<uint64_t>(m.rows), pitch, scale_box);
    };
    if (!encode(w, kBlockM, kBlockM, &map_w, &map_ws) || !encode(x, static_cast<uint32_t>(a.x_box), static_cast<uint32_t>(a.xs_box), &map_x, &map_xs)) return context_free_fail(LM_ERR_CUDA, "lm_mx_matmul: cuTensorMapEncodeTiled is unavailable or failed");
    const auto kernel = mx_matmul_kernel<BN, PAIR, FOUR>;
    static std::atomic<uint64_t> configured{0};  // devices whose limit is raised
    if (const cudaError_t e = set_smem_limit_once(kernel, C::kSmemBytes, configured); e != cudaSuccess) return context_free_finish(e);
    cudaLaunchConfig_t cfg{};
    const int ctas = PAIR ? 2 : a.split;
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tiles, kSms / ctas) * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = static_cast<unsigned>(ctas);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    return context_free_finish(cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, map_ws, map_xs, a));
}

// Whether `count` CTAs that gave up on the device are news to the stream.  Nothing on the device is
// cleared: each stream is told on its own, whichever asks first, since a captured product may have
// run on any of them.  Streams are noted by the ids that CUDA never gives twice, once something stalled.
bool news(int device, unsigned long long stream_id, unsigned count) {
    static std::mutex lock;
    static std::map<std::pair<int, unsigned long long>, unsigned> told;
    const std::lock_guard<std::mutex> guard(lock);
    const std::pair<int, unsigned long long> key{device, stream_id};
    const auto it = told.find(key);
    if (it == told.end() ? count == 0 : count == it->second) return false;
    told[key] = count;
    return count != 0;  // 0: the device was reset since
}

}  // namespace

// Testing only (lm_ops_debug_set).
std::atomic<uint64_t> g_wait_limit_ns{0};
std::atomic<int> g_stall{0};

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
    const Span to(out, rows, out_stride * elem_size(out_dtype), n * elem_size(out_dtype));
    const int64_t w_rows = groups * n, scale_pitch = mx_scale_pitch(k);
    if (overlap(to, {x, rows * mx_data_pitch(x_format, k)}) || overlap(to, {x_scales, rows * scale_pitch}) || overlap(to, {w, w_rows * mx_data_pitch(LM_MX_E2M1, k)}) ||
        overlap(to, {w_scales, w_rows * scale_pitch}) || overlap(to, {offsets, (int64_t{groups} + 1) * 4}))
        return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_mx_matmul: out overlaps an input");
    // The tile's width by the average rows of a group: of the buffer, since how many of them there are
    // stands in the offsets on the device (768 rows of 64 groups in a buffer of 6144: 46 us, in one of 768
    // 39; 96 of 8 groups in 768: 12.9, in 96 11.4).  Groups are ragged, so a tile is wide enough for
    // most of them: a second tile reads the group's weights again.  (64 experts of 2816 x 2048, us with
    // 16, 32, 64 rows a tile and with a pair's 128, E4M3 rows: 4 a group 39, 41, 45, 49; 16: 51, 40, 44,
    // 47; 40: 101, 64, 45, 49; 48: 64 rows 48, a pair 49; 59: 55 and 50.  Packed E2M1 rows: 4 a group 33,
    // 34, 32, 41; 16: 35, 34, 33, 40; 59: 64 rows 36, a pair 41; 66: 42 and 42.)
    const bool four = x_format == LM_MX_E2M1;
    const int64_t each = (rows + groups - 1) / groups;
    int bn = each <= 6 ? 16 : each <= 18 ? 32 : each <= (four ? 64 : 48) ? 64 : 128;
    if (groups == 1) bn = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;  // not ragged
    const auto tiles = [&](int64_t m_blocks) { return m_blocks * ((rows + bn - 1) / bn + std::min<int64_t>(groups, rows) - 1); };  // at most
    const int64_t m_blocks = (n + kBlockM - 1) / kBlockM, k_words = mx_padded_cols(k) / 128;  // of scales
    if (tiles(m_blocks) > INT32_MAX - kSms) return context_free_fail(LM_ERR_UNSUPPORTED, "lm_mx_matmul: more than 2^31 tiles");
    // Pairs of CTAs where 128 rows a tile give them work (384 rows a group: 195 us without, 170 with).
    const bool pair = bn == 128 && tiles(m_blocks) * 2 > kSms;
    // Fewer tiles than half the SMs: narrower tiles, and clusters of two or four CTAs that share a tile's
    // columns, at least 512 each (2048 packed), and add their sums through distributed shared memory, without a
    // workspace.  Many columns are shared before tiles get narrower, few after.  (One row, 10944 columns
    // to 2048: one CTA a tile 24 us, two 17, four 12.6; eight, of which not all clusters fit the GPU at
    // once, were slower than four.  128 rows of them: 64 rows a tile shared by four 14 us, 16 rows unshared
    // 23.  256 rows of 2048 columns: 128 shared by four 10.6, 32 unshared 8.8.
    // Packed: 33 rows of 2048 columns to 1408 unshared 6.4, shared by four 7.4.)
    const int64_t least = four ? 32 : 8;  // words of columns that two CTAs may share
    int split = 1;
    for (const bool share_first = k_words >= 32; !pair; bn /= 2) {
        const auto few = [&] { return tiles(m_blocks) * split * 2 <= kSms; };
        while ((share_first || bn == 16) && split < kMaxSplit && few() && k_words >= least * split) split *= 2;
        if (bn == 16 || !few()) break;
    }
    Args a{};
    a.offsets = offsets;
    a.out = out;
    a.out_stride = out_stride;
    a.rows = static_cast<int>(rows);
    a.groups = groups;
    a.n = static_cast<int>(n);
    a.k_boxes = static_cast<int>(four ? (k_words + 1) / 2 : k_words);
    a.split = split;
    a.out_dtype = out_dtype;
    a.out_pairs = out_stride % 2 == 0 && aligned(out, 4);
    a.stall = g_stall.load(std::memory_order_relaxed);
    a.wait_limit_ns = g_wait_limit_ns.load(std::memory_order_relaxed);
    if (a.wait_limit_ns == 0) a.wait_limit_ns = kWaitLimitNs;
    if (const cudaError_t e = ops_status(&a.status); e != cudaSuccess) return context_free_finish(e);
    const Matrix mw{w, w_scales, groups * n}, mx{x, x_scales, rows};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    lm_status st = LM_OK;
    with_bool(four, [&](auto f) {
        constexpr bool FOUR = decltype(f)::value;
        if (pair) st = launch<128, true, FOUR>(mw, mx, k, a, tiles((n + 2 * kBlockM - 1) / (2 * kBlockM)), s);
        else if (bn == 16) st = launch<16, false, FOUR>(mw, mx, k, a, tiles(m_blocks), s);
        else if (bn == 32) st = launch<32, false, FOUR>(mw, mx, k, a, tiles(m_blocks), s);
        else if (bn == 64) st = launch<64, false, FOUR>(mw, mx, k, a, tiles(m_blocks), s);
        else st = launch<128, false, FOUR>(mw, mx, k, a, tiles(m_blocks), s);
    });
    return st;
}

lm_status lm_ops_debug_set(int32_t knob, int64_t value) {
    if (knob == LM_DEBUG_WAIT_LIMIT_NS && value >= 0 && value <= static_cast<int64_t>(kWaitLimitNs)) {
        g_wait_limit_ns.store(static_cast<uint64_t>(value), std::memory_order_relaxed);
        return LM_OK;
    }
    if (knob == LM_DEBUG_PRODUCT_STALL && value >= 0 && value <= LM_STALL_TMEM_EMPTY) {
        g_stall.store(static_cast<int>(value), std::memory_order_relaxed);
        return LM_OK;
    }
    return context_free_fail(LM_ERR_INVALID_ARGUMENT, "lm_ops_debug_set: an unknown knob, a limit above 2 s or an unknown barrier");
}

lm_status lm_ops_sync(void* stream) {
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned count = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&count, g_stalls, sizeof count, 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    unsigned long long id = 0;
    int device = 0;
    if (e == cudaSuccess) e = cudaStreamGetId(s, &id);
    if (e == cudaSuccess) e = cudaGetDevice(&device);
    if (e != cudaSuccess) return context_free_finish(e);
    try {
        if (!news(device, id, count)) return LM_OK;
    } catch (...) {  // no memory or lock to note it: told again at the next call
        if (count == 0) return LM_OK;
    }
    return context_free_fail(LM_ERR_DEVICE_TIMEOUT, "lm_ops_sync: a kernel gave up waiting; its results are invalid");
}

}  // extern "C"
