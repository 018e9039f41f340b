// ptx.cuh -- inline-PTX wrappers for sm_100a: mbarriers, TMA tile loads, tcgen05
// (TMEM allocation, UMMA issue/commit, TMEM loads), programmatic dependent launch.
//
// Every wait on an mbarrier is bounded: after kWaitLimitNs of global time the
// waiter records a status code in device memory, raises the CTA's abort flag and
// returns false, so a broken pipeline ends the kernel with an error instead of a
// hang.  Every copy here is issued by the CTA whose shared memory receives it.
#pragma once

#include <cstdint>
#include <cuda.h>

namespace lm {

constexpr uint64_t kWaitLimitNs = 2000000000ull;  // 2 s

// Status codes written to the context's device status word.
constexpr int kDevOk = 0;
constexpr int kDevTimeoutProducer = 1;
constexpr int kDevTimeoutMma = 2;
constexpr int kDevTimeoutEpilogue = 3;
constexpr int kDevBadTile = 4;
constexpr int kDevTimeoutGrid = 5;  // a grid-wide arrival counter never reached its target
constexpr int kDevBadRow = 6;       // an output row index outside its buffer (the store was skipped)
constexpr int kDevTimeoutExchange = 7;  // a peer's readiness flag never reached this forward's epoch

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_timer_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// ── programmatic dependent launch ─────────────────────────────────────────
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ── mbarrier ──────────────────────────────────────────────────────────────
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void fence_mbar_init() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
                 : "memory");
}
// CLUSTER_TMEM: a barrier that threads of the pair's other CTA arrive on with mbar_arrive_cluster_tmem.
// The wait observes them at the cluster's scope and orders no memory; the tcgen05 fence behind it orders
// TMEM.
template <bool CLUSTER_TMEM = false>
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    if constexpr (CLUSTER_TMEM)
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
    return done != 0;
}

// One look, without waiting.
template <bool CLUSTER_TMEM = false>
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    if constexpr (CLUSTER_TMEM)
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.test_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
    return done != 0;
}

// Waits for the phase with the given parity to complete.  Returns false when the
// CTA's abort flag is raised or the time limit passes (then it records `code`).
template <bool CLUSTER_TMEM = false>
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          int* status, int code, uint64_t limit_ns = kWaitLimitNs) {
    if (mbar_try_wait<CLUSTER_TMEM>(bar, parity)) return true;
    const uint64_t start = global_timer_ns();
    while (true) {
        if (mbar_try_wait<CLUSTER_TMEM>(bar, parity)) return true;
        if (*abort_flag) return false;
        if (global_timer_ns() - start > limit_ns) {
            *abort_flag = 1;
            atomicCAS(status, 0, code);
            return false;
        }
    }
}

// A wait used only while shutting down after an abort: bounded, ignores the flag.
__device__ __forceinline__ bool mbar_wait_drain(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
    const uint64_t start = global_timer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (global_timer_ns() - start > limit_ns) return false;
    }
    return true;
}

// ── grid-wide arrival counters (cooperative launches only) ───────────────
// A launch waits for gridDim.x arrivals on each counter; the last CTA to leave the
// kernel sets the counters back to zero, so every launch (a CUDA graph replay too)
// starts from zero without any host-side bookkeeping.
__device__ __forceinline__ unsigned long long ld_acquire_u64(const unsigned long long* p) {
    unsigned long long v;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void red_release_add_u64(unsigned long long* p, unsigned long long v) {
    asm volatile("red.release.gpu.global.add.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned long long atom_acq_rel_add_u64(unsigned long long* p, unsigned long long v) {
    unsigned long long old;
    asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], %2;" : "=l"(old) : "l"(p), "l"(v) : "memory");
    return old;
}
// Orders this thread's generic-proxy global writes before later async-proxy (TMA)
// reads of the same memory, in this CTA or another.
__device__ __forceinline__ void fence_proxy_async_global() {
    asm volatile("fence.proxy.async.global;" ::: "memory");
}
// Bounded wait until *ctr >= target.  Gives up when the CTA's abort flag is raised,
// when another CTA has already recorded an error in the status word, or after
// limit_ns (then it records `code`).
__device__ __forceinline__ bool grid_wait(const unsigned long long* ctr, unsigned long long target,
                                          volatile int* abort_flag, int* status, int code,
                                          uint64_t limit_ns = kWaitLimitNs) {
    if (ld_acquire_u64(ctr) >= target) return true;
    const uint64_t start = global_timer_ns();
    while (true) {
        if (ld_acquire_u64(ctr) >= target) return true;
        if (*abort_flag || *reinterpret_cast<volatile int*>(status) != 0) {
            *abort_flag = 1;
            return false;
        }
        if (global_timer_ns() - start > limit_ns) {
            *abort_flag = 1;
            atomicCAS(status, 0, code);
            return false;
        }
        __nanosleep(32);
    }
}

__device__ __forceinline__ int ld_acquire_s32(const int* p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void red_release_add_s32(int* p, int v) {
    asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// Bounded wait until *ctr >= target (a 32-bit count), with grid_wait's exits.
__device__ __forceinline__ bool count_wait_s32(const int* ctr, int target, volatile int* abort_flag, int* status,
                                               int code, uint64_t limit_ns = kWaitLimitNs) {
    if (ld_acquire_s32(ctr) >= target) return true;
    const uint64_t start = global_timer_ns();
    while (true) {
        if (ld_acquire_s32(ctr) >= target) return true;
        if (*abort_flag || *reinterpret_cast<volatile int*>(status) != 0) {
            *abort_flag = 1;
            return false;
        }
        if (global_timer_ns() - start > limit_ns) {
            *abort_flag = 1;
            atomicCAS(status, 0, code);
            return false;
        }
        __nanosleep(32);
    }
}

// Orders this thread's generic-proxy shared-memory accesses before later async-proxy
// (TMA, bulk copy) writes to the same memory.
__device__ __forceinline__ void fence_proxy_async_shared() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Copy `bytes` (a multiple of 16) of global memory at `src` (16-byte aligned) into this
// CTA's shared memory at `smem_dst` (16-byte aligned), completing the bytes on `bar`.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            smem_u32(smem_dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// Hint: bring `bytes` (a multiple of 16) of global memory at `src` (16-byte aligned)
// into L2.  Nothing to wait for.
__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// ── TMA ───────────────────────────────────────────────────────────────────
__device__ __forceinline__ void tma_prefetch_desc(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// 2-D tile load global -> shared, completing `bytes` on `bar`.  x is the
// innermost coordinate in elements and must be a multiple of 16 bytes.
__device__ __forceinline__ void tma_load_2d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x,
                                            int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(smem_u32(smem_dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y)
        : "memory");
}

// Same with an L2 eviction-priority hint (a createpolicy value).
__device__ __forceinline__ void tma_load_2d_hint(void* smem_dst, const CUtensorMap* map, uint64_t* bar,
                                                 int32_t x, int32_t y, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
        "[%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(smem_dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "l"(policy)
        : "memory");
}

__device__ __forceinline__ uint64_t policy_evict_first() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t policy_evict_last() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}

// ── tcgen05 ───────────────────────────────────────────────────────────────
__device__ __forceinline__ void tmem_alloc(uint32_t* dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T, bf16 inputs, f32 accumulate (kind::f16).
__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrives once on `bar` when every tcgen05.mma issued so far by this thread completes.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_u32(bar))
                 : "memory");
}

// Instruction descriptor: bf16 A and B, both K-major, f32 accumulator, M x N.
__host__ __device__ constexpr uint32_t umma_idesc_bf16(int M, int N) {
    return (1u << 4)                                  // D format: f32
           | (1u << 7)                                // A format: bf16
           | (1u << 10)                               // B format: bf16
           | (static_cast<uint32_t>(N >> 3) << 17)    // N / 8
           | (static_cast<uint32_t>(M >> 4) << 24);   // M / 16
}

// Shared-memory matrix descriptor for a K-major tile written by TMA with 128-byte
// swizzle: rows of 64 bf16 (128 B), 8-row atoms 1024 B apart.  The tile must start
// on a 1024-byte boundary; stepping K by 16 elements adds 32 bytes to the start.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4)  // start address
           | (static_cast<uint64_t>(1) << 16)                   // leading byte offset (unused here)
           | (static_cast<uint64_t>(1024 >> 4) << 32)           // stride byte offset: 8 rows
           | (static_cast<uint64_t>(1) << 46)                   // descriptor version (sm_100)
           | (static_cast<uint64_t>(2) << 61);                  // swizzle: 128 B
}

// 32 lanes x 32 bits, 16 consecutive columns per thread.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ── block-scaled MMA: 8- and 4-bit operands with E8M0 scales of 32 columns ──
// D[tmem] (+)= (A * 2^sa) * (B * 2^sb)^T, with A and B in shared memory as 128-byte swizzled rows.
//   FOUR = false  kind::mxf8f6f4, 32 columns: 8-bit codes, or 4-bit ones spread as TMA's 16U4_ALIGN16B
//                 type writes them (16 codes in 8 bytes, then 8 unused bytes)
//   FOUR = true   kind::mxf4, 64 columns: both operands 4-bit and packed
// Scales sit in TMEM: word (lane i, column c) of `sfa` holds four scale bytes of row 32 c + i, the same
// in each 32-lane quadrant; the descriptor names the byte, or the first of the two bytes of 64 columns.
// PAIR: over a CTA pair (M = 256, issued by the first): each CTA holds half of A's rows with their
// scales, half of B's rows, and the scales of all of B's rows.
template <bool PAIR, bool FOUR>
__device__ __forceinline__ void umma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, uint32_t accumulate) {
#define LM_UMMA_MX(CTAS, KIND)                                                                                             \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"                                                            \
                 " tcgen05.mma.cta_group::" CTAS ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d_tmem),     \
                 "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                  \
                 : "memory")
    if constexpr (FOUR && PAIR) LM_UMMA_MX("2", "mxf4.block_scale.scale_vec::2X");
    else if constexpr (FOUR) LM_UMMA_MX("1", "mxf4.block_scale.scale_vec::2X");
    else if constexpr (PAIR) LM_UMMA_MX("2", "mxf8f6f4.block_scale.scale_vec::1X");
    else LM_UMMA_MX("1", "mxf8f6f4.block_scale.scale_vec::1X");
#undef LM_UMMA_MX
}
// Operand formats of kind::mxf8f6f4 and of kind::mxf4.
constexpr uint32_t kUmmaE4M3 = 0, kUmmaE2M1 = 5, kUmmaPackedE2M1 = 1;
__host__ __device__ constexpr uint32_t umma_idesc_mx(uint32_t a_format, uint32_t b_format, int M, int N, int scale_byte) {
    return (static_cast<uint32_t>(scale_byte) << 4)     // B's scale byte
           | (a_format << 7) | (b_format << 10)
           | (static_cast<uint32_t>(N >> 3) << 17)      // N / 8
           | (1u << 23)                                 // scales are E8M0
           | (static_cast<uint32_t>(M >> 4) << 24)      // M / 16
           | (static_cast<uint32_t>(scale_byte) << 29); // A's scale byte
}
// 32 lanes x 32 bits, 16 consecutive columns per thread; tmem_st_wait before the fence that publishes them.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ── CTA pairs (clusters of 2) ─────────────────────────────────────────────
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The shared::cluster address of the same shared-memory object in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa_shared(uint32_t smem_addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar_addr) : "memory");
}
// The same for a barrier that orders TMEM accesses only, which the tcgen05 fences around it do: the
// arrival itself releases no memory, at the scope of the waiter in the other CTA.  (A release at that
// scope waits for the thread's earlier memory accesses, 1700 cycles.)
__device__ __forceinline__ void mbar_arrive_cluster_tmem(uint32_t cluster_bar_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar_addr) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}
// TMA tile load into this CTA's shared memory whose completion is counted on an
// mbarrier of the pair's leader CTA (`leader_bar` is a shared::cluster address).
// Each CTA loads its own half of the operands.
__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, uint32_t leader_bar,
                                                 int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%3, %4}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(map), "r"(leader_bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D[tmem of both CTAs] (+)= A[smem of both] * B[smem of both]^T, issued by the leader.
__device__ __forceinline__ void umma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives once on the mbarrier at shared::cluster address `cluster_bar` (this CTA's
// or the peer's) when the leader's MMAs issued so far complete.  Called once per
// CTA of the pair to signal both.
__device__ __forceinline__ void umma_commit_pair(uint32_t cluster_bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(cluster_bar)
                 : "memory");
}

// Arrives once on the mbarrier at this shared-memory offset in both CTAs of the pair when the
// leader's MMAs issued so far complete.
__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
// Named barrier for a subset of warps.
__device__ __forceinline__ void named_bar_sync(uint32_t id, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// True in one lane of a converged warp, the same one every time; the branch on it stays uniform.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ uint32_t elect_one_lane() { return (threadIdx.x & 31u) == 0u; }

}  // namespace lm
