// Inline-PTX wrappers for the sm_100a features the kernels use: mbarrier,
// TMA bulk-tensor copies, tcgen05 (tensor memory, UMMA, commit, loads) and the
// proxy fences that order generic shared-memory accesses against them.
//
// Every wait in this library is bounded: mbar_wait() gives up after a wall
// clock budget and reports failure instead of spinning for ever, so a wrong
// descriptor or a lost arrival ends the kernel with a status word rather than a
// hung device.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace i4l {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_timer_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ bool elect_one() {
    uint32_t pred = 0;
    asm volatile(
        "{\n\t"
        ".reg .pred P;\n\t"
        "elect.sync _|P, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t"
        "}\n"
        : "=r"(pred));
    return pred != 0;
}

// ----------------------------------------------------------------- cluster --

__device__ __forceinline__ uint32_t cluster_cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_id_x() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_count_x() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%nclusterid.x;" : "=r"(r));
    return r;
}
// Full barrier over every thread of the cluster (hardware barrier; all threads
// always reach it because every software wait before it is bounded).
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The two halves of the same barrier, for code that has useful work between them.  Every thread
// executes an arrive and a wait exactly once.
// Arrive: warp-convergent forms.  `relaxed` is for warps that have written nothing the peer will
// read (a release at cluster scope costs on the order of a thousand cycles).
__device__ __forceinline__ void cluster_arrive_release() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
// Wait: convergent form, and one for a warp whose lanes have diverged.
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait_divergent() {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// Named CTA barrier `id` over the first/any `threads` threads that call it (a multiple of 32).
__device__ __forceinline__ void named_barrier_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// ---------------------------------------------------------------- mbarrier --

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

// Makes freshly initialised barriers visible to other threads and to the
// async proxy (TMA / tcgen05.commit arrive on them).
__device__ __forceinline__ void mbar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Arrive, but not before the value `loaded` exists: for handing a buffer back right after LOADING
// from it.  A load that has been issued has not yet read its data; the arrival's release does not
// wait for it, and the buffer's next writer (TMA) could overwrite what the load is about to read.
// Making the arrive instruction depend on a value computed from the loads' destination registers
// holds it back until the data has arrived (either branch arrives; the predicate is the dependency).
__device__ __forceinline__ void mbar_arrive_after(uint32_t bar, uint32_t loaded) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.eq.u32 p, %1, 0x5bd1e995;\n\t"
        "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
        "@!p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
        "}\n" ::"r"(bar), "r"(loaded)
        : "memory");
}

// Arrive on the barrier at the same shared-memory offset in CTA `cta` of this cluster.
// Release semantics at CTA scope (the default), as for a local arrive: the data the
// arrival publishes was written to shared memory through the generic proxy and fenced
// towards the async proxy by its writers, which is all the consumer (UMMA) needs.  A
// cluster-scope release here costs over a thousand cycles per arrival.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar, uint32_t cta) {
    asm volatile(
        "{\n\t"
        ".reg .b32 remote;\n\t"
        "mapa.shared::cluster.u32 remote, %0, %1;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [remote];\n\t"
        "}\n" ::"r"(bar), "r"(cta)
        : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred P;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t"
        "}\n"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// Longest time any single wait may last before the kernel declares itself
// broken.  Far above the run time of the largest supported launch.
constexpr uint64_t kWaitBudgetNs = 1000ull * 1000ull * 1000ull;

// Wait for the phase with the given parity to complete.  Returns false (after
// raising *abort_flag, a shared-memory word all roles poll) if the budget runs
// out or another thread already aborted.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          uint64_t budget_ns = kWaitBudgetNs) {
    uint64_t t0 = 0;
    for (uint32_t spin = 0;; ++spin) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 63u) == 63u) {
            if (*abort_flag) return false;
            uint64_t now = global_timer_ns();
            if (t0 == 0 || now < t0) t0 = now;  // (the timer is not promised to be monotonic: restart the budget if it steps back)
            else if (now - t0 > budget_ns) { *abort_flag = 1; return false; }
        }
    }
}

// The same for a whole warp: every lane polls, a vote makes the outcome uniform, and the warp leaves
// the call converged.  Lanes can leave the polling loop in different iterations, and nothing else
// brings them back together; use this form where a .sync.aligned tensor-memory instruction follows
// the wait (those require a converged warp).  In a hot loop that only loads and stores, the plain
// form is measurably cheaper (2.6 % of the 8192^3 GEMM).
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    const bool ok = mbar_wait(bar, parity, abort_flag);
    return __all_sync(0xFFFFFFFFu, ok) != 0;
}

// ------------------------------------------------------------------ fences --

// Orders this thread's generic-proxy shared-memory writes before later
// async-proxy reads (UMMA operand fetch, TMA store).
__device__ __forceinline__ void fence_proxy_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void tc_fence_before_sync() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after_sync() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// --------------------------------------------------------------------- TMA --

__device__ __forceinline__ void tma_prefetch_desc(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

// 2-D tiled load global -> this CTA's shared memory, completion counted in
// bytes on `bar`.  c0 is the innermost coordinate (must make a 16-byte
// aligned start), c1 the row.  No multicast.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}

// The address of this CTA's barrier `bar` at the same offset in CTA `cta` of the cluster.
__device__ __forceinline__ uint32_t cluster_address(uint32_t bar, uint32_t cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(bar), "r"(cta));
    return r;
}
// The tiled load of a CTA pair: the data go to this CTA's shared memory, the bytes are counted on a barrier in
// either CTA of the pair (cluster_address()).  No multicast.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* m, uint32_t cluster_bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(cluster_bar), "r"(c0), "r"(c1)
        : "memory");
}

// Untiled bulk load global -> this CTA's shared memory: both addresses 16-byte aligned, bytes a multiple of 16.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
        : "memory");
}

// 2-D tiled store shared -> global (bulk-group completion).  Elements of the
// box that fall outside the tensor are not written.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* m, uint32_t src, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
        ::"l"(reinterpret_cast<uint64_t>(m)), "r"(src), "r"(c0), "r"(c1)
        : "memory");
}
// The same as a reduction: every int32 of the box is ADDED to the element in global memory
// (performed at the L2 as an atomic add; boxes from different CTAs may overlap in time).
__device__ __forceinline__ void tma_reduce_add_2d(const CUtensorMap* m, uint32_t src, int c0, int c1) {
    asm volatile(
        "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
        ::"l"(reinterpret_cast<uint64_t>(m)), "r"(src), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_store_commit() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Wait until at most N of this thread's store groups still READ shared memory.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void tma_store_wait_all() {
    asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory");
}

// ----------------------------------------------------------- tensor memory --

// Whole-warp collective.  Writes the allocated base address to *dst (shared).
template <int kCtaGroup>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t ncols) {
    if constexpr (kCtaGroup == 1)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(ncols) : "memory");
    else
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(ncols) : "memory");
}
template <int kCtaGroup>
__device__ __forceinline__ void tmem_relinquish() {
    if constexpr (kCtaGroup == 1)
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    else
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
template <int kCtaGroup>
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    if constexpr (kCtaGroup == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// ------------------------------------------------------------------- UMMA --

// Shared-memory matrix descriptor for a K-major operand tile stored as rows of
// 128 bytes with the 128-byte swizzle (16-byte chunk index XOR row%8), rows
// grouped in 8-row / 1024-byte atoms that follow one another.
//   bits  0-13  start address >> 4
//   bits 16-29  leading byte offset >> 4 (unused for swizzled K-major; 1)
//   bits 32-45  stride byte offset  >> 4 (1024 B between 8-row atoms -> 64)
//   bits 46-47  descriptor version (1 on sm_100)
//   bits 61-63  layout type (2 = SWIZZLE_128B)
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Instruction descriptor for kind::i8, signed 8-bit A and B (both K-major),
// int32 accumulator, no saturation, dense.
//   bits 4-5 D format (2 = s32); 7-9 A format (1 = s8); 10-12 B format (1 = s8);
//   15/16 A/B major (0 = K); 17-22 N>>3; 24-28 M>>4.
__host__ __device__ constexpr uint32_t umma_idesc_s8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// D[tmem] (+)= A[smem] * B[smem]^T, issued by ONE thread.
template <int kCtaGroup>
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kCtaGroup == 1)
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}

// The same with the A operand read from tensor memory: lane = row, each 32-bit column holds four
// consecutive K bytes, 8 columns per instruction (K = 32).  B from shared memory.  One CTA.
__device__ __forceinline__ void umma_i8_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor for the block-scaled 4-bit kinds: A and B e2m1 (format 1), both K-major, fp32
// accumulator, dense, K = 64 per instruction.
//   bits 4-5 / 29-30 scale-factor id of B / A; 7-9, 10-12 operand formats (1 = e2m1);
//   17-22 N>>3; 23 scale type (0 = ue4m3, 1 = ue8m0); 24-28 M>>4.
// A scale-factor id names the first byte an instruction uses of each 32-bit scale word (0 or 2 when a
// word serves two instructions: mxfp4; 0 when it serves one: nvfp4).
__host__ __device__ constexpr uint32_t umma_idesc_fp4(int m, int n, bool ue8m0, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (ue8m0 ? 1u << 23 : 0u) | (static_cast<uint32_t>(m >> 4) << 24) | (sf_id << 29);
}

// D[tmem] (+)= (A[smem] scaled) * (B[smem] scaled)^T, K = 64, scales in tensor memory (a row's scale word in
// lane row % 32, column row / 32, the 32 lanes repeated in all four quarters).  Issued by ONE thread.
// kBlock16: nvfp4 (a ue4m3 scale per 16 elements), else mxfp4 (a ue8m0 scale per 32).
// The operand descriptors are those of umma_desc_sw128, given by their low words (address and leading offset): the high
// word is a constant, and the issuing warp, whose instructions bound the step, adds 32 bits instead of 64.
__device__ __forceinline__ uint32_t umma_desc_sw128_low(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }
constexpr uint32_t kUmmaDescSw128High = (1024u >> 4) | (1u << 14) | (2u << 29);

template <int kCtaGroup, bool kBlock16>
__device__ __forceinline__ void umma_fp4(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                         uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
#define I4L_UMMA_FP4(GROUP, KIND)                                                                        \
    asm volatile(                                                                                        \
        "{\n\t"                                                                                          \
        ".reg .pred p;\n\t"                                                                              \
        ".reg .b64 da, db;\n\t"                                                                          \
        "mov.b64 da, {%1, %7};\n\t"                                                                      \
        "mov.b64 db, {%2, %7};\n\t"                                                                      \
        "setp.ne.b32 p, %6, 0;\n\t"                                                                      \
        "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], da, db, %3, [%4], [%5], p;\n\t"           \
        "}\n" ::"r"(d_tmem), "r"(a_low), "r"(b_low), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem),           \
        "r"(accumulate), "r"(kUmmaDescSw128High) : "memory")
    if constexpr (kCtaGroup == 1) {
        if constexpr (kBlock16) I4L_UMMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
        else I4L_UMMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
    } else {
        if constexpr (kBlock16) I4L_UMMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
        else I4L_UMMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
    }
#undef I4L_UMMA_FP4
}

// Copies one 512-byte scale tile (32 rows of 16 bytes, no swizzle: 8-row groups of 128 bytes that follow one another;
// tcgen05.cp 32x128b) into 4 columns of tensor memory, repeated in the four lane quarters.  `low` is the tile's
// shared-memory address >> 4.  Issued by the thread that issues the UMMAs reading it: copies and UMMAs of one thread are
// executed in order.
__device__ __forceinline__ uint32_t scale_tile_low(uint32_t smem_addr) { return (smem_addr & 0x3FFFFu) >> 4; }
template <int kCtaGroup>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint32_t low) {
    constexpr uint32_t kHigh = (128u >> 4) | (1u << 14);
    if constexpr (kCtaGroup == 1)
        asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}\n" ::"r"(taddr), "r"(low), "r"(kHigh) : "memory");
    else
        asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}\n" ::"r"(taddr), "r"(low), "r"(kHigh) : "memory");
}

// Instruction descriptor for kind::f16 with bfloat16 operands and an fp32 accumulator.
//   bits 4-5 D format (1 = f32); 7-9, 10-12 operand formats (1 = bf16); 15/16 A/B major (0 = K, 1 = MN);
//   17-22 N>>3; 24-28 M>>4.
__host__ __device__ constexpr uint32_t umma_idesc_bf16(int m, int n, bool a_mn_major, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn_major ? 1u << 15 : 0u) | (b_mn_major ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Issued by one thread for both CTAs of a pair.
__device__ __forceinline__ void umma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Descriptor of an MN-major 16-bit operand with the 128-byte swizzle: atoms of 64 (MN) x 8 (K) elements,
// 1024 bytes; atoms follow one another along K, `chunk_bytes` apart along MN.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t chunk_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(chunk_bytes >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Arrive once on `bar` when every UMMA this thread issued so far has finished
// (implies tcgen05.fence::before_thread_sync).
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 2-CTA form: arrives on the barrier at this offset in each CTA named by mask.
__device__ __forceinline__ void umma_commit_2cta(uint32_t bar, uint16_t cta_mask) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"(cta_mask) : "memory");
}

// Each thread of the warp reads 32 consecutive 32-bit columns of its own TMEM
// lane (lane = 32*(warp%4) + thread).  Asynchronous until tmem_ld_wait().
__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
// Each thread of the warp writes 32 consecutive 32-bit columns of its own tensor-memory lane (the
// warp's index modulo 4 selects the quarter of the 128 lanes it may touch).
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        :: "r"(taddr),
           "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
           "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
           "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
           "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// --------------------------------------------------------- shared memory --

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

}  // namespace i4l
