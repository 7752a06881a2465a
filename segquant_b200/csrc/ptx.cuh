// PTX wrappers shared by the tensor-core kernels: mbarriers with bounded waits, TMA loads, tensor memory, descriptors.
//
// Every wait is bounded: when one runs out the kernel records a code in its translation unit's status word, raises a
// CTA-wide abort flag and every role leaves its loop.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace sq {

// Written (first writer wins) when a bounded wait gives up: (block index << 8) | WaitCode.
// One copy per translation unit and device; read and cleared through tu_read_status().
static __device__ unsigned long long g_wait_status = 0ull;

// ---------------------------------------------------------------------------------------------
// PTX wrappers
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrival on a barrier of this CTA or of the other CTA of the pair (cluster address).  Default semantics (release at CTA
// scope): what the waiter consumes is tensor memory, ordered by the tcgen05 fences on both sides, or shared memory written
// for the async proxy, ordered by the writer's fence.proxy.async; a cluster-scope release here was measured at 1100-1900
// cycles per arrival (it was the longest step of the int4 expansion warps and of every accumulator hand-back of a pair).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done;
}
// The same test with a suspend-time hint (nanoseconds): the thread may sleep in hardware until the phase completes instead
// of returning early to poll again.  Used by the MMA issuer of the one-CTA kernel with 8-bit weights: that kernel runs at
// its shared-memory roofline, every poll of a barrier is one more shared-memory access, and with the hint its K = 1536
// layers are 4-6 % faster when run back to back (8192 x 6144 x 1536: 71.2 -> 67.9 us; inside the MMDiT step, among other
// kernels, the difference is within noise).  Measured and left alone: the same hint on the producer's,
// table builders' and epilogue's waits (no change), on the int4 expansion path (3 % slower) and on the pair kernel's
// issuer (1 % slower on the headline layer).
__device__ __forceinline__ uint32_t mbar_try_wait_relaxed(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(20000)
        : "memory");
    return done;
}
__device__ __forceinline__ unsigned long long global_timer_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Bounded wait: gives up after `limit` SM cycles (GemmParams::wait_cycles, 4e9 = about 2 s unless the host changed
// it), or as soon as another role has raised the abort flag.  (Backing off with nanosleep was measured: no gain for the epilogue, slower hand-offs.)  The timeout uses the SM-local cycle counter: reading %globaltimer costs microseconds.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code, long long limit,
                                          bool relaxed = false) {
    if (relaxed ? mbar_try_wait_relaxed(bar, parity) : mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
#pragma unroll 1
    for (uint32_t it = 1;; ++it) {
        if (relaxed ? mbar_try_wait_relaxed(bar, parity) : mbar_try_wait(bar, parity)) return true;
        if ((it & 1023u) == 0u) {
            if (*abort_flag) return false;
            if (clock64() - t0 > limit) {
                atomicCAS(&g_wait_status, 0ull, (static_cast<unsigned long long>(blockIdx.x) << 8) | static_cast<unsigned>(code));
                *abort_flag = 1;
                __threadfence_block();
                return false;
            }
        }
    }
}

// The same wait by all lanes of a warp that has to stay whole behind it (warp-wide instructions, named barriers): either all of them
// give up or none.  Lanes give up where all 32 arrive at it together.  A part of the warp there means that the other lanes have seen
// the phase complete, and goes on with them.  (A vote behind every wait of the attention's softmax warps was measured at 332 -> 340 us
// for 4429 tokens, 24 heads, two samples; nothing of this lies on the way of a wait that succeeds.)
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code, long long limit) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
#pragma unroll 1
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 1023u) == 0u && (*abort_flag || clock64() - t0 > limit)) {
            if (__activemask() != 0xffffffffu) return true;
            atomicCAS(&g_wait_status, 0ull, (static_cast<unsigned long long>(blockIdx.x) << 8) | static_cast<unsigned>(code));
            *abort_flag = 1;
            __threadfence_block();
            return false;
        }
    }
}

// The record of a wait that gave up, for a thread that watches several barriers.
__device__ __forceinline__ void wait_gave_up(int code) {
    atomicCAS(&g_wait_status, 0ull, (static_cast<unsigned long long>(blockIdx.x) << 8) | static_cast<unsigned>(code));
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_tmap(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// tcgen05.commit: the mbarrier gets one arrival when every tcgen05.mma issued so far by this
// thread has finished reading shared memory and writing tensor memory.
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

template <uint32_t N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <uint32_t N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// Shared-memory matrix descriptor of a K-major operand tile stored as rows of 128 bytes with the
// 128-byte swizzle (what TMA SWIZZLE_128B writes).  Low word: start address >> 4 (14 bits) and the
// leading-dimension offset (unused for swizzled K-major layouts, set to 1).  High word: 8-row groups
// are 1024 bytes apart (SBO = 64), descriptor version 1 = Blackwell (bit 46), layout type 2 =
// SWIZZLE_128B (bits 61-63).  Stepping K by one MMA (32 bytes) adds 2 to the low word.
constexpr uint32_t kSmemDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t smem_desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint64_t smem_desc(uint32_t lo) { return (static_cast<uint64_t>(kSmemDescHi) << 32) | lo; }

}  // namespace sq
