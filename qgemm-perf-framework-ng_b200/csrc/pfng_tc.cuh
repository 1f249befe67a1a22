// pfng_tc.cuh -- tcgen05 / tensor memory primitives and bounded waits shared
// by the kernels that use the 5th-generation tensor cores.
#pragma once

#include "pfng_common.cuh"

namespace pfng {

// ---- TMA / tcgen05 / proxy primitives ----------------------------------------
PFNG_DEV void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
PFNG_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
PFNG_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

PFNG_DEV void tmem_alloc(uint32_t *holder, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)),
                 "r"(ncols)
                 : "memory");
}
PFNG_DEV void tmem_relinquish() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory"); }
PFNG_DEV void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Arrives on `bar` once every tcgen05.mma this thread issued before has completed.
PFNG_DEV void umma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// Shared-memory matrix descriptor, K-major operand with the 128-byte swizzle:
// rows of 128 bytes, 8-row atoms of 1024 bytes stored back to back (stride
// byte offset 1024), the 16-byte chunk j of row r stored at chunk j ^ (r % 8)
// -- the layout a TMA copy with CU_TENSOR_MAP_SWIZZLE_128B and a 128-byte
// inner box writes.  `saddr` is the operand's first byte for this MMA (atom
// base + k offset).
PFNG_DEV uint64_t sw128_desc(uint32_t saddr) {
    uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);  // start address, 16-byte units
    d |= static_cast<uint64_t>(1u) << 16;                         // leading byte offset (unused with this swizzle)
    d |= static_cast<uint64_t>(1024u >> 4) << 32;                 // stride byte offset between 8-row atoms
    d |= static_cast<uint64_t>(1u) << 46;                         // descriptor version of sm_100
    d |= static_cast<uint64_t>(2u) << 61;                         // layout: 128-byte swizzle
    return d;
}
// Bounded wait that also gives up (false) once the CTA's abort flag is up.
// Each attempt is a hardware-suspended try_wait, so a waiting warp issues
// almost nothing; the abort flag is looked at every 16 attempts.
PFNG_DEV bool wait_bar(uint64_t *bar, uint32_t parity, const int *abort_flag, int *err, int code) {
    for (uint32_t i = 0; i < kWaitAttempts; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 15u) == 15u && *reinterpret_cast<const volatile int *>(abort_flag)) return false;
    }
    report_error(err, code);
    return false;
}
PFNG_DEV bool aborted(const int *abort_flag) { return *reinterpret_cast<const volatile int *>(abort_flag) != 0; }
// The wait of the roles off the critical path (producer, MMA issuer): each
// attempt may suspend the thread for up to 20 us (or until the phase
// completes), so that its polling does not take issue slots from the fold
// warps on its scheduler; the wait is bounded by ~1 s of wall time
// (%globaltimer), whatever the suspensions actually last.
PFNG_DEV uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
PFNG_DEV bool mbar_try_wait_long(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
PFNG_DEV bool wait_bar_sleep(uint64_t *bar, uint32_t parity, const int *abort_flag, int *err, int code) {
    if (mbar_try_wait_long(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
        if (mbar_try_wait_long(bar, parity)) return true;
        if (*reinterpret_cast<const volatile int *>(abort_flag)) return false;
        if (global_ns() - t0 > 1000000000ull) break;
    }
    report_error(err, code);
    return false;
}

}  // namespace pfng
