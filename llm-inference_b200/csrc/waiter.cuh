// Bounded waits of kernels whose warps hand ring stages to one another.
//
// A wait that gives up must not leave anything behind: the roles go on without waiting, so that every barrier of the
// CTA still sees its arrivals; what loads stops loading, because a stage may still be owed to a load before; and
// the CTA ends only when all copies and products that it has started have ended, too.
#pragma once

#include "common.cuh"

namespace q3 {

// Polls a barrier a few thousand times. The loop is four instructions, and what follows a wait that gives up is out
// of line: the roles' loops compete for the instruction cache.
__device__ __forceinline__ bool poll(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
        "mov.u32 n, 4096;\n\t"
        "again:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra done;\n\t"
        "sub.u32 n, n, 1;\n\t"
        "setp.ne.u32 q, n, 0;\n\t"
        "@q bra again;\n\t"
        "done:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

static __device__ __noinline__ bool wait_clocked(uint64_t *bar, uint32_t parity, unsigned *err, int *down) {
    const bool ok = mbar_wait(bar, parity, err);
    if (!ok) *reinterpret_cast<volatile int *>(down) = 1;
    return ok;
}

// Waits until one has given up, which is noted in the CTA's shared word `down` (zero at the start) before this thread's
// next arrival; from then on it returns at once.
struct Waiter {
    unsigned *err;
    int *down;
    bool dead = false;
    __device__ __forceinline__ Waiter(unsigned *err, int *down) : err(err), down(down) {}
    __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
        if (!dead && !poll(bar, parity)) dead = !wait_clocked(bar, parity, err, down);
    }
    // For a warp that loads, all lanes, after it has waited for an empty stage: whether any role has given up, this
    // one or that which emptied the stage. Then no more loads.
    __device__ __forceinline__ bool stopped() {
        dead = __any_sync(0xffffffffu, dead || *reinterpret_cast<volatile int *>(down) != 0);
        return dead;
    }
};

// The end of the CTA's work, all threads. After a wait that gave up: what was issued until then ends well within this time.
__device__ __forceinline__ void settle(const Waiter &wait) {
    if (!__syncthreads_or(wait.dead)) return;
    const uint64_t t = globaltimer();
    while (globaltimer() - t < 1000000) {
    }
}

}  // namespace q3
