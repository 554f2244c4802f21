// Bounded waits of kernels whose warps hand ring stages to one another.
//
// A wait that gives up must not leave anything behind. The roles go on without waiting, so that the CTA comes to its end.
// Loading stops, because a load that never came may still be owed to a stage: either who has given up releases no more
// stages, so that the loading warps starve and give up in turn (that costs their loop nothing), or, where the tensor
// core releases them, the loading warps look at a shared word. And the CTA ends only when the copies and products that it
// has started have ended, too.
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

// After a wait that gave up, at the end: what was issued until then ends well within this time.
static __device__ __noinline__ void settle() {
    const uint64_t t = globaltimer();
    while (globaltimer() - t < 1000000) {
    }
}

}  // namespace q3
