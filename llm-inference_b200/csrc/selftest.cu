// Self-test of the kernels' bounded waits: a wait that nothing will ever complete must give up
// after its time limit, record DEV_ERR_WAIT_TIMEOUT in the device error word and return, leaving
// the context usable. The kernel here runs the same wait primitive the pipelined kernels use
// (mbar_wait, common.cuh) on an mbarrier whose phase never completes: one thread arrives with an
// expected transaction count that no copy will ever deliver. Nothing faults, traps or hangs:
// the wait ends at WAIT_LIMIT_NS.
//
// The second kernel does the same in the middle of a ring between a warp that loads and one that reads (waiter.cuh): once
// the reader has given up, the loading warp must stop, and all that it had loaded must have arrived before the end: in
// either of the ways that are in use.
#include "waiter.cuh"

namespace q3 {
namespace {

__device__ unsigned g_dev_error;

__global__ void wait_timeout_kernel(int *done) {
    __shared__ __align__(8) uint64_t bar;
    if (threadIdx.x != 0) return;
    mbar_init(&bar, 1);
    fence_barrier_init();
    mbar_arrive_expect_tx(&bar, 16);  // 16 bytes that no copy brings: phase 0 never completes
    const bool ok = mbar_wait(&bar, 0, &g_dev_error);
    *done = ok ? 1 : 2;
}

constexpr int RING_STAGES = 2, RING_STEPS = 64, RING_STUCK = 2;

__global__ void ring_timeout_kernel(int *out, const int *src, bool starve) {
    __shared__ __align__(16) int ring[RING_STAGES][4];
    __shared__ __align__(8) uint64_t full[RING_STAGES], empty[RING_STAGES];
    __shared__ int down;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x < RING_STAGES * 4) ring[threadIdx.x / 4][threadIdx.x % 4] = 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < RING_STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        fence_barrier_init();
        down = 0;
    }
    fence_proxy_async();
    __syncthreads();
    Waiter wait(&g_dev_error, &down);
    int loaded = 0;
    for (int u = 0; u < RING_STEPS; u++) {
        const int s = u % RING_STAGES;
        const uint32_t ph = u / RING_STAGES & 1;
        if (warp == 1) {
            if (u == RING_STUCK + RING_STAGES) {  // waits for the reader's stage later than the reader for its load, so that it gives up first
                const uint64_t t = globaltimer();
                while (globaltimer() - t < WAIT_LIMIT_NS / 4) {
                }
            }
            wait(&empty[s], ph ^ 1);
            if (starve ? __any_sync(0xffffffffu, wait.dead) : wait.stopped()) break;
            if (lane == 0) {
                // one step expects 16 bytes more than come: its phase never completes
                mbar_arrive_expect_tx(&full[s], u == RING_STUCK ? 32 : 16);
                bulk_g2s(ring[s], src + 4 * u, 16, &full[s]);
            }
            loaded++;
        } else {
            wait(&full[s], ph);
            __syncwarp();
            if (lane == 0 && !(starve && wait.dead)) mbar_arrive(&empty[s]);
        }
    }
    if (__syncthreads_or(wait.dead)) settle();
    if (threadIdx.x == 32) {
        out[0] = wait.dead ? 2 : 1;
        out[1] = loaded;
        for (int s = 0; s < RING_STAGES; s++) out[2 + s] = *reinterpret_cast<volatile int *>(&ring[s][3]);
    }
}

}  // namespace

unsigned take_error_selftest() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v)) != cudaSuccess) return 0;
    if (v) cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return v;
}

}  // namespace q3

// Runs one wait that must time out (about WAIT_LIMIT_NS, two seconds) on `stream`; *done (device
// memory) becomes 2 when the wait gave up, 1 if it had completed. q3_device_error then reports
// Q3_DEV_ERR_WAIT_TIMEOUT.
extern "C" int q3_selftest_wait_timeout(int *done, void *stream) {
    if (!done) return Q3_ERR_ARG;
    q3::wait_timeout_kernel<<<1, 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(done);
    return q3::record_cuda_error(cudaGetLastError());
}

// The same for a ring of two stages between a loading and a reading warp, 64 steps of 16 bytes of `src` (256 ints of device
// memory). The reader gives up at the third; out (four ints): 2 if the loading warp stopped, the loads that it issued,
// and the last word of either stage.
extern "C" int q3_selftest_ring_timeout(int *out, const int *src, int starve, void *stream) {
    if (!out || !src) return Q3_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(src) % 16 != 0) return Q3_ERR_ALIGN;
    q3::ring_timeout_kernel<<<1, 64, 0, reinterpret_cast<cudaStream_t>(stream)>>>(out, src, starve != 0);
    return q3::record_cuda_error(cudaGetLastError());
}
