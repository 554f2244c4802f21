// Low-rank adapters of many requests beside a shared projection (q3_lora_plan, q3_lora_add, q3_lora_gate_up):
// out = base + s_i B_i (A_i x) for the rows of adapter i, A_i [rank, k], B_i [n, rank], up to three projections of one x.
//
// The plan sorts a step's rows by their adapter, once for all layers, and cuts them into tiles, so that rows of one adapter
// anywhere in the batch share its weights. A cluster of CTAs takes a tile: each CTA multiplies its part of k, the partial
// A x are added up through distributed shared memory, and each CTA expands its part of the columns; nothing goes through global
// memory between the two products. Both run on warp-level matrix instructions, with operands loaded straight into
// registers but for the first product of long or wide tiles, whose operands come through shared memory: the contraction's order is free as long as both operands have the same, so a lane takes eight (A x) or four
// (B h) neighbouring elements of its row, and its four columns of eight-column tiles are dealt out so that a lane writes eight
// neighbouring outputs. What cannot be done without is the bytes of x, base, out and the present adapters' weights (a rank of 64 is 64
// products for each element of x, a tenth of what the tensor cores could do meanwhile). Few rows are bound by the chain of loads
// and two cluster barriers (one row through q, k and v 8.4 us, 32 rows 9.6), long steps by that chain in each warp beside the
// bytes (2079 rows 36 us; of 36.8 before the bases' early fetch the first product alone took 14, the second alone 26.6, that without the
// bases' loads 20.8, without the stores 22.2, without matrix instructions 23.5, without B's loads 24.9).
//
// A x is held in 32 bits and enters the second product as two bf16 numbers, which together have 16 bits of it: its
// rounding to one would be as large as the output's own.
#include <math.h>

#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "common.cuh"
#include "tc_common.cuh"
#include "waiter.cuh"

namespace cg = cooperative_groups;

namespace q3 {
int check_device();

namespace {

__device__ unsigned g_dev_error;

constexpr int LA_MAX_ROWS = 1 << 16;
constexpr int LA_MAX_ADAPTERS = 8192;
constexpr int LA_MAX_RANK = 128;
constexpr int LA_MAX_SLICES = 3;
constexpr int LA_MAX_CLUSTER = 8;

// A tile's record: the adapter (-1: rows without one), how many rows, two unused, and the rows.
constexpr int LA_HEAD = 4;

// Rows of a tile: of a step of few rows as many as one matrix instruction takes; more share an adapter's weights in
// longer tiles. 2079 rows, 8 adapters of rank 64, q, k and v: 37 us with tiles of 32, 47 with tiles of 64, which halve the weights' traffic but
// not the products, and fill fewer SMs.
__host__ __device__ constexpr int lora_tile_rows(int n_rows) { return n_rows <= 128 ? 16 : 32; }

struct LoraPlanLayout {
    int max_tiles, record;  // record: ints of a tile
    size_t bytes;           // the number of tiles, then the records
};
__host__ __device__ inline LoraPlanLayout lora_plan_layout(int n_rows, int n_adapters) {
    LoraPlanLayout l = {};
    const int kinds = n_rows < n_adapters + 1 ? n_rows : n_adapters + 1, tile_rows = lora_tile_rows(n_rows);
    l.max_tiles = kinds + n_rows / tile_rows;
    l.record = LA_HEAD + tile_rows;
    l.bytes = 16 + (size_t)l.max_tiles * l.record * 4;
    return l;
}

// ------------------------------------------------------------------ plan

constexpr int LP_THREADS = 1024;
constexpr int LP_COUNTERS = 49152;  // 192 KB of them

// Parts that the rows are cut into: a warp each, as far as there are rows for them and room for their counters.
__host__ __device__ inline int lora_plan_parts(int n_rows, int n_adapters) {
    const int rows = (n_rows + 31) / 32, room = LP_COUNTERS / (n_adapters + 1) - 1;
    return rows < room ? (rows < 32 ? rows : 32) : room < 32 ? room : 32;
}

// A stable sort: counts for each part of the rows and adapter, running sums over both, and each part placed by its warp.
// A chain of loads and, in a part, of steps of 32 rows; with one part, whose rows all warps went through for adapters of their
// own, 2079 rows took 20 us and 65536 559. Now 2.9 us for 32 rows, 4.7 for 2079 of 8 adapters, 40 for 65536 (199 if of 8192); once
// per step.
__global__ void __launch_bounds__(LP_THREADS, 1) lora_plan_kernel(char *plan, int n_rows, int n_adapters, const int *index) {
    extern __shared__ int la_smem_plan[];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, tile_rows = lora_tile_rows(n_rows), kinds = n_adapters + 1;
    const int parts = lora_plan_parts(n_rows, n_adapters), part_rows = (n_rows + 32 * parts - 1) / (32 * parts) * 32;
    int *next = la_smem_plan;           // [parts][kinds]: a part's rows of each adapter, then where the next of them goes; the last kind: without one
    int *first = next + parts * kinds;  // [kinds]: its first tile
    int *sums = first + kinds;          // [32]
    const LoraPlanLayout l = lora_plan_layout(n_rows, n_adapters);
    int *tiles = reinterpret_cast<int *>(plan + 16);
    for (int i = tid; i < parts * kinds; i += LP_THREADS) next[i] = 0;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    auto kind = [&](int row) {
        const int i = index[row];
        return i < 0 || i >= n_adapters ? n_adapters : i;
    };
    for (int row = tid; row < n_rows; row += LP_THREADS) {
        if (index[row] >= n_adapters) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
        atomicAdd(&next[row / part_rows * kinds + kind(row)], 1);
    }
    __syncthreads();
    // running sums: of an adapter's rows over the parts, of tiles over the adapters, 1024 of them at a time
    int tile0 = 0;
    for (int i0 = 0; i0 < kinds; i0 += LP_THREADS) {
        const int i = i0 + tid;
        int n = 0;
        for (int p = 0; i < kinds && p < parts; p++) {
            const int c = next[p * kinds + i];
            next[p * kinds + i] = n;
            n += c;
        }
        const int t = (n + tile_rows - 1) / tile_rows;
        int run = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, run, o);
            run += lane >= o ? y : 0;
        }
        if (lane == 31) sums[warp] = run;
        __syncthreads();
        int all = 0, before = 0;
        for (int w = 0; w < 32; w++) {
            before += w < warp ? sums[w] : 0;
            all += sums[w];
        }
        const int tile = tile0 + before + run - t;
        if (i < kinds) first[i] = tile;
        for (int k = 0; k < t; k++) *reinterpret_cast<int4 *>(tiles + (tile + k) * l.record) = make_int4(i < n_adapters ? i : -1, min(tile_rows, n - k * tile_rows), 0, 0);
        tile0 += all;
        __syncthreads();
    }
    if (tid == 0) *reinterpret_cast<int *>(plan) = tile0;
    if (warp >= parts) return;
    next += warp * kinds;
    const int r1 = min(n_rows, (warp + 1) * part_rows), shift = __ffs(tile_rows) - 1;
    int k_next = warp * part_rows + lane < r1 ? kind(warp * part_rows + lane) : -1;
    for (int r0 = warp * part_rows; r0 < r1; r0 += 32) {
        const int row = r0 + lane, k = k_next;
        k_next = row + 32 < r1 ? kind(row + 32) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, k);
        if (k >= 0) {
            const int at = next[k] + __popc(peers & ((1u << lane) - 1));
            tiles[(first[k] + (at >> shift)) * l.record + LA_HEAD + (at & (tile_rows - 1))] = row;
        }
        __syncwarp();
        if (k >= 0 && lane == __ffs(peers) - 1) next[k] += __popc(peers);
        __syncwarp();
    }
}

// ------------------------------------------------------------------ products

struct LoraSlice {
    bf16 *out;
    const bf16 *base, *a, *b;
    long long out_stride, base_stride;
    int n;
};
struct LoraArgs {
    LoraSlice slice[LA_MAX_SLICES];
    const bf16 *x;
    long long x_stride;
    const int *ranks;
    const float *scale;
    const char *plan;
    bf16 *act;  // gate_up
    long long act_stride;
    int n_slices, k, rank, n_rows, n_adapters;
    int wide;   // columns of A x in shared memory: each slice's rank rounded up to 32
    int pitch;  // and of its bf16 parts: an odd number of 64 bytes, so that the two rows that eight lanes read lie in other banks
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// whole 16-byte lines
__device__ __forceinline__ void prefetch_l2(const void *p, int bytes) { asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory"); }
// 16 bytes to shared memory, zeros if not `in`
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}

// Whether any of eight numbers is infinite or NaN: 0 times it is not 0.
__device__ __forceinline__ bool not_finite(const uint4 &v) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v), zero = __floats2bfloat162_rn(0.0f, 0.0f);
    __nv_bfloat162 z = zero;
#pragma unroll
    for (int e = 0; e < 4; e++) z = __hfma2(h[e], zero, z);
    return *reinterpret_cast<const uint32_t *>(&z) & 0x7fff7fffu;
}

// Which slice an eight-column tile of A x belongs to (each has tiles_each), and where it begins.
__device__ __forceinline__ int slice_of(int nt, int tiles_each) { return nt < tiles_each ? 0 : nt < 2 * tiles_each ? 1 : 2; }

// One CTA an SM: all of it is chains of loads, which sixteen warps overlap.
constexpr int LA_THREADS = 512;
constexpr int LA_WARPS = LA_THREADS / 32;

// A x of a short tile of up to 48 columns, this CTA's part of k: each warp a part of that for all columns, operands from global memory straight
// into registers, then the warps' parts added up in their order.
// PASS: its eight-column tiles, whose sums stay in registers; the kernel is built for 2, 4 and 6, and takes the least that holds
// all: code for more that is stepped over costs 64 rows through the down projection 12.7 -> 15.3 us. Wider ones take the long tiles'
// way: 32 rows through q, k and v of rank 32 9.5 us where this way takes 11.7, 4 rows of rank 64 11.3 and 18.0.
// meanwhile() runs once, while the first loads are on their way.
template <int PASS, typename F>
__device__ __forceinline__ void shrink_short(const LoraArgs &a, float *h, float *part, const int *row_s, int rows, int adapter, int r, int C, int rank_c,
                                             F meanwhile) {
    constexpr int COLS = 8 * PASS;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4, each = a.wide / a.n_slices;
    const int steps = (a.k + 31) / 32, parts = C * LA_WARPS, p = rank_c * LA_WARPS + warp;
    const int s0 = (int)((long long)steps * p / parts), s1 = (int)((long long)steps * (p + 1) / parts);
    const bf16 *x0 = a.x + row_s[g] * a.x_stride, *x1 = a.x + row_s[g + 8] * a.x_stride;
    const int tiles_each = (r + 7) / 8, n_tiles = tiles_each * a.n_slices;
    float acc[PASS][4] = {};
    const bf16 *w[PASS];
#pragma unroll
    for (int j = 0; j < PASS; j++) {
        const int nt = j, sl = slice_of(nt, tiles_each), row = (nt - sl * tiles_each) * 8 + g;
        w[j] = nt < n_tiles && row < r ? a.slice[sl].a + ((long long)adapter * a.rank + row) * a.k : nullptr;
    }
    uint4 u, v, b[PASS];
    auto load = [&](int s) {
        const int k = 32 * s + 8 * t;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const bool in = s < s1 && k < a.k;
        u = in ? __ldg(reinterpret_cast<const uint4 *>(x0 + k)) : zero;
        v = in ? __ldg(reinterpret_cast<const uint4 *>(x1 + k)) : zero;
#pragma unroll
        for (int j = 0; j < PASS; j++) b[j] = in && w[j] ? __ldg(reinterpret_cast<const uint4 *>(w[j] + k)) : zero;
    };
    load(s0);
    meanwhile();
#pragma unroll 1
    for (int s = s0; s < s1; s++) {
        const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
        for (int j = 0; j < PASS; j++)
            if (j < n_tiles) {
                mma(acc[j], a0, b[j].x, b[j].y);
                mma(acc[j], a1, b[j].z, b[j].w);
            }
        load(s + 1);
    }
    float *own = part + warp * 16 * COLS;
#pragma unroll
    for (int j = 0; j < PASS; j++) {
        *reinterpret_cast<float2 *>(own + g * COLS + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2 *>(own + (g + 8) * COLS + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = tid; i < rows * COLS; i += LA_THREADS) {
        const int row = i / COLS, col = i % COLS, nt = col / 8;
        if (nt >= n_tiles) continue;
        float f[LA_WARPS];
#pragma unroll
        for (int q = 0; q < LA_WARPS; q++) f[q] = part[(q * 16 + row) * COLS + col];
#pragma unroll
        for (int q = 1; q < LA_WARPS; q++) f[0] += f[q];
        const int sl = slice_of(nt, tiles_each);
        h[row * a.wide + sl * each + (nt - sl * tiles_each) * 8 + col % 8] = f[0];
    }
    __syncthreads();
}

// A x of a long tile, or a wide one, this CTA's part of k: x and A come through shared memory in stages of 64 elements of k (a row is 128 bytes,
// its 16-byte lines exchanged by the row's lowest bits, so that the eight rows of a matrix lie in different banks), so
// that each is read once. Twelve warps have a pair of eight-column tiles each, for all rows. One asks for A, up to 64 rows a copy; two
// copy the rows of x, which may lie anywhere. From registers alone, with each warp reading all of A for its rows, this part took
// 2079 rows of rank 64 three times as long; with 16-byte copies for A, too, their number was the limit (44.6 us in all, then 36.7).
constexpr int LA_STAGES = 4, LA_KC = 64, LA_COLS = 192;  // columns at a time
__host__ __device__ constexpr int lora_stage_bytes(int rows) { return (rows + LA_COLS) * LA_KC * 2; }
constexpr int LA_READERS = LA_COLS / 16;  // warps; then one for A
constexpr int LA_X_THREADS = 64;

struct LoraMaps {
    CUtensorMap a[LA_MAX_SLICES];  // of long tiles: [n_adapters * rank][k], boxes of `box` rows and 64 elements
    int box;                       // a power of two up to 64 that divides rank
};

// ring: 1024-byte aligned; bars: full, then empty, of each stage; down: zero, set when a wait has given up
template <int ROWS, typename F>
__device__ __forceinline__ void shrink_long(const LoraArgs &a, const LoraMaps &maps, float *h, unsigned char *ring, uint64_t *bars, int *down,
                                            const int *row_s, int rows, int adapter, int r, int C, int rank_c, F meanwhile) {
    constexpr int MT = ROWS / 16, LA_STAGE_BYTES = lora_stage_bytes(ROWS);
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, each = a.wide / a.n_slices;
    const int k64 = (a.k + LA_KC - 1) / LA_KC, c0 = (int)((long long)k64 * rank_c / C), chunks = (int)((long long)k64 * (rank_c + 1) / C) - c0;
    const int tiles_each = (r + maps.box - 1) / maps.box * (maps.box / 8), n_tiles = tiles_each * a.n_slices;  // whole boxes
    const uint32_t ring_at = smem_u32(ring);
    Waiter wait(&g_dev_error, down);
    int it = 0;  // chunks so far
    // Readers that gave up release no stages, so that the loaders starve and give up in turn.
    if (warp == LA_READERS) {
#pragma unroll 1
        for (int n0 = 0; n0 < n_tiles; n0 += LA_COLS / 8) {
            const int tiles = min(LA_COLS / 8, n_tiles - n0), nt = n0 + lane * (maps.box / 8), sl = slice_of(nt, tiles_each);
            const int y = adapter * a.rank + 8 * (nt - sl * tiles_each);
#pragma unroll 1
            for (int c = 0; c < chunks; c++, it++) {
                const int st = it % LA_STAGES;
                if (it >= LA_STAGES) wait(bars + LA_STAGES + st, (it / LA_STAGES - 1) & 1);
                if (wait.stopped()) continue;
                if (lane == 0) mbar_arrive_expect_tx(bars + st, tiles * 8 * LA_KC * 2);
                __syncwarp();
                if (nt < n0 + tiles) tma_load_2d(ring + st * LA_STAGE_BYTES + (ROWS + maps.box * lane) * LA_KC * 2, &maps.a[sl], (c0 + c) * LA_KC, y, bars + st);
            }
        }
    } else if (warp > LA_READERS) {
        const int own = tid - 32 * (LA_READERS + 1), row0 = own / 8, q = own % 8;
        if (own < LA_X_THREADS) {
            constexpr int STEP = LA_X_THREADS / 8;
            const bf16 *from[ROWS / STEP];
#pragma unroll
            for (int j = 0; j < ROWS / STEP; j++) from[j] = a.x + row_s[row0 + j * STEP] * a.x_stride + 8 * q;
#pragma unroll 1
            for (int n0 = 0; n0 < n_tiles; n0 += LA_COLS / 8)
#pragma unroll 1
                for (int c = 0; c < chunks; c++, it++) {
                    const int st = it % LA_STAGES, k = (c0 + c) * LA_KC;
                    if (it >= LA_STAGES) wait(bars + LA_STAGES + st, (it / LA_STAGES - 1) & 1);
                    if (wait.dead) continue;
#pragma unroll
                    for (int j = 0; j < ROWS / STEP; j++) {
                        const int row = row0 + j * STEP;
                        const bool in = row < rows && k + 8 * q < a.k;
                        copy16(ring_at + st * LA_STAGE_BYTES + row * (LA_KC * 2) + ((q ^ (row & 7)) << 4), in ? from[j] + k : a.x, in);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bars + st)) : "memory");
                }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            meanwhile();
        }
    } else {
#pragma unroll 1
        for (int n0 = 0; n0 < n_tiles; n0 += LA_COLS / 8) {
            const int cols = min(LA_COLS, (n_tiles - n0) * 8);
            float acc[MT][2][4] = {};
#pragma unroll 1
            for (int c = 0; c < chunks; c++, it++) {
                const int st = it % LA_STAGES;
                wait(bars + st, it / LA_STAGES & 1);
                if (16 * warp < cols) {
                    const uint32_t x_at = ring_at + st * LA_STAGE_BYTES, w_at = x_at + ROWS * LA_KC * 2;
#pragma unroll
                    for (int s = 0; s < LA_KC / 16; s++) {
                        uint32_t am[MT][4], bm[4];
#pragma unroll
                        for (int m = 0; m < MT; m++) {
                            const int row = m * 16 + lane % 16, q = 2 * s + lane / 16;
                            load_matrices(am[m], x_at + row * (LA_KC * 2) + ((q ^ (row & 7)) << 4));
                        }
                        const int row = warp * 16 + lane / 16 * 8 + lane % 8, q = 2 * s + lane / 8 % 2;
                        load_matrices(bm, w_at + row * (LA_KC * 2) + ((q ^ (row & 7)) << 4));
#pragma unroll
                        for (int m = 0; m < MT; m++) {
                            mma(acc[m][0], am[m], bm[0], bm[1]);
                            mma(acc[m][1], am[m], bm[2], bm[3]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0 && !wait.dead) mbar_arrive(bars + LA_STAGES + st);
            }
            // h may be where the ring is, if this is the only pass
            asm volatile("bar.sync 1, %0;" ::"n"(32 * LA_READERS) : "memory");
            const int g = lane / 4, t = lane % 4;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int nt = n0 + 2 * warp + j, sl = slice_of(nt, tiles_each);
                if (8 * (nt - n0) < cols) {
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        float *to = h + (m * 16 + g) * a.wide + sl * each + (nt - sl * tiles_each) * 8 + 2 * t;
                        *reinterpret_cast<float2 *>(to) = make_float2(acc[m][j][0], acc[m][j][1]);
                        *reinterpret_cast<float2 *>(to + 8 * a.wide) = make_float2(acc[m][j][2], acc[m][j][3]);
                    }
                }
            }
        }
    }
    __syncthreads();
    if (*reinterpret_cast<volatile int *>(down)) settle();  // copies may still be on their way
    __syncthreads();
}

// silu(g) u. The divisor is from 1 to 2 for either sign, since __fdividef gives 0 for one past 2^126. (the compiler's own divide, with
// a branch for rare operands, costs the kernel registers and twice its time)
__device__ __forceinline__ float silu_times(float g, float u) {
    const float e = __expf(-fabsf(g));
    return __fdividef(g < 0.0f ? g * e : g, 1.0f + e) * u;
}

// A column of a row's sum in fp32, A x whole again: h, and its lower parts `lower` further on; b: the column's row of B.
__device__ __forceinline__ float column_again(const bf16 *h, int lower, const bf16 *b, int r) {
    float sum = 0.0f;
#pragma unroll 1
    for (int e0 = 0; e0 < r; e0 += 8) {
        const bf16x8 x = lds128(h + e0), y = lds128(h + lower + e0), w = ldg128(b + e0);
        const bf16 *xe = reinterpret_cast<const bf16 *>(&x), *ye = reinterpret_cast<const bf16 *>(&y), *we = reinterpret_cast<const bf16 *>(&w);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e0 + e < r) sum = fmaf(__bfloat162float(xe[e]) + __bfloat162float(ye[e]), __bfloat162float(we[e]), sum);
    }
    return sum;
}
__device__ __forceinline__ bool has_nan(const bf16 *h, int r) {
    bool any = false;
    for (int e = 0; e < r; e++) any |= __hisnan(h[e]);
    return any;
}

// GATE_UP: slices 0 and 1 are gate and up, and what is written is silu(gate) * up. PASS: 0 for a first product through shared memory.
template <int ROWS, bool GATE_UP, int PASS>
__global__ void __launch_bounds__(LA_THREADS, 1) lora_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraMaps maps) {
    constexpr int THREADS = LA_THREADS, WARPS = LA_WARPS, MT = ROWS == 16 || GATE_UP ? 1 : 2;  // MT: 16-row tiles of a warp in the second product
    extern __shared__ __align__(16) unsigned char la_smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank_c = cluster.block_rank(), tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int g = lane / 4, t = lane % 4;
    const int wide = a.wide, pitch = a.pitch, each = wide / a.n_slices;
    uint64_t *bars = reinterpret_cast<uint64_t *>(la_smem);                 // [2 LA_STAGES]
    int *row_s = reinterpret_cast<int *>(bars + 2 * LA_STAGES), *head_s = row_s + ROWS;  // [ROWS], [LA_HEAD]
    float *h = reinterpret_cast<float *>(head_s + LA_HEAD);                 // [ROWS][wide]: this CTA's part of A x
    // [ROWS][pitch]: A x, scaled, upper and lower bits; before that the first product's buffers, those of a long tile over h,
    // too, if that is written once
    unsigned char *rest = reinterpret_cast<unsigned char *>(h + ROWS * wide);
    bf16 *hi = reinterpret_cast<bf16 *>(rest), *lo = hi + ROWS * pitch;

    if (PASS == 0 && tid == 0) {
        for (int st = 0; st < LA_STAGES; st++) {
            mbar_init(bars + st, 1 + LA_X_THREADS);
            mbar_init(bars + LA_STAGES + st, LA_READERS);
        }
        fence_barrier_init();
    }
    pdl_trigger();
    pdl_wait();
    const int tile = blockIdx.x / C;
    const int *record = reinterpret_cast<const int *>(a.plan + 16) + tile * (LA_HEAD + ROWS);
    const int n_plan = *reinterpret_cast<const int *>(a.plan);
    const int mine = tid < LA_HEAD + ROWS ? record[tid] : 0;  // past the rows of a tile, or the tiles: anything
    if (tile >= n_plan) return;  // the whole cluster
    if (tid < LA_HEAD) head_s[tid] = tid < 2 ? mine : 0;
    __syncthreads();
    const int adapter = head_s[0], rows = head_s[1];
    if (GATE_UP && adapter < 0) return;  // the whole cluster: act is right already
    if (tid >= LA_HEAD && tid < LA_HEAD + rows) row_s[tid - LA_HEAD] = mine;
    if (tid >= LA_HEAD + rows && tid < LA_HEAD + ROWS) row_s[tid - LA_HEAD] = record[LA_HEAD + rows - 1];  // read there, never written
    int r = 0;
    float scale = 1.0f;
    if (adapter >= 0) {
        r = a.ranks ? max(0, min(a.ranks[adapter], a.rank)) : a.rank;
        if (a.scale) scale = a.scale[adapter];
    }
    __syncthreads();

    if (!GATE_UP && r == 0) {  // nothing to add; in place there is nothing to do at all
        bool copies = false;
        for (int sl = 0; sl < a.n_slices; sl++) copies |= a.slice[sl].out != a.slice[sl].base;
        if (!copies) return;  // the whole cluster
    }
    int units = 0;
    for (int sl = 0; sl < (GATE_UP ? 1 : a.n_slices); sl++) units += (a.slice[sl].n + 31) / 32;
    bool waiting = false;
    if (r > 0) {
        if constexpr (PASS > 0) {
            auto ask = [&] {  // for what the second product will read
                for (int u = rank_c * WARPS + warp; u < units; u += C * WARPS) {
                    int sl = 0, n0 = u;
                    if (!GATE_UP)
                        while (n0 >= (a.slice[sl].n + 31) / 32) n0 -= (a.slice[sl++].n + 31) / 32;
                    n0 = 32 * n0 + lane;
                    for (int pr = 0; pr < (GATE_UP ? 2 : 1); pr++)
                        if (n0 < a.slice[sl].n) prefetch_l2(a.slice[sl + pr].b + ((long long)adapter * a.slice[sl].n + n0) * a.rank);
                }
            };
            shrink_short<PASS>(a, h, reinterpret_cast<float *>(rest), row_s, rows, adapter, r, C, rank_c, ask);
        } else {
            // A warp has the L2 fetch the bases while the others multiply, a lane a row, 512 columns at a time: where they are not in
            // it yet, 2079 rows of rank 64 take 35.0 us instead of 36.8, where they are, 31.8 and 31.6. The taps of a gate and up are.
            auto ask = [&] {
                if (GATE_UP || lane >= rows) return;
                for (int i = rank_c * WARPS; i < units; i += C * WARPS) {
                    int q0 = i, q1 = min(units, i + WARPS);  // units of 32 columns, in the slices
                    for (int sl = 0; sl < a.n_slices; sl++) {
                        const int n = a.slice[sl].n, n0 = 32 * q0, n1 = min(32 * q1, n);
                        if (n0 < n1) prefetch_l2(a.slice[sl].base + row_s[lane] * a.slice[sl].base_stride + n0, 2 * (n1 - n0));
                        q0 = max(0, q0 - (n + 31) / 32);
                        q1 -= (n + 31) / 32;
                    }
                }
            };
            shrink_long<ROWS>(a, maps, h, align_shared<1024>(wide <= LA_COLS ? reinterpret_cast<unsigned char *>(h) : rest), bars, head_s + LA_HEAD - 1, row_s, rows, adapter, r, C, rank_c, ask);
        }
        // the CTAs' parts, in their order. Few: each CTA adds up all of them; more: each some of the columns for all.
        if (C > 1) cluster.sync();
        const int octets = rows * wide / 8;
        const bool all = octets * C <= 512;  // remote shared memory gives some 9 bytes a cycle: 2000 cycles
        const int q0 = all ? 0 : (int)((long long)octets * rank_c / C), q1 = all ? octets : (int)((long long)octets * (rank_c + 1) / C);
        for (int q = q0 + tid; q < q1; q += THREADS) {
            const int row = 8 * q / wide, col = 8 * q % wide, left = r - col % each;  // of the adapter's rank from here
            float v[8] = {};
            constexpr int AT_ONCE = ROWS == 16 ? LA_MAX_CLUSTER : 4;
            if (left > 0) {
#pragma unroll 1
                for (int c0 = 0; c0 < C; c0 += AT_ONCE) {
                    float4 f[AT_ONCE][2];  // all loads before the first sum
#pragma unroll
                    for (int c = 0; c < AT_ONCE; c++)
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            f[c][half] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (c0 + c < C) f[c][half] = *reinterpret_cast<const float4 *>((C > 1 ? cluster.map_shared_rank(h, c0 + c) : h) + 8 * q + 4 * half);
                        }
#pragma unroll
                    for (int c = 0; c < AT_ONCE; c++)
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            v[4 * half] += f[c][half].x;
                            v[4 * half + 1] += f[c][half].y;
                            v[4 * half + 2] += f[c][half].z;
                            v[4 * half + 3] += f[c][half].w;
                        }
                }
            }
            uint32_t up[4], low[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float s[2], b[2], l[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    s[k] = 2 * e + k < left ? scale * v[2 * e + k] : 0.0f;
                    const bool finite = isfinite(s[k]);
                    b[k] = round_bf16(s[k]);
                    if (finite) b[k] = fminf(fmaxf(b[k], -0x1.fep127f), 0x1.fep127f);  // the largest bf16 number
                    l[k] = finite ? s[k] - b[k] : 0.0f;
                }
                up[e] = pack2(b[0], b[1]);
                low[e] = pack2(l[0], l[1]);
            }
            const int at = row * pitch + col;
            for (int c = all ? rank_c : 0; c < (all ? rank_c + 1 : C); c++) {
                *reinterpret_cast<uint4 *>((C > 1 ? cluster.map_shared_rank(hi, c) : hi) + at) = make_uint4(up[0], up[1], up[2], up[3]);
                *reinterpret_cast<uint4 *>((C > 1 ? cluster.map_shared_rank(lo, c) : lo) + at) = make_uint4(low[0], low[1], low[2], low[3]);
            }
        }
        if (all || C == 1) {
            __syncthreads();
            if (C > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // has read the others' parts
            waiting = C > 1;
        } else {
            cluster.sync();
        }
    }

    // ---- out: units of 32 columns, and of those MT row tiles, a warp each. While one step of 32 of the rank is multiplied, the
    // next one's B is on its way, and after a unit the next unit's base. What lies past the columns or rows is loaded from the
    // last ones and not written.
    constexpr int PAIR = GATE_UP ? 2 : 1;
    const int k_steps = (r + 31) / 32, two = rows > 16 * MT, items = units << two;
    const int end0 = (a.slice[0].n + 31) / 32, end1 = end0 + (a.slice[1].n + 31) / 32;
    struct Unit {
        int sl, n0, m0;
    };
    auto unit = [&](int i) {
        const int at = i >> two, sl = GATE_UP ? 0 : (at >= end0) + (at >= end1);
        return Unit{sl, 32 * (at - (sl == 0 ? 0 : sl == 1 ? end0 : end1)), two ? i % 2 * MT : 0};
    };
    uint4 b[4], base[PAIR][MT][2];
    auto load_b = [&](const Unit &u, int pr, int s) {
        const LoraSlice &c = a.slice[u.sl + pr];
        const int k = 32 * s + 8 * t;
        const bf16 *from = c.b + (long long)adapter * c.n * a.rank + (k < r ? k : 0);
#pragma unroll
        for (int j = 0; j < 4; j++)
            b[j] = __ldg(reinterpret_cast<const uint4 *>(from + (long long)min(u.n0 + 8 * (g / 2) + 2 * j + g % 2, c.n - 1) * a.rank));
    };
    auto load_base = [&](const Unit &u) {  // a lane has eight neighbouring columns of rows g and g + 8 of each tile
#pragma unroll
        for (int pr = 0; pr < PAIR; pr++) {
            const LoraSlice &c = a.slice[u.sl + pr];
            const bf16 *from = c.base + min(u.n0 + 8 * t, c.n - 8);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int q = 0; q < 2; q++) base[pr][m][q] = *reinterpret_cast<const uint4 *>(from + row_s[(u.m0 + m) * 16 + g + 8 * q] * c.base_stride);
        }
    };
    // The first unit in which a result that this lane has of a row is not finite: from there on it writes nothing of that row, and takes
    // it again at the end.
    int i = rank_c * WARPS + warp, again[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++) again[m][0] = again[m][1] = items;
    Unit u = unit(min(i, items - 1));
    if (i < items) {
        if (r > 0) load_b(u, 0, 0);
        load_base(u);
    }
#pragma unroll 1
    for (; i < items; i += C * WARPS) {
        const Unit next = unit(min(i + C * WARPS, items - 1));
        float acc[PAIR][MT][4][4] = {};
#pragma unroll
        for (int pr = 0; pr < PAIR; pr++)
#pragma unroll 1
            for (int s = 0; s < k_steps; s++) {
                uint4 now[4] = {b[0], b[1], b[2], b[3]};
                const int left = r - (32 * s + 8 * t);
                if (r - 32 * s < 32) {  // what is past the adapter's rank may be anything
                    auto keep = [&](int e) { return left > e + 1 ? 0xffffffffu : left > e ? 0xffffu : 0u; };
#pragma unroll
                    for (int j = 0; j < 4; j++) now[j] = make_uint4(now[j].x & keep(0), now[j].y & keep(2), now[j].z & keep(4), now[j].w & keep(6));
                }
                if (s + 1 < k_steps) load_b(u, pr, s + 1);
                else if (pr + 1 < PAIR) load_b(u, pr + 1, 0);
                else load_b(next, 0, 0);
                const int at = (u.m0 * 16 + g) * pitch + (u.sl + pr) * each + 32 * s + 8 * t;
#pragma unroll
                for (int m = 0; m < MT; m++) {
#pragma unroll
                    for (int part = 0; part < 2; part++) {
                        const bf16 *from = (part ? lo : hi) + at + m * 16 * pitch;
                        const uint4 v = *reinterpret_cast<const uint4 *>(from), w = *reinterpret_cast<const uint4 *>(from + 8 * pitch);
                        const uint32_t a0[4] = {v.x, w.x, v.y, w.y}, a1[4] = {v.z, w.z, v.w, w.w};
#pragma unroll
                        for (int j = 0; j < 4; j++) mma(acc[pr][m][j], a0, now[j].x, now[j].y);
#pragma unroll
                        for (int j = 0; j < 4; j++) mma(acc[pr][m][j], a1, now[j].z, now[j].w);
                    }
                }
            }
        const int col = u.n0 + 8 * t;
        const bool inside = col < a.slice[u.sl].n;
        bf16 *to = (GATE_UP ? a.act : a.slice[u.sl].out) + col;
        const long long to_stride = GATE_UP ? a.act_stride : a.slice[u.sl].out_stride;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const int at = (u.m0 + m) * 16 + g + 8 * q;
                uint32_t y[4];
                const __nv_bfloat162 *p0 = reinterpret_cast<const __nv_bfloat162 *>(&base[0][m][q]), *p1 = reinterpret_cast<const __nv_bfloat162 *>(&base[PAIR - 1][m][q]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = __bfloat1622float2(p0[j]);
                    const float v0 = f.x + acc[0][m][j][2 * q], v1 = f.y + acc[0][m][j][2 * q + 1];
                    if constexpr (GATE_UP) {
                        const float2 fu = __bfloat1622float2(p1[j]);
                        const float u0 = fu.x + acc[1][m][j][2 * q], u1 = fu.y + acc[1][m][j][2 * q + 1];
                        y[j] = pack2(silu_times(v0, u0), silu_times(v1, u1));
                    } else {
                        y[j] = pack2(v0, v1);
                    }
                }
                const uint4 out = r > 0 || GATE_UP ? make_uint4(y[0], y[1], y[2], y[3]) : base[0][m][q];
                if (inside && at < rows) {
                    if (r > 0 && not_finite(out)) again[m][q] = min(again[m][q], i);
                    if (i < again[m][q]) *reinterpret_cast<uint4 *>(to + row_s[at] * to_stride) = out;
                }
            }
        u = next;
        if (i + C * WARPS < items) load_base(u);
    }
    // What two parts of A x make of an infinite weight, or of one whose products overflow, need not be what their sum does (0 inf,
    // inf - inf). The check costs 2079 rows 0.9 us of 36.3, one row 0.2 of 8.4; calls inside the loop took 3 and 0.2. 2079 rows of NaN take
    // 86 us, with an infinite base in each row 410.
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll 1
            for (i = again[m][q]; i < items; i += C * WARPS) {
                u = unit(i);
                const int at = (u.m0 + m) * 16 + g + 8 * q, col0 = u.n0 + 8 * t;
                if (at >= rows || col0 >= a.slice[u.sl].n) continue;
                bf16 *to = (GATE_UP ? a.act : a.slice[u.sl].out) + row_s[at] * (GATE_UP ? a.act_stride : a.slice[u.sl].out_stride) + col0;
                const bf16 *x = hi + at * pitch + u.sl * each;
                if (has_nan(x, r) || (GATE_UP && has_nan(x + each, r))) {  // so is all of it
                    *reinterpret_cast<uint4 *>(to) = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
                    continue;
                }
#pragma unroll 1
                for (int col = 0; col < 8; col++) {
                    float v[PAIR];
#pragma unroll
                    for (int pr = 0; pr < PAIR; pr++) {
                        const LoraSlice &c = a.slice[u.sl + pr];
                        v[pr] = __bfloat162float(c.base[row_s[at] * c.base_stride + col0 + col]) +
                                column_again(x + pr * each, ROWS * pitch, c.b + ((long long)adapter * c.n + col0 + col) * a.rank, r);
                    }
                    to[col] = __float2bfloat16(GATE_UP ? silu_times(v[0], v[PAIR - 1]) : v[0]);
                }
            }
    if (waiting) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // the others have read this one's part
}

int wide_of(int n_slices, int rank) { return n_slices * ((rank + 31) / 32 * 32); }

int pitch_of(int wide) { return wide / 32 % 2 ? wide : wide + 32; }

template <int ROWS, int PASS>
size_t lora_smem(int wide) {
    const size_t h = (size_t)ROWS * wide * 4, both = h + 2 * (size_t)ROWS * pitch_of(wide) * 2;
    const size_t first = PASS > 0 ? h + (size_t)LA_WARPS * 16 * 8 * PASS * 4
                                    : (wide <= LA_COLS ? 0 : h) + 1024 + (size_t)LA_STAGES * lora_stage_bytes(ROWS);
    return 2 * LA_STAGES * 8 + (size_t)(ROWS + LA_HEAD) * 4 + std::max(first, both);
}

// Whether two matrices of as many rows share any element.
bool overlap(const void *a, long long a_stride, int a_width, const void *b, long long b_stride, int b_width, int rows) {
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    const uintptr_t a1 = a0 + 2 * ((rows - 1) * a_stride + a_width), b1 = b0 + 2 * ((rows - 1) * b_stride + b_width);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a_stride != b_stride) return true;
    // column slices of one buffer
    const long long s = 2 * a_stride;
    long long d = (long long)(b0 - a0) % s;
    if (d < 0) d += s;
    return d < 2LL * a_width || d + 2LL * b_width > s;
}

// Clusters of c CTAs that the device holds at once, a CTA an SM: fewer than its SMs would make, since a cluster stays within one of its parts
// (148 SMs: 148, 74, 45, 33, 26, 22, 15, 15).
int clusters_at_once(int c) {
    static std::atomic<int> known[64][LA_MAX_CLUSTER + 1];
    int d = 0;
    cudaGetDevice(&d);
    std::atomic<int> &n = known[d < 0 || d >= 64 ? 0 : d][c];
    if (n.load(std::memory_order_relaxed) == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(c * num_sms()));
        cfg.blockDim = dim3(LA_THREADS);
        cfg.dynamicSmemBytes = 48 * 1024;
        cudaLaunchAttribute shape;
        shape.id = cudaLaunchAttributeClusterDimension;
        shape.val.clusterDim.x = c;
        shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
        cfg.attrs = &shape;
        cfg.numAttrs = 1;
        int held = 0;
        if (cudaOccupancyMaxActiveClusters(&held, lora_kernel<32, false, 0>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            held = 0;
        }
        n.store(held > 0 ? held : num_sms() / c, std::memory_order_relaxed);
    }
    return n.load(std::memory_order_relaxed);
}

template <int ROWS, bool GATE_UP, int PASS>
int launch_lora(const LoraArgs &args, int tiles, cudaStream_t s) {
    auto kernel = lora_kernel<ROWS, GATE_UP, PASS>;
    const size_t smem = lora_smem<ROWS, PASS>(args.wide);
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    // CTAs of a tile: as many as the SMs hold at once for the tiles there may be. Of a short step as many as if each row took an adapter at
    // random (64 rows, 64 adapters, 41 tiles: clusters of 2 take 16.1 us, of 3 12.9, of 4 21.1; 100 rows, 30 adapters of rank 64, 30
    // tiles: of 3 18.2, of 4 15.2, of 5 25.3). A long step is mostly a chunk of one prompt: its tiles, and those of 32 rows of other
    // adapters (831 rows, 53 adapters of rank 32: clusters of 1 take 41 us, of 2 25, of 4 16 if all rows are of one adapter, 30 if each is of
    // any; 300 rows, 64 adapters: of 2 24, of 3 19 with such a chunk and 33 without).
    const double kinds = args.n_adapters + 1, rows = args.n_rows, each = rows / kinds;
    const double tiles_of = ROWS == 16 ? kinds * (1.0 - exp(-each)) * std::max(1.0, each / ROWS + 0.5)
                                       : args.n_adapters * (1.0 - exp(-32.0 / kinds)) + (rows - 32.0) / ROWS;
    int cluster = LA_MAX_CLUSTER;
    while (cluster > 1 && clusters_at_once(cluster) < tiles_of) cluster--;
    LoraMaps maps = {};
    maps.box = std::min(64, args.rank & -args.rank);
    if (PASS == 0)
        for (int i = 0; i < args.n_slices; i++)
            if (!make_map_strided(&maps.a[i], args.slice[i].a, (long long)args.n_adapters * args.rank, args.k, args.k, maps.box)) return Q3_ERR_ARG;
    Q3_TRY_LAUNCH(launch(kernel, dim3((unsigned)tiles * cluster), dim3(LA_THREADS), smem, s, cluster, args, maps));
    return Q3_OK;
}
template <bool GATE_UP>
int launch_lora(const LoraArgs &args, int tiles, cudaStream_t s) {
    if (lora_tile_rows(args.n_rows) == 32) return launch_lora<32, GATE_UP, 0>(args, tiles, s);
    const int columns = args.n_slices * args.rank;
    if (columns <= 16) return launch_lora<16, GATE_UP, 2>(args, tiles, s);
    if (columns <= 32) return launch_lora<16, GATE_UP, 4>(args, tiles, s);
    if (columns <= 48) return launch_lora<16, GATE_UP, 6>(args, tiles, s);
    return launch_lora<16, GATE_UP, 0>(args, tiles, s);
}

int plan_check(int n_rows, int n_adapters) {
    return n_rows >= 0 && n_rows <= LA_MAX_ROWS && n_adapters > 0 && n_adapters <= LA_MAX_ADAPTERS ? Q3_OK : Q3_ERR_SHAPE;
}

int lora(const q3_lora_slice *slices, int n_slices, const q3_lora *l, bool gate_up, q3_bf16 *act, long long act_stride, void *stream) {
    if (!slices || !l) return Q3_ERR_ARG;
    if (n_slices < 1 || n_slices > LA_MAX_SLICES || plan_check(l->n_rows, l->n_adapters) != Q3_OK || l->k <= 0 || l->k % 8 || l->rank <= 0 ||
        l->rank % 8 || l->rank > LA_MAX_RANK || l->x_stride < l->k || l->x_stride % 8)
        return Q3_ERR_SHAPE;
    LoraArgs a = {};
    for (int i = 0; i < n_slices; i++) {
        const q3_lora_slice &c = slices[i];
        if (c.n <= 0 || c.n % 8 || c.base_stride < c.n || c.base_stride % 8 || (!gate_up && (c.out_stride < c.n || c.out_stride % 8)) ||
            (gate_up && c.n != slices[0].n))
            return Q3_ERR_SHAPE;
        a.slice[i] = {reinterpret_cast<bf16 *>(c.out), reinterpret_cast<const bf16 *>(c.base), reinterpret_cast<const bf16 *>(c.a),
                      reinterpret_cast<const bf16 *>(c.b), c.out_stride, c.base_stride, c.n};
    }
    if (gate_up && (act_stride < slices[0].n || act_stride % 8)) return Q3_ERR_SHAPE;
    if (l->n_rows == 0) return Q3_OK;  // before the pointers: tensors of no elements have none
    if (!l->x || !l->plan || (gate_up && !act)) return Q3_ERR_ARG;
    uintptr_t all = reinterpret_cast<uintptr_t>(l->x) | reinterpret_cast<uintptr_t>(l->plan) | reinterpret_cast<uintptr_t>(act);
    for (int i = 0; i < n_slices; i++) {
        const q3_lora_slice &c = slices[i];
        if (!c.base || !c.a || !c.b || (!gate_up && !c.out)) return Q3_ERR_ARG;
        all |= reinterpret_cast<uintptr_t>(c.base) | reinterpret_cast<uintptr_t>(c.a) | reinterpret_cast<uintptr_t>(c.b);
        const q3_bf16 *out = gate_up ? act : c.out;
        const long long out_stride = gate_up ? act_stride : c.out_stride;
        all |= reinterpret_cast<uintptr_t>(out);
        // an output is written while other CTAs still read x; in place of its base it is written by who read it
        if (overlap(out, out_stride, c.n, l->x, l->x_stride, l->k, l->n_rows)) return Q3_ERR_ARG;
        for (int j = 0; j < n_slices; j++) {
            const q3_lora_slice &d = slices[j];
            const bool same = out == d.base && out_stride == d.base_stride && (gate_up || i == j);
            if (!same && overlap(out, out_stride, c.n, d.base, d.base_stride, d.n, l->n_rows)) return Q3_ERR_ARG;
            if (!gate_up && j < i && overlap(out, out_stride, c.n, d.out, d.out_stride, d.n, l->n_rows)) return Q3_ERR_ARG;
        }
    }
    if (all & 15) return Q3_ERR_ALIGN;
    const int st = check_device();
    if (st != Q3_OK) return st;
    a.x = reinterpret_cast<const bf16 *>(l->x);
    a.x_stride = l->x_stride;
    a.ranks = l->ranks;
    a.scale = l->scale;
    a.plan = static_cast<const char *>(l->plan);
    a.act = reinterpret_cast<bf16 *>(act);
    a.act_stride = act_stride;
    a.n_slices = n_slices;
    a.k = l->k;
    a.rank = l->rank;
    a.n_rows = l->n_rows;
    a.n_adapters = l->n_adapters;
    a.wide = wide_of(n_slices, l->rank);
    a.pitch = pitch_of(a.wide);
    const int tiles = lora_plan_layout(l->n_rows, l->n_adapters).max_tiles;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return gate_up ? launch_lora<true>(a, tiles, s) : launch_lora<false>(a, tiles, s);
}

}  // namespace

unsigned take_error_lora() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v)) != cudaSuccess) return 0;
    if (v) cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return v;
}

}  // namespace q3

using namespace q3;

extern "C" {

size_t q3_lora_plan_bytes(int n_rows, int n_adapters) {
    return plan_check(n_rows, n_adapters) == Q3_OK ? lora_plan_layout(n_rows, n_adapters).bytes : 0;
}

int q3_lora_plan(void *plan, int n_rows, int n_adapters, const int *index, void *stream) {
    if (plan_check(n_rows, n_adapters) != Q3_OK) return Q3_ERR_SHAPE;
    if (n_rows == 0) return Q3_OK;
    if (!plan || !index) return Q3_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(plan) & 15) return Q3_ERR_ALIGN;
    const int st = check_device();
    if (st != Q3_OK) return st;
    const size_t smem = (size_t)((lora_plan_parts(n_rows, n_adapters) + 1) * (n_adapters + 1) + 32) * 4;
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(lora_plan_kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(lora_plan_kernel, dim3(1), dim3(LP_THREADS), smem, (cudaStream_t)stream, 1,
                         static_cast<char *>(plan), n_rows, n_adapters, index));
    return Q3_OK;
}

int q3_lora_add(const q3_lora_slice *slices, int n_slices, const q3_lora *l, void *stream) {
    return lora(slices, n_slices, l, false, nullptr, 0, stream);
}

int q3_lora_gate_up(q3_bf16 *act, long long act_stride, const q3_lora_slice *gate_up, const q3_lora *l, void *stream) {
    return lora(gate_up, 2, l, true, act, act_stride, stream);
}

}  // extern "C"
