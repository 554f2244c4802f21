// Low-rank adapters of many requests beside a shared projection (q3_lora_plan, q3_lora_add, q3_lora_gate_up):
// out = base + s_i B_i (A_i x) for the rows of adapter i, A_i [rank, k], B_i [n, rank], up to three projections of one x.
//
// The plan sorts a step's rows by their adapter, once for all layers, and cuts them into tiles, so that rows of one adapter
// anywhere in the batch share its weights. A cluster of CTAs takes a tile: each CTA multiplies its part of k, the partial
// A x are added up through distributed shared memory, and each CTA expands its part of the columns; nothing goes through global
// memory between the two products. Both run on warp-level matrix instructions with operands loaded straight into
// registers: the contraction's order is free as long as both operands have the same, so a lane takes eight (A x) or four
// (B h) neighbouring elements of its row, and its four columns of eight-column tiles are dealt out so that a lane writes eight
// neighbouring outputs. Bound by the bytes of x, base, out and the present adapters' weights (a rank of 64 is 64 products for each
// element of x, a tenth of what the tensor cores could do meanwhile) and, for few rows, by the chain of loads.
//
// A x is held in 32 bits and enters the second product as two bf16 numbers, which together have 16 bits of it: its
// rounding to one would be as large as the output's own.
#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace q3 {
int check_device();

namespace {

__device__ unsigned g_dev_error;

constexpr int LA_THREADS = 256;
constexpr int LA_WARPS = LA_THREADS / 32;
constexpr int LA_MAX_ROWS = 1 << 16;
constexpr int LA_MAX_ADAPTERS = 8192;
constexpr int LA_MAX_RANK = 128;
constexpr int LA_MAX_SLICES = 3;
constexpr int LA_PASS = 8;  // eight-column tiles of A x at a time: their sums stay in registers

struct LoraTile {
    int adapter, first, rows, unused;  // adapter -1: rows without one
};

// Rows of a tile: of a step of few rows as many as one matrix instruction takes.
__host__ __device__ constexpr int lora_tile_rows(int n_rows) { return n_rows <= 128 ? 16 : 64; }

struct LoraPlanLayout {
    size_t tiles, order, bytes;  // after the number of tiles
    int max_tiles;
};
__host__ __device__ inline LoraPlanLayout lora_plan_layout(int n_rows, int n_adapters) {
    LoraPlanLayout l = {};
    const int kinds = n_rows < n_adapters + 1 ? n_rows : n_adapters + 1;
    l.max_tiles = kinds + n_rows / lora_tile_rows(n_rows);
    l.tiles = 16;
    l.order = l.tiles + (size_t)l.max_tiles * sizeof(LoraTile);
    l.bytes = l.order + ((size_t)n_rows * 4 + 15) / 16 * 16;
    return l;
}

// ------------------------------------------------------------------ plan

constexpr int LP_THREADS = 1024;

__global__ void __launch_bounds__(LP_THREADS, 1) lora_plan_kernel(char *plan, int n_rows, int n_adapters, const int *index) {
    extern __shared__ int la_next[];  // [n_adapters + 1]: rows of each adapter, then where its next row goes; the last: none
    __shared__ int sums[2][32];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, tile_rows = lora_tile_rows(n_rows), kinds = n_adapters + 1;
    const LoraPlanLayout l = lora_plan_layout(n_rows, n_adapters);
    LoraTile *tiles = reinterpret_cast<LoraTile *>(plan + l.tiles);
    int *order = reinterpret_cast<int *>(plan + l.order);
    for (int i = tid; i < kinds; i += LP_THREADS) la_next[i] = 0;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    auto kind = [&](int row) {
        const int i = index[row];
        return i < 0 || i >= n_adapters ? n_adapters : i;
    };
    for (int row = tid; row < n_rows; row += LP_THREADS) {
        if (index[row] >= n_adapters) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
        atomicAdd(&la_next[kind(row)], 1);
    }
    __syncthreads();
    // running sums of rows and tiles, 1024 adapters at a time
    int row0 = 0, tile0 = 0;
    for (int i0 = 0; i0 < kinds; i0 += LP_THREADS) {
        const int i = i0 + tid, n = i < kinds ? la_next[i] : 0, t = (n + tile_rows - 1) / tile_rows;
        int rn = n, rt = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int yn = __shfl_up_sync(0xffffffffu, rn, o), yt = __shfl_up_sync(0xffffffffu, rt, o);
            rn += lane >= o ? yn : 0;
            rt += lane >= o ? yt : 0;
        }
        if (lane == 31) {
            sums[0][warp] = rn;
            sums[1][warp] = rt;
        }
        __syncthreads();
        int all_n = 0, all_t = 0, before_n = 0, before_t = 0;
        for (int w = 0; w < 32; w++) {
            if (w == warp) before_n = all_n, before_t = all_t;
            all_n += sums[0][w];
            all_t += sums[1][w];
        }
        const int first = row0 + before_n + rn - n, tile = tile0 + before_t + rt - t;
        if (i < kinds) la_next[i] = first;
        for (int k = 0; k < t; k++) tiles[tile + k] = {i < n_adapters ? i : -1, first + k * tile_rows, min(tile_rows, n - k * tile_rows), 0};
        row0 += all_n;
        tile0 += all_t;
        __syncthreads();
    }
    if (tid == 0) *reinterpret_cast<int *>(plan) = tile0;
    // each warp places the rows of its adapters, in their order
    for (int r0 = 0; r0 < n_rows; r0 += 32) {
        const int row = r0 + lane, k = row < n_rows ? kind(row) : -1;
        const bool mine = k >= 0 && k % (LP_THREADS / 32) == warp;
        if (!__any_sync(0xffffffffu, mine)) continue;
        const unsigned peers = __match_any_sync(0xffffffffu, mine ? k : -1);
        const int at = mine ? la_next[k] : 0;
        __syncwarp();
        if (mine) order[at + __popc(peers & ((1u << lane) - 1))] = row;
        if (mine && lane == __ffs(peers) - 1) la_next[k] = at + __popc(peers);
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
    int wide;  // columns of A x in shared memory: each slice's rank rounded up to 16
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

// GATE_UP: slices 0 and 1 are gate and up, and what is written is silu(gate) * up.
template <int ROWS, bool GATE_UP>
__global__ void __launch_bounds__(LA_THREADS) lora_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int M_TILES = ROWS / 16, K_SPLITS = LA_WARPS / M_TILES;
    extern __shared__ __align__(16) unsigned char la_smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank_c = cluster.block_rank(), tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int g = lane / 4, t = lane % 4;
    const int wide = a.wide;
    float *part = reinterpret_cast<float *>(la_smem);              // [LA_WARPS][16][8 * LA_PASS]
    float *h = part + LA_WARPS * 16 * 8 * LA_PASS;                 // [ROWS][wide]: this CTA's part of A x
    bf16 *hi = reinterpret_cast<bf16 *>(h + ROWS * wide);          // [ROWS][wide + 8]: the whole, scaled, upper and lower bits
    bf16 *lo = hi + ROWS * (wide + 8);
    __shared__ int row_s[ROWS];

    pdl_trigger();
    pdl_wait();
    const LoraPlanLayout l = lora_plan_layout(a.n_rows, a.n_adapters);
    const int tile = blockIdx.x / C;
    if (tile >= *reinterpret_cast<const int *>(a.plan)) return;  // the whole cluster
    const LoraTile job = reinterpret_cast<const LoraTile *>(a.plan + l.tiles)[tile];
    const int *order = reinterpret_cast<const int *>(a.plan + l.order) + job.first;
    const int rows = job.rows, adapter = job.adapter;
    if (tid < ROWS) row_s[tid] = order[min(tid, rows - 1)];  // past the last row: that row again, never written
    __syncthreads();

    int r = 0;
    float scale = 1.0f;
    if (adapter >= 0) {
        r = a.ranks ? max(0, min(a.ranks[adapter], a.rank)) : a.rank;
        if (a.scale) scale = a.scale[adapter];
    } else if (GATE_UP) {
        return;  // the whole cluster: act is right already
    }

    // ---- A x: warp (m tile, part of k)
    if (r > 0) {
        const int mt = warp % M_TILES, ks = warp / M_TILES;
        const int steps = (a.k + 31) / 32, parts = C * K_SPLITS, p = rank_c * K_SPLITS + ks;
        const int s0 = (int)((long long)steps * p / parts), s1 = (int)((long long)steps * (p + 1) / parts);
        const bool live = mt * 16 < rows;
        const bf16 *x0 = a.x + row_s[mt * 16 + g] * a.x_stride, *x1 = a.x + row_s[mt * 16 + g + 8] * a.x_stride;
        const int tiles_each = (r + 7) / 8, n_tiles = tiles_each * a.n_slices;
        for (int n0 = 0; n0 < n_tiles; n0 += LA_PASS) {
            float acc[LA_PASS][4] = {};
            const bf16 *w[LA_PASS];
#pragma unroll
            for (int j = 0; j < LA_PASS; j++) {
                const int nt = n0 + j, sl = nt / tiles_each, row = (nt - sl * tiles_each) * 8 + g;
                w[j] = nt < n_tiles && row < r ? a.slice[sl].a + ((long long)adapter * a.rank + row) * a.k : nullptr;
            }
            if (live) {
#pragma unroll 2
                for (int s = s0; s < s1; s++) {
                    const int k = 32 * s + 8 * t;
                    const uint4 zero = make_uint4(0, 0, 0, 0);
                    const bool in = k < a.k;
                    const uint4 u = in ? __ldg(reinterpret_cast<const uint4 *>(x0 + k)) : zero, v = in ? __ldg(reinterpret_cast<const uint4 *>(x1 + k)) : zero;
                    uint4 b[LA_PASS];
#pragma unroll
                    for (int j = 0; j < LA_PASS; j++) b[j] = in && w[j] ? __ldg(reinterpret_cast<const uint4 *>(w[j] + k)) : zero;
                    const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
                    for (int j = 0; j < LA_PASS; j++)
                        if (n0 + j < n_tiles) {
                            mma(acc[j], a0, b[j].x, b[j].y);
                            mma(acc[j], a1, b[j].z, b[j].w);
                        }
                }
            }
            float *mine = part + warp * 16 * 8 * LA_PASS;
#pragma unroll
            for (int j = 0; j < LA_PASS; j++) {
                *reinterpret_cast<float2 *>(mine + g * 8 * LA_PASS + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
                *reinterpret_cast<float2 *>(mine + (g + 8) * 8 * LA_PASS + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
            }
            __syncthreads();
            // the warps' parts, in their order
            for (int i = tid; i < rows * 8 * LA_PASS; i += LA_THREADS) {
                const int row = i / (8 * LA_PASS), col = i % (8 * LA_PASS), nt = n0 + col / 8;
                if (nt >= n_tiles) continue;
                float sum = 0.0f;
#pragma unroll
                for (int q = 0; q < K_SPLITS; q++) sum += part[((q * M_TILES + row / 16) * 16 + row % 16) * 8 * LA_PASS + col];
                const int sl = nt / tiles_each;
                h[row * wide + sl * (wide / a.n_slices) + (nt - sl * tiles_each) * 8 + col % 8] = sum;
            }
            __syncthreads();
        }
    }
    // ---- the CTAs' parts, in their order, each CTA some of the columns for all
    if (r > 0) {
        if (C > 1) cluster.sync();
        const int each = wide / a.n_slices, quads = rows * wide / 4, q0 = (int)((long long)quads * rank_c / C), q1 = (int)((long long)quads * (rank_c + 1) / C);
        for (int q = q0 + tid; q < q1; q += LA_THREADS) {
            const int row = 4 * q / wide, col = 4 * q % wide;
            float v[4] = {};
            if (col % each < r) {
                for (int c = 0; c < C; c++) {
                    const float4 f = *reinterpret_cast<const float4 *>((C > 1 ? cluster.map_shared_rank(h, c) : h) + 4 * q);
                    v[0] += f.x;
                    v[1] += f.y;
                    v[2] += f.z;
                    v[3] += f.w;
                }
            }
            float up[4], low[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float s = col % each + e < r ? scale * v[e] : 0.0f;
                up[e] = round_bf16(s);
                low[e] = isfinite(up[e]) ? s - up[e] : 0.0f;
            }
            const uint2 uh = make_uint2(pack2(up[0], up[1]), pack2(up[2], up[3])), ul = make_uint2(pack2(low[0], low[1]), pack2(low[2], low[3]));
            for (int c = 0; c < C; c++) {
                *reinterpret_cast<uint2 *>((C > 1 ? cluster.map_shared_rank(hi, c) : hi) + row * (wide + 8) + col) = uh;
                *reinterpret_cast<uint2 *>((C > 1 ? cluster.map_shared_rank(lo, c) : lo) + row * (wide + 8) + col) = ul;
            }
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
    }

    // ---- out: units of 32 columns, a warp each
    constexpr int PAIR = GATE_UP ? 2 : 1;
    const int each = wide / a.n_slices, k_steps = (r + 15) / 16;
    int units = 0;
    for (int sl = 0; sl < (GATE_UP ? 1 : a.n_slices); sl++) units += (a.slice[sl].n + 31) / 32;
    for (int u = rank_c * LA_WARPS + warp; u < units; u += C * LA_WARPS) {
        int sl = 0, n0 = u;
        if (!GATE_UP)
            while (n0 >= (a.slice[sl].n + 31) / 32) n0 -= (a.slice[sl++].n + 31) / 32;
        n0 *= 32;
        const int n = a.slice[sl].n;
        if (r == 0 && !GATE_UP && a.slice[sl].out == a.slice[sl].base) continue;
        for (int m = 0; m * 16 < rows; m++) {
            float acc[PAIR][4][4] = {};
            for (int s = 0; s < k_steps; s++) {
#pragma unroll
                for (int pr = 0; pr < PAIR; pr++) {
                    const LoraSlice &c = a.slice[sl + pr];
                    const int col = (sl + pr) * each + 16 * s + 4 * t, at = (m * 16 + g) * (wide + 8) + col;
                    uint2 q[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int nn = n0 + 8 * (g / 2) + 2 * j + g % 2, left = r - (16 * s + 4 * t);
                        q[j] = make_uint2(0, 0);
                        if (nn < n && left > 0) {
                            q[j] = __ldg(reinterpret_cast<const uint2 *>(c.b + ((long long)adapter * n + nn) * a.rank + 16 * s + 4 * t));
                            if (left < 4) {  // what is past the adapter's rank may be anything
                                q[j].x &= left == 1 ? 0xffffu : 0xffffffffu;
                                q[j].y &= left == 3 ? 0xffffu : 0u;
                            }
                        }
                    }
                    const uint2 u0 = *reinterpret_cast<const uint2 *>(hi + at), u1 = *reinterpret_cast<const uint2 *>(hi + at + 8 * (wide + 8));
                    const uint2 l0 = *reinterpret_cast<const uint2 *>(lo + at), l1 = *reinterpret_cast<const uint2 *>(lo + at + 8 * (wide + 8));
                    const uint32_t ah[4] = {u0.x, u1.x, u0.y, u1.y}, al[4] = {l0.x, l1.x, l0.y, l1.y};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        mma(acc[pr][j], ah, q[j].x, q[j].y);
                        mma(acc[pr][j], al, q[j].x, q[j].y);
                    }
                }
            }
            // a lane has eight neighbouring columns of rows g and g + 8
            const int col = n0 + 8 * t;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int i = m * 16 + g + 8 * half;
                if (i >= rows || col >= n) continue;
                const long long row = row_s[i];
                uint32_t y[4];
                if constexpr (GATE_UP) {
                    const uint4 bg = *reinterpret_cast<const uint4 *>(a.slice[0].base + row * a.slice[0].base_stride + col);
                    const uint4 bu = *reinterpret_cast<const uint4 *>(a.slice[1].base + row * a.slice[1].base_stride + col);
                    const __nv_bfloat162 *pg = reinterpret_cast<const __nv_bfloat162 *>(&bg), *pu = reinterpret_cast<const __nv_bfloat162 *>(&bu);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 fg = __bfloat1622float2(pg[j]), fu = __bfloat1622float2(pu[j]);
                        const float g0 = fg.x + acc[0][j][2 * half], g1 = fg.y + acc[0][j][2 * half + 1];
                        const float u0 = fu.x + acc[1][j][2 * half], u1 = fu.y + acc[1][j][2 * half + 1];
                        y[j] = pack2(g0 / (1.0f + __expf(-g0)) * u0, g1 / (1.0f + __expf(-g1)) * u1);
                    }
                    *reinterpret_cast<uint4 *>(a.act + row * a.act_stride + col) = make_uint4(y[0], y[1], y[2], y[3]);
                } else {
                    const LoraSlice &c = a.slice[sl];
                    uint4 b = *reinterpret_cast<const uint4 *>(c.base + row * c.base_stride + col);
                    if (r > 0) {
                        const __nv_bfloat162 *pb = reinterpret_cast<const __nv_bfloat162 *>(&b);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float2 f = __bfloat1622float2(pb[j]);
                            y[j] = pack2(f.x + acc[0][j][2 * half], f.y + acc[0][j][2 * half + 1]);
                        }
                        b = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                    *reinterpret_cast<uint4 *>(c.out + row * c.out_stride + col) = b;
                }
            }
        }
    }
}

int wide_of(int n_slices, int rank) { return n_slices * ((rank + 15) / 16 * 16); }

size_t lora_smem(int rows, int wide) {
    return (size_t)LA_WARPS * 16 * 8 * LA_PASS * 4 + (size_t)rows * wide * 4 + 2 * (size_t)rows * (wide + 8) * 2;
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

template <int ROWS, bool GATE_UP>
int launch_lora(const LoraArgs &args, int tiles, int cluster, cudaStream_t s) {
    auto kernel = lora_kernel<ROWS, GATE_UP>;
    const size_t smem = lora_smem(ROWS, args.wide);
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(kernel, dim3((unsigned)tiles * cluster), dim3(LA_THREADS), smem, s, cluster, args));
    return Q3_OK;
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
    const int tiles = lora_plan_layout(l->n_rows, l->n_adapters).max_tiles;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (lora_tile_rows(l->n_rows) == 16) return gate_up ? launch_lora<16, true>(a, tiles, 8, s) : launch_lora<16, false>(a, tiles, 8, s);
    return gate_up ? launch_lora<64, true>(a, tiles, 4, s) : launch_lora<64, false>(a, tiles, 4, s);
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
    Q3_TRY_LAUNCH(launch(lora_plan_kernel, dim3(1), dim3(LP_THREADS), (size_t)(n_adapters + 1) * 4, (cudaStream_t)stream, 1,
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
