// Attention of each sequence's new tokens over its pages (q3_paged_attention).
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = 2^(c q.k_t - m),  c = scale * log2(e)
//
// in one pass over the positions, with a running reference m per row that the sums are rescaled to when it
// grows. Partial results (o, m, l) of a row over disjoint positions combine as
// m = max m_i, o = sum 2^(m_i - m) o_i, l = sum 2^(m_i - m) l_i.
//
// Persistent CTAs, one per SM, take the pieces the plan gave them (paged.cuh). Two producer warps stream K and V
// by TMA, one box per run of positions inside a page, into a ring of stages. There are two kernels, by the rows of the
// items; in a step that has both, they run side by side on SMs that the plan has shared out.
//
// Few rows (a decode step): bound by the bytes of K and V, with 160 KB of loads in flight on each SM. Warp-level matrix
// instructions are enough for that; each warp owns whole 16 KB stages (32 positions at head_dim 128) with its own
// running maximum, so warps meet only at the end of a piece. 32 sequences at 4096, 32 query heads on 8: 85 us,
// 0.96 of the measured copy bandwidth; one sequence at 256: 5.4 us in a graph.
//
// Many rows (a chunk of a prompt): bound by the tensor cores and the chain between their products. 128 rows -- all
// query heads of a kv head side by side, token after token -- make a tcgen05 tile; two tiles share each K and V
// tile and alternate, one in its softmax while the other multiplies. S = Q K^T goes to tensor memory, two threads
// per row read it, write P back over it as bf16, and P is the A operand of O += P V from tensor memory. A step of two
// tiles takes 3550 cycles: per tile 2000 of softmax and 1400 of products (1024 of them multiplying), of which only the
// two tiles' overlap hides any. 2048 tokens at 8192, 32 query heads on 8: 310 to 320 us in a row, when the power limit
// holds the SMs near 1.67 GHz (1.0 PFLOP/s, 0.60 of the measured matrix rate), 270 in the first calls, at 1.97 GHz, with one
// set of inputs as with three. What did not help this kernel: 12 to 50 % of the exponentials by polynomial (272 to 307 us
// against 266, all in short runs). What did not help the forms before it: half-steps of 64 columns (388 to 397 us against
// 391, later 390 against 363), a product thread per tile (460, it spilled).
//
// Bad values behind the mask: a masked score is replaced, whatever it is, but a zero probability times a NaN
// or infinite v would still be NaN. Rows of V past the item's end are zeroed in shared memory; the few
// rows that some tokens of the item see and others do not are checked, and if one holds such a value that step's
// second product runs on the CUDA cores, skipping what each row does not see.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged.cuh"
#include "tc_common.cuh"
#include "waiter.cuh"

namespace q3 {
namespace {

__device__ unsigned g_dev_error;

constexpr int BOX64 = 16384;        // bytes of 128 rows x 64 columns, half a tile of K or V at head_dim 128
constexpr int BIG_STAGE = 32768;    // a ring stage in the kernel for many rows: one such tile
constexpr int BIG_STAGES = 5;
constexpr int SMALL_PRODUCERS = 2;  // warps that load, in the kernel for few rows
constexpr int BIG_THREADS = 128 + 512;  // loads, products; four softmax warpgroups, two threads a row
constexpr float GROW = 8.0f;        // many rows: the reference follows the maximum in steps of 2^8

struct PaArgs {
    bf16 *out;
    const bf16 *q;
    long long out_stride, q_stride;
    const int *table;
    const int2 *ctas;
    const PagedPiece *pieces, *splits;
    int *counters, *ready;
    float *small_o, *big_o;
    float2 *small_ml, *big_ml;
    int rep, tile_tok, head_dim, page_size, max_pages, n_tokens, row_elems;
    int small_box, big_box;  // rows of a TMA box: the largest power of two that divides a page, at most a step
    int small_step_pages, small_step_slots, big_step_pages, big_step_slots;  // a producer's step in pages and slots
    float scale_log2;
    uint32_t idesc_qk, idesc_pv;
};

// ---------------------------------------------------------------- helpers

// The kernel for few rows, launched behind the one for many, starts while that still runs, so its own
// griddepcontrol.wait would come too late, and what the other grid's wait made visible it did so to that grid alone.
// So CTA i of the kernel for many rows, after its wait, passes that on to CTA i of this one: a release, taken here
// by an acquire that also puts the flag back to rest. Every CTA of the other kernel has released before this one can
// start (it triggers after that), so the loop hardly ever turns.
__device__ __forceinline__ void give_ready(int *flag) {
    asm volatile("st.release.gpu.global.b32 [%0], 1;" ::"l"(flag) : "memory");
}
__device__ bool take_ready(int *flag) {
    const uint64_t start = globaltimer();
    for (;;) {
        int seen;
        asm volatile("atom.acquire.gpu.global.exch.b32 %0, [%1], 0;" : "=r"(seen) : "l"(flag) : "memory");
        if (seen != 0) return true;
        if (globaltimer() - start > WAIT_LIMIT_NS) {
            atomicOr(&g_dev_error, DEV_ERR_WAIT_TIMEOUT);
            return false;
        }
    }
}
// Orders what was written before by plain stores and is visible to this thread before its later TMA loads.
__device__ __forceinline__ void fence_proxy_async_global() { asm volatile("fence.proxy.async.global;" ::: "memory"); }

template <int N>
struct Ring {
    int s = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next(int by = 1) {
        s += by;
        if (s >= N) {
            s -= N;
            ph ^= 1;
        }
    }
    __device__ __forceinline__ void advance(int by) {  // any number of stages
        next(by % N);
        ph ^= by / N & 1;
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the disjunction over the N threads that meet at barrier `id`
template <int N>
__device__ __forceinline__ bool any_at(int id, bool x) {
    int y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %2, 0;\n\t"
        "barrier.cta.red.or.pred.aligned q, %1, %3, p;\n\t"
        "selp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(y)
        : "r"(id), "r"((int)x), "n"(N)
        : "memory");
    return y != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ void tma_page(void *dst, const CUtensorMap *map, int x, int slot, int head, int page,
                                         uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// the 8 x 8 matrix of 16-bit values that a warp holds as a fragment, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// one of two packed bf16 is NaN or infinite
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ bool not_finite8(const uint4 &u) {
    return not_finite2(u.x) || not_finite2(u.y) || not_finite2(u.z) || not_finite2(u.w);
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The step's description was refused as a whole (a negative piece count): every row is padding.
__device__ __forceinline__ void zero_rows(const PaArgs &a) {
    for (int t = blockIdx.x; t < a.n_tokens; t += gridDim.x)
        for (int i = threadIdx.x; i < a.row_elems / 8; i += blockDim.x)
            reinterpret_cast<uint4 *>(a.out + t * a.out_stride)[i] = make_uint4(0, 0, 0, 0);
}

// The position from which on at least one row of the piece's item is masked.
__device__ __forceinline__ int first_masked(const PagedPiece &p) { return p.pos0 + 1; }

// ---------------------------------------------------------------- few rows: producer

// A position's page-table index and slot, stepped without dividing.
struct PageWalk {
    int idx, slot;
    __device__ __forceinline__ PageWalk(int at, int page_size) : idx(at / page_size), slot(at % page_size) {}
    __device__ __forceinline__ void step(int pages, int slots, int page_size) {
        idx += pages;
        slot += slots;
        if (slot >= page_size) {
            slot -= page_size;
            idx++;
        }
    }
};

// NP warps stream a piece's steps: K and V of UPOS positions, NB = DP / 64 halves of 64 columns each, in the
// 128-byte swizzle. A warp fills every NP-th stage; each lane issues one box and looks up its page of the
// warp's next step before this one waits for room. The loop's length bounds the kernel: with one
// warp that divided by the page size it took 1360 cycles a stage, half of the time at which HBM delivers.
template <int DP, int NST, int NP>
__device__ void small_produce(const PaArgs &a, const CUtensorMap *mk, const CUtensorMap *mv, const PagedPiece &p,
                              unsigned char *ring, uint64_t *full, uint64_t *empty, Ring<NST> &r, int pid, Waiter &wait,
                              int step_pages, int step_slots) {
    constexpr int NB = DP / 64, UPOS = SMALL_STAGE / (4 * DP);
    static_assert(NST % NP == 0, "a stage belongs to one producer");
    const int lane = threadIdx.x % 32, box = a.small_box, nsub = UPOS / box;
    const int sub = lane % nsub, part = lane / nsub, half = part % NB;
    const bool active = part < 2 * NB, is_v = part >= NB;
    const int *tab = a.table + (size_t)p.seq * a.max_pages;
    const uint32_t off = (is_v ? NB : 0) * (UPOS * 128) + half * (UPOS * 128) + sub * box * 128;
    const CUtensorMap *map = is_v ? mv : mk;
    const int skip = (pid - r.s % NP + NP) % NP;  // steps of this piece before this warp's first
    const int units = max(1, (p.kv1 - p.kv0 + UPOS - 1) / UPOS);
    int at = p.kv0 + skip * UPOS + sub * box, p0 = p.kv0 + skip * UPOS;
    PageWalk w(at, a.page_size);
    Ring<NST> mine = r;
    mine.next(skip);
    int page = active && at < p.kv1 ? __ldg(tab + w.idx) : 0, slot = w.slot;
    for (int u = skip; u < units; u += NP) {
        w.step(step_pages, step_slots, a.page_size);
        const bool on = active && at < p.kv1;
        at += NP * UPOS;
        const int next_page = active && at < p.kv1 ? __ldg(tab + w.idx) : 0;
        wait(&empty[mine.s], mine.ph ^ 1);
        __syncwarp();
        if (lane == 0 && !wait.dead) {
            const int n = min(UPOS, max(0, p.kv1 - p0) + box - 1) & -box;
            mbar_arrive_expect_tx(&full[mine.s], (uint32_t)(n * 128 * NB * 2));
        }
        __syncwarp();
        if (on && !wait.dead) tma_page(ring + (size_t)mine.s * SMALL_STAGE + off, map, half * 64, slot, p.kvh, page, &full[mine.s]);
        mine.next(NP);
        p0 += NP * UPOS;
        page = next_page;
        slot = w.slot;
    }
    r.advance(units);
}

// ---------------------------------------------------------------- few rows: consumers

// Each warp owns whole stages. The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that positions
// and head columns fill the instruction's 16 rows and the query rows its 8 columns, in NQ tiles of them. Against queries
// as the 16 rows (most of them padding at 4 query heads per kv head) this halves products, exponentials and
// accumulators; P^T moves from accumulator to operand layout by an 8 x 8 transpose in registers.
// One tile keeps its queries in registers; more read them from q_s, laid out as the instruction's operand, and take
// a stage 32 positions at a time.
// merge_o is [NW][8][DP] fp32, columns permuted by row against bank conflicts; merge_ml (m, l); one tile at a time.
template <int DP, int NQ, int NW, int NST>
__device__ void small_consume(const PaArgs &a, const PagedPiece &p, unsigned char *ring, uint64_t *full,
                              uint64_t *empty, Ring<NST> &r, Waiter &wait, int cw, uint2 *q_s, int2 *lim_s, float *merge_o,
                              float2 *merge_ml, int *flag_s) {
    constexpr int NB = DP / 64, UPOS = SMALL_STAGE / (4 * DP), MT = NQ == 1 ? UPOS / 16 : 2, KS = DP / 16;
    const int lane = threadIdx.x % 32, g = lane / 4, tq = lane % 4, l7 = lane % 8, mi = lane / 8;
    const int rows = p.n_tok * a.rep, tid = cw * 32 + lane;
    // operand words of lane `ln`: queries of row 8 nq + ln / 4, columns 16 k + 8 j + 2 (ln % 4) and the one after
    auto queries = [&](int ln, int nq, int k) {
        const int row = 8 * nq + ln / 4, col = 16 * k + 2 * (ln % 4);
        const bf16 *src = a.q + (p.tok0 + row / a.rep) * a.q_stride + (long long)(p.kvh * a.rep + row % a.rep) * a.head_dim + col;
        return make_uint2(row < rows && col < a.head_dim ? *reinterpret_cast<const uint32_t *>(src) : 0u,
                          row < rows && col + 8 < a.head_dim ? *reinterpret_cast<const uint32_t *>(src + 8) : 0u);
    };
    // rows 8 nq + 2 tq and the next are this thread's columns of S^T and O^T, and see the positions before these; the last
    // step may reach past the piece, where nothing was loaded
    auto limit = [&](int row) { return min(p.pos0 + row / a.rep + 1, p.kv1); };
    uint2 qb[NQ == 1 ? KS : 1];
    int2 lim1;
    if (NQ == 1) {
#pragma unroll
        for (int k = 0; k < KS; k++) qb[k] = queries(lane, 0, k);
        lim1 = make_int2(limit(2 * tq), limit(2 * tq + 1));
    } else {
        for (int i = tid; i < KS * NQ * 32; i += NW * 32) q_s[i] = queries(i % 32, i / 32 % NQ, i / 32 / NQ);
        if (tid < 4 * NQ) lim_s[tid] = make_int2(limit(2 * tid), limit(2 * tid + 1));
        bar_sync(1, NW * 32);
    }
    auto limits = [&](int nq) { return NQ == 1 ? lim1 : lim_s[4 * nq + tq]; };
    const int lim_min = min(first_masked(p), p.kv1);
    float o[NQ][KS][4], m[NQ][2], l[NQ][2];  // o: head columns 16 i + g and + 8
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        m[nq][0] = m[nq][1] = -INFINITY;
        l[nq][0] = l[nq][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; i++) o[nq][i][0] = o[nq][i][1] = o[nq][i][2] = o[nq][i][3] = 0.0f;
    }
    // ldmatrix rows of this lane: K as [position][column] (operand rows = positions), V transposed
    const uint32_t k_row = ((mi & 1) * 8 + l7) * 128, v_row = ((mi >> 1) * 8 + l7) * 128;

    int p0 = p.kv0;
    do {
        if (r.s % NW == cw) {
            unsigned char *stage = ring + (size_t)r.s * SMALL_STAGE;
            const uint32_t kb = smem_u32(stage), vb = kb + NB * UPOS * 128;
            wait(&full[r.s], r.ph);
            __syncwarp();
            const bool masked = p0 + UPOS > lim_min;
            bool slow = false;
            if (p0 + UPOS > p.kv1) {  // rows past the end: zero
                const int t0 = max(0, p.kv1 - p0), n = (UPOS - t0) * 8;
                for (int h = 0; h < NB; h++)
                    for (int i = lane; i < n; i += 32)
                        reinterpret_cast<uint4 *>(stage + (NB + h) * (UPOS * 128) + t0 * 128)[i] = make_uint4(0, 0, 0, 0);
                fence_proxy_async();  // these writes, before the next TMA write of the stage
                __syncwarp();
            }
            if (masked && p.n_tok > 1) {  // rows that only some tokens see
                const int t0 = max(0, lim_min - p0), n = (min(UPOS, p.kv1 - p0) - t0) * 8;
                for (int h = 0; h < NB; h++)
                    for (int i = lane; i < n; i += 32)
                        slow |= not_finite8(reinterpret_cast<const uint4 *>(stage + (NB + h) * (UPOS * 128) + t0 * 128)[i]);
                slow = __any_sync(0xffffffffu, slow);
            }
#pragma unroll 1
            for (int h0 = 0; h0 < UPOS; h0 += 16 * MT) {  // 16 MT positions
                float s[NQ][MT][4];
#pragma unroll
                for (int nq = 0; nq < NQ; nq++)
#pragma unroll
                    for (int i = 0; i < MT; i++) s[nq][i][0] = s[nq][i][1] = s[nq][i][2] = s[nq][i][3] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const int c = 2 * k + (mi >> 1);
                    const uint32_t at = kb + h0 * 128 + k_row + (k / 4) * (UPOS * 128) + (((c % 8) ^ l7) << 4);
                    uint2 q[NQ];
#pragma unroll
                    for (int nq = 0; nq < NQ; nq++) q[nq] = NQ == 1 ? qb[k] : q_s[(k * NQ + nq) * 32 + lane];
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        uint32_t ka[4];
                        ldsm4(ka, at + i * 16 * 128);
#pragma unroll
                        for (int nq = 0; nq < NQ; nq++) mma16816(s[nq][i], ka, q[nq].x, q[nq].y);
                    }
                }
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) {
                    float x[2] = {-INFINITY, -INFINITY};
                    const int2 lim = masked ? limits(nq) : make_int2(INT_MAX, INT_MAX);
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            s[nq][i][j] *= a.scale_log2;
                            if (p0 + h0 + 16 * i + 8 * (j >> 1) + g >= (j & 1 ? lim.y : lim.x)) s[nq][i][j] = -INFINITY;
                            x[j & 1] = fmaxf(x[j & 1], s[nq][i][j]);
                        }
#pragma unroll
                    for (int off = 4; off < 32; off *= 2) {
                        x[0] = fmaxf(x[0], __shfl_xor_sync(0xffffffffu, x[0], off));
                        x[1] = fmaxf(x[1], __shfl_xor_sync(0xffffffffu, x[1], off));
                    }
                    if (__any_sync(0xffffffffu, x[0] > m[nq][0] || x[1] > m[nq][1])) {
                        float f[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float top = fmaxf(m[nq][e], x[e]);
                            f[e] = top == -INFINITY ? 1.0f : ex2(m[nq][e] - top);
                            m[nq][e] = top;
                            l[nq][e] *= f[e];
                        }
#pragma unroll
                        for (int i = 0; i < KS; i++)
#pragma unroll
                            for (int j = 0; j < 4; j++) o[nq][i][j] *= f[j & 1];
                    }
                    const float base[2] = {m[nq][0] == -INFINITY ? 0.0f : m[nq][0], m[nq][1] == -INFINITY ? 0.0f : m[nq][1]};
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            s[nq][i][j] = ex2(s[nq][i][j] - base[j & 1]);
                            l[nq][j & 1] += s[nq][i][j];
                        }
                }
                if (!slow) {
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        uint32_t pb[NQ][2];
#pragma unroll
                        for (int nq = 0; nq < NQ; nq++) {
                            pb[nq][0] = transpose8(pack_bf16(s[nq][t][0], s[nq][t][1]));
                            pb[nq][1] = transpose8(pack_bf16(s[nq][t][2], s[nq][t][3]));
                        }
#pragma unroll
                        for (int i = 0; i < KS; i++) {
                            const int c = 2 * i + (mi & 1);
                            uint32_t va[4];
                            ldsm4_t(va, vb + h0 * 128 + v_row + t * 16 * 128 + (i / 4) * (UPOS * 128) + (((c % 8) ^ l7) << 4));
#pragma unroll
                            for (int nq = 0; nq < NQ; nq++) mma16816(o[nq][i], va, pb[nq][0], pb[nq][1]);
                        }
                    }
                } else {  // position by position, skipping what each row does not see; the probabilities by way of this
                          // warp's part of the merge buffer, [16 MT][8]
                    float *ps = merge_o + cw * 8 * DP;
#pragma unroll
                    for (int nq = 0; nq < NQ; nq++) {
                        const int2 lim = limits(nq);
#pragma unroll
                        for (int i = 0; i < MT; i++)
#pragma unroll
                            for (int j = 0; j < 4; j++) ps[(16 * i + 8 * (j >> 1) + g) * 8 + 2 * tq + (j & 1)] = s[nq][i][j];
                        __syncwarp();
#pragma unroll 1
                        for (int t = h0; t < h0 + 16 * MT; t++) {
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                if (p0 + t >= (e ? lim.y : lim.x)) continue;
                                const float w = ps[(t - h0) * 8 + 2 * tq + e];
#pragma unroll
                                for (int c = 0; c < 2 * KS; c++)  // columns 8 c + g
                                    o[nq][c / 2][c % 2 * 2 + e] +=
                                        w * __bfloat162float(*reinterpret_cast<const bf16 *>(
                                                stage + (NB + c / 8) * (UPOS * 128) + t * 128 + (((c % 8) ^ (t & 7)) << 4) + 2 * g));
                            }
                        }
                        __syncwarp();
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && !wait.dead) mbar_arrive(&empty[r.s]);  // a load that never came may still be owed to this stage
        }
        r.next();
        p0 += UPOS;
    } while (p0 < p.kv1);

    // ---- merge the warps
    // four columns of a row of the output; a row without positions is zero
    auto put = [&](int row, int d, const float *acc, float sum) {
        const float inv = 1.0f / sum;
        bf16 *dst = a.out + (p.tok0 + row / a.rep) * a.out_stride + (long long)(p.kvh * a.rep + row % a.rep) * a.head_dim + d;
        if (d < a.head_dim)
            *reinterpret_cast<uint2 *>(dst) =
                p.pos0 + row / a.rep < 0 ? make_uint2(0u, 0u)
                                         : make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
    };
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int off = 4; off < 32; off *= 2) {
            l[nq][0] += __shfl_xor_sync(0xffffffffu, l[nq][0], off);
            l[nq][1] += __shfl_xor_sync(0xffffffffu, l[nq][1], off);
        }
#pragma unroll 1
    for (int at = 0; at < NQ; at++) {
        const int here = min(8, rows - 8 * at);
        if (here <= 0) break;
        if (at > 0) bar_sync(1, NW * 32);  // the tile before has been read
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            if (nq != at) continue;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int row = 2 * tq + e;
                if (row < here) {
                    float *dst = merge_o + (cw * 8 + row) * DP;
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        dst[(16 * i + g) ^ (tq * 8)] = o[nq][i][e];
                        dst[(16 * i + 8 + g) ^ (tq * 8)] = o[nq][i][2 + e];
                    }
                    if (g == 0) merge_ml[cw * 8 + row] = make_float2(m[nq][e], l[nq][e]);
                }
            }
        }
        bar_sync(1, NW * 32);
        for (int i = tid; i < here * (DP / 4); i += NW * 32) {
            const int row = i / (DP / 4), d = i % (DP / 4) * 4;
            float top = -INFINITY, sum = 0.0f, acc[4] = {};
#pragma unroll
            for (int w = 0; w < NW; w++) top = fmaxf(top, merge_ml[w * 8 + row].x);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float2 ml = merge_ml[w * 8 + row];
                const float f = ex2(ml.x - base);
                const float4 v = *reinterpret_cast<const float4 *>(merge_o + (w * 8 + row) * DP + (d ^ ((row >> 1 & 3) * 8)));
                sum += f * ml.y;
                acc[0] += f * v.x;
                acc[1] += f * v.y;
                acc[2] += f * v.z;
                acc[3] += f * v.w;
            }
            if (p.part < 0) {
                put(8 * at + row, d, acc, sum);
            } else {
                const size_t to = (size_t)p.part * (8 * NQ) + 8 * at + row;
                __stcg(reinterpret_cast<float4 *>(a.small_o + to * DP + d), make_float4(acc[0], acc[1], acc[2], acc[3]));
                if (d == 0) __stcg(a.small_ml + to, make_float2(top, sum));
            }
        }
    }
    if (p.part >= 0) {  // the item's last piece to finish adds the parts up, in their order
        __threadfence();
        bar_sync(1, NW * 32);
        if (tid == 0) *flag_s = atomicAdd(a.counters + p.first, 1) == p.n_parts - 1;
        bar_sync(1, NW * 32);
        if (*flag_s) {
            __threadfence();
            for (int i = tid; i < rows * (DP / 4); i += NW * 32) {
                const int row = i / (DP / 4), d = i % (DP / 4) * 4;
                float top = -INFINITY, sum = 0.0f, acc[4] = {};
                for (int w = 0; w < p.n_parts; w++)
                    top = fmaxf(top, __ldcg(a.small_ml + (size_t)part_slot(p.first, w) * (8 * NQ) + row).x);
                const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
                for (int w = 0; w < p.n_parts; w++) {
                    const size_t at = (size_t)part_slot(p.first, w) * (8 * NQ) + row;
                    const float2 ml = __ldcg(a.small_ml + at);
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(a.small_o + at * DP + d));
                    const float f = ex2(ml.x - base);
                    sum += f * ml.y;
                    acc[0] += f * v.x;
                    acc[1] += f * v.y;
                    acc[2] += f * v.z;
                    acc[3] += f * v.w;
                }
                put(row, d, acc, sum);
            }
            if (tid == 0) a.counters[p.first] = 0;
        }
    }
    bar_sync(1, NW * 32);  // the merge buffer is free again
}

// ---------------------------------------------------------------- partial results of many rows

// Where a partial result keeps columns d .. d + 3 of a row, in scratch slot `slot`: four columns of all rows side by
// side, so that a warp's 32 rows are one run of memory (row by row, its accesses took a sector each, and 20 us a piece).
template <int DP>
__device__ __forceinline__ float4 *big_part(const PaArgs &a, int slot, int d, size_t row) {
    return reinterpret_cast<float4 *>(a.big_o + (size_t)slot * (2 * BIG_TILE) * DP) + (size_t)(d / 4) * (2 * BIG_TILE) + row;
}

// Adds up the parts of big items that were cut. The kernel for few rows ends with it, once the
// other one has finished; as a launch of its own it cost 2 to 3 us more. A CTA takes 16 columns each of GROUPS items, a
// different GROUPS-th of all items for each group of columns, and their rows one after the other, a thread per row.
template <int DP>
__device__ void combine_big(const PaArgs &a) {
    constexpr int GROUPS = DP / 16;
    auto item = [&](int i) { return a.splits + (blockIdx.x + i * (gridDim.x / GROUPS)) % gridDim.x; };
    int rows[GROUPS], total = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; i++) rows[i] = item(i)->n_parts > 1 ? item(i)->n_tok * a.rep : 0;
#pragma unroll
    for (int i = 0; i < GROUPS; i++) total += rows[i];
#pragma unroll 1
    for (int at = threadIdx.x; at < total; at += blockDim.x) {
        int g = 0, r = at;
#pragma unroll
        for (int i = 0; i < GROUPS - 1; i++)
            if (g == i && r >= rows[i]) {
                r -= rows[i];
                g++;
            }
        const int d = g * 16;
        if (d >= a.head_dim) continue;
        const PagedPiece p = *item(g);
        const int tt = r / a.rep, x = tt / a.tile_tok, row = x * BIG_TILE + (tt - x * a.tile_tok) * a.rep + r % a.rep;
        float m = -INFINITY, l = 0.0f, acc[16] = {};
#pragma unroll 1
        for (int w0 = 0; w0 < p.n_parts; w0 += 4) {  // four parts' loads in flight
            float2 ml[4];
            float4 v[4][4];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                ml[w] = make_float2(-INFINITY, 0.0f);
                if (w0 + w >= p.n_parts) continue;
                const int slot = part_slot(p.first, w0 + w);
                ml[w] = __ldcg(a.big_ml + (size_t)slot * (2 * BIG_TILE) + row);
#pragma unroll
                for (int q = 0; q < 4; q++) v[w][q] = __ldcg(big_part<DP>(a, slot, d, row) + q * (2 * BIG_TILE));
            }
            const float top = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
            const float base = top == -INFINITY ? 0.0f : top, f0 = ex2(m - base);
            m = top;
            l *= f0;
#pragma unroll
            for (int e = 0; e < 16; e++) acc[e] *= f0;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if (w0 + w >= p.n_parts) continue;
                const float f = ex2(ml[w].x - base);
                l += f * ml[w].y;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    acc[4 * q] += f * v[w][q].x;
                    acc[4 * q + 1] += f * v[w][q].y;
                    acc[4 * q + 2] += f * v[w][q].z;
                    acc[4 * q + 3] += f * v[w][q].w;
                }
            }
        }
        const float inv = 1.0f / l;
        bf16 *dst = a.out + (p.tok0 + tt) * a.out_stride + (long long)(p.kvh * a.rep + r % a.rep) * a.head_dim + d;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = pack_bf16(acc[8 * e + 2 * q] * inv, acc[8 * e + 2 * q + 1] * inv);
            if (d + 8 * e < a.head_dim)  // a row without positions is zero
                reinterpret_cast<uint4 *>(dst)[e] = p.pos0 + tt < 0 ? make_uint4(0, 0, 0, 0) : make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ---------------------------------------------------------------- kernel for few rows alone

constexpr int SMALL_WARPS = 10;  // consumers, each with a stage of its own

template <int DP, int NQ>
struct SmallSmem {
    alignas(1024) unsigned char ring[SMALL_WARPS * SMALL_STAGE];
    float merge_o[SMALL_WARPS * 8 * DP];
    float2 merge_ml[SMALL_WARPS * 8];
    uint2 q[NQ == 1 ? 1 : DP / 16 * NQ * 32];
    int2 lim[4 * NQ];
    uint64_t full[SMALL_WARPS], empty[SMALL_WARPS];
    int flag, go, down;
};

// AFTER_BIG: launched behind the kernel for many rows, whose results are needed at the end only.
template <int DP, int NQ, bool AFTER_BIG>
__global__ void __launch_bounds__((SMALL_PRODUCERS + SMALL_WARPS) * 32, 1)
    paged_small_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                       const __grid_constant__ PaArgs a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    SmallSmem<DP, NQ> &sm = *reinterpret_cast<SmallSmem<DP, NQ> *>(align_shared<1024>(smem_raw));
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        for (int i = 0; i < SMALL_WARPS; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        fence_barrier_init();
        sm.down = 0;
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    // The kernel before is the plan or whatever wrote q, K and V; or it is the kernel for many rows, whose CTA says when
    // it has waited for those.
    if (AFTER_BIG && threadIdx.x == 32) sm.go = take_ready(a.ready + blockIdx.x);
    __syncthreads();
    pdl_trigger();
    int2 work = make_int2(0, 0);
    if (!AFTER_BIG) pdl_wait();
    else fence_proxy_async_global();
    if (!AFTER_BIG || sm.go) work = a.ctas[blockIdx.x];
    if (work.y < 0) zero_rows(a);
    Ring<SMALL_WARPS> r;
    Waiter wait(&g_dev_error, &sm.down);
    for (int i = 0; i < work.y; i++) {
        const PagedPiece p = a.pieces[work.x + i];
        // every load is waited for by a consumer before the CTA ends; one that has given up gets no more
        if (warp >= SMALL_WARPS)
            small_produce<DP, SMALL_WARPS, SMALL_PRODUCERS>(a, &mk, &mv, p, sm.ring, sm.full, sm.empty, r, warp - SMALL_WARPS, wait,
                                                             a.small_step_pages, a.small_step_slots);
        else
            small_consume<DP, NQ, SMALL_WARPS, SMALL_WARPS>(a, p, sm.ring, sm.full, sm.empty, r, wait, warp, sm.q, sm.lim, sm.merge_o, sm.merge_ml,
                                                         &sm.flag);
    }
    if (wait.dead) settle();
    if constexpr (AFTER_BIG) {  // whoever waits for this kernel waits for that one, too
        pdl_wait();
        combine_big<DP>(a);
    }
}

// ---------------------------------------------------------------- many rows

// D[tmem] (+)= A[tmem] B[smem], bf16
__device__ __forceinline__ void mma_bf16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

#define Q3_R16(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), \
    "=r"(r[o + 6]), "=r"(r[o + 7]), "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]), "=r"(r[o + 11]), \
    "=r"(r[o + 12]), "=r"(r[o + 13]), "=r"(r[o + 14]), "=r"(r[o + 15])

// 32 columns of this thread's tensor-memory lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : Q3_R16(r, 0), Q3_R16(r, 16)
        : "r"(taddr)
        : "memory");
}
#undef Q3_R16

#define Q3_W16(r) "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), \
    "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        Q3_W16(r)
        : "memory");
}
#undef Q3_W16

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int DP>
struct BigSmem {
    alignas(1024) unsigned char q[DP / 64 * 2 * BOX64];  // two query tiles
    alignas(1024) unsigned char ring[BIG_STAGES * BIG_STAGE];
    float stat[2][2][BIG_TILE];  // by tile and half of the columns: a row's maximum, at the end its sum
    uint64_t full[BIG_STAGES], empty[BIG_STAGES], q_full, q_empty, s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int slow[2];  // by tile: this step's second product is not the tensor core's
    int down;
};

// Tensor memory: S of tile x at column 128 x, O at 256 + DP x. P of positions 0 .. 63 lies over the first 32 columns of
// their scores, P of 64 .. 127 over the first 32 of theirs.
__device__ __forceinline__ uint32_t tmem_s(uint32_t base, int x) { return base + 128 * x; }
template <int DP>
__device__ __forceinline__ uint32_t tmem_o(uint32_t base, int x) {
    return base + 256 + DP * x;
}

__device__ __forceinline__ int big_steps(const PagedPiece &p) { return max(1, (p.kv1 - p.kv0 + BIG_TILE - 1) / BIG_TILE); }

// One warp loads a piece's queries, then K of each 128-position step, another one V; each lane issues one box.
template <int DP>
__device__ void big_produce(const PaArgs &a, const CUtensorMap *mq, const CUtensorMap *mk, const CUtensorMap *mv,
                            const PagedPiece &p, BigSmem<DP> &sm, Ring<BIG_STAGES> &r, uint32_t &q_ph, int pid, Waiter &wait) {
    constexpr int NB = DP / 64;
    const int lane = threadIdx.x % 32, tiles = p.n_tok > a.tile_tok ? 2 : 1, n = big_steps(p);
    Ring<BIG_STAGES> mine = r;
    r.advance(2 * n);
    if (pid == 0) {
        wait(&sm.q_empty, q_ph ^ 1);
        q_ph ^= 1;
        if (wait.stopped()) return;
        if (lane == 0) mbar_arrive_expect_tx(&sm.q_full, (uint32_t)(tiles * NB * a.tile_tok * a.rep * 128));
        __syncwarp();
        if (lane < tiles * NB)
            tma_load_3d(sm.q + lane * BOX64, mq, lane % NB * 64, p.kvh * a.rep, p.tok0 + lane / NB * a.tile_tok, &sm.q_full);
    } else {
        mine.next();
    }
    const CUtensorMap *map = pid == 0 ? mk : mv;
    const int box = a.big_box, nsub = BIG_TILE / box, sub = lane % nsub, half = lane / nsub;
    const bool active = half < NB;
    const int *tab = a.table + (size_t)p.seq * a.max_pages;
    int at = p.kv0 + sub * box, p0 = p.kv0;
    PageWalk w(at, a.page_size);
    int page = active && at < p.kv1 ? __ldg(tab + w.idx) : 0, slot = w.slot;
    for (int j = 0; j < n; j++) {
        w.step(a.big_step_pages, a.big_step_slots, a.page_size);
        const bool on = active && at < p.kv1;
        at += BIG_TILE;
        const int next_page = active && at < p.kv1 ? __ldg(tab + w.idx) : 0;
        const uint32_t bytes = (uint32_t)((min(BIG_TILE, max(0, p.kv1 - p0) + box - 1) & -box) * 128 * NB);
        wait(&sm.empty[mine.s], mine.ph ^ 1);
        if (wait.stopped()) return;
        if (lane == 0) mbar_arrive_expect_tx(&sm.full[mine.s], bytes);
        __syncwarp();
        if (on)
            tma_page(sm.ring + (size_t)mine.s * BIG_STAGE + half * BOX64 + sub * box * 128, map, half * 64, slot, p.kvh, page,
                     &sm.full[mine.s]);
        mine.next(2);
        page = next_page;
        slot = w.slot;
        p0 += BIG_TILE;
    }
}

// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t y;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(y));
    return y != 0;
}
// a value that is the same in every lane, in a way that the compiler sees it
template <typename T>
__device__ __forceinline__ T uniform(T x) {
    return __shfl_sync(0xffffffffu, x, 0);
}

// One thread of a warp issues the products of both tiles in turn: O += P V of this step, then S = Q K^T of the next one
// over the columns that P was read from (the tensor core takes one thread's products in order). A tile's
// two products run back to back while the other tile is in its softmax. s_full of a step says, too, that the
// product of the step before has finished; o_full says it of the last one. Neither can move on
// twice before its softmax has seen the first time.
//
// This warp's own instructions are what the tensor core idles for, so they are few: one wait per step and tile, for P,
// with another warp's arrival on the same barrier (big_ready) saying that V and the next K have landed; control
// flow that is the same for all lanes, with what it depends on broadcast, so that operands of the products are made
// in uniform registers (as one lane's code, a product took up to 95 cycles to issue instead of 56).
template <int DP>
__device__ void big_multiply(const PaArgs &a, const PagedPiece &p, BigSmem<DP> &sm, uint32_t tmem_any, Ring<BIG_STAGES> &r,
                             uint32_t &q_ph, uint32_t &p_ph, Waiter &wait) {
    const int tiles = uniform(p.n_tok > a.tile_tok ? 2 : 1), n = uniform(big_steps(p));
    const int first = uniform((first_masked(p) - p.kv0) / BIG_TILE);  // rows are masked from this step on
    const uint32_t tmem = uniform(tmem_any), ring = smem_u32(sm.ring);
    const uint64_t q_desc = smem_desc_sw128(smem_u32(sm.q)), k_desc = smem_desc_sw128(ring),
                   v_desc = smem_desc_sw128(ring, BOX64, 1024);  // descriptors count in 16 bytes
    auto scores = [&](int x, int stage) {
        const uint64_t qd = q_desc + x * (DP / 64 * BOX64 >> 4), kd = k_desc + stage * (BIG_STAGE >> 4);
#pragma unroll
        for (int k = 0; k < DP / 16; k++)
            mma_bf16(tmem_s(tmem, x), qd + k / 4 * (BOX64 >> 4) + k % 4 * 2, kd + k / 4 * (BOX64 >> 4) + k % 4 * 2, a.idesc_qk, k > 0);
        mma_commit(&sm.s_full[x]);
    };
    wait(&sm.q_full, q_ph);
    q_ph ^= 1;
    wait(&sm.full[r.s], r.ph);
    if (__any_sync(0xffffffffu, wait.dead)) return;
    tc_fence_after();
    int stage = uniform(r.s);
    r.advance(2 * n);
    if (elect_one()) {
        scores(0, stage);
        if (tiles > 1) scores(1, stage);
        mma_commit(&sm.empty[stage]);
        if (n == 1) mma_commit(&sm.q_empty);
    }
    __syncwarp();
    stage = stage + 1 == BIG_STAGES ? 0 : stage + 1;
#pragma unroll 1
    for (int j = 0; j < n; j++) {
        const bool more = j + 1 < n;
        const int v_stage = stage, k_stage = stage + 1 == BIG_STAGES ? 0 : stage + 1;
        stage = k_stage + 1 == BIG_STAGES ? 0 : k_stage + 1;
        const uint64_t vd = v_desc + v_stage * (BIG_STAGE >> 4);
#pragma unroll
        for (int x = 0; x < 2; x++) {
            if (x == 1 && tiles == 1) break;
            wait(&sm.p_full[x], p_ph >> x & 1);
            p_ph ^= 1u << x;
            tc_fence_after();
            const bool slow = j >= first && *(const volatile int *)&sm.slow[x];
            if (elect_one()) {
                if (!slow) {
#pragma unroll
                    for (int k = 0; k < BIG_TILE / 16; k++)
                        mma_bf16_ta(tmem_o<DP>(tmem, x), tmem_s(tmem, x) + k / 4 * 64 + k % 4 * 8, vd + k * (2048 >> 4), a.idesc_pv, j > 0 || k > 0);
                }
                if (more) scores(x, k_stage);
                else mma_commit(&sm.o_full[x]);
                if (x == tiles - 1) {
                    mma_commit(&sm.empty[v_stage]);
                    if (more) mma_commit(&sm.empty[k_stage]);
                    if (j + 2 == n) mma_commit(&sm.q_empty);
                }
            }
            __syncwarp();
        }
    }
}

// One thread waits for V of each step and K of the next, and passes that on with P's arrivals. Their stages are not
// released before it has arrived. A piece's first K is not waited for here: the products release it without asking
// this thread, which could come so late that its stage has been filled once more, a phase it would wait for in vain.
template <int DP>
__device__ void big_ready(const PaArgs &a, const PagedPiece &p, BigSmem<DP> &sm, Ring<BIG_STAGES> &r, uint32_t &p_ph,
                          Waiter &wait) {
    const int tiles = p.n_tok > a.tile_tok ? 2 : 1, n = big_steps(p);
    r.next();
    for (int j = 0; j < n; j++) {
        wait(&sm.full[r.s], r.ph);
        r.next();
        if (j + 1 < n) {
            wait(&sm.full[r.s], r.ph);
            r.next();
        }
        for (int x = 0; x < tiles; x++) {
            wait(&sm.p_full[x], p_ph >> x & 1 ^ 1);  // the step before has its P: this arrival counts for this one
            p_ph ^= 1u << x;
            if (wait.dead) return;
            mbar_arrive(&sm.p_full[x]);
        }
    }
}

// 64 scores of a row: their largest (in `top`), P against the row's reference as bf16, and P's sum. Columns at or past
// `seen` are left out.
template <bool MASKED>
__device__ __forceinline__ float exp64(uint32_t ts, int seen, uint64_t c2, uint64_t base2, uint32_t *pk, float &top) {
    uint32_t u[64];
    tmem_ld32(ts, u);
    tmem_ld32(ts + 32, u + 32);
    tmem_wait_ld();
    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    uint64_t sum[2] = {};
#pragma unroll
    for (int e = 0; e < 32; e++) {
        float s0 = __uint_as_float(u[2 * e]), s1 = __uint_as_float(u[2 * e + 1]);
        if (MASKED && 2 * e >= seen) s0 = -INFINITY;
        if (MASKED && 2 * e + 1 >= seen) s1 = -INFINITY;
        x[e & 3] = max3(x[e & 3], s0, s1);
        const uint64_t y = fma2(pair(s0, s1), c2, base2);
        const float2 w = unpair(y);
        const float p0 = ex2(w.x), p1 = ex2(w.y);
        sum[e & 1] = add2(sum[e & 1], pair(p0, p1));
        pk[e] = pack_bf16(p0, p1);
    }
    top = fmaxf(max3(x[0], x[1], x[2]), x[3]);
    const float2 w = unpair(add2(sum[0], sum[1]));
    return w.x + w.y;
}

// Two warpgroups per tile, two threads per row: each takes 64 of a step's columns and half of the output's.
template <int DP>
__device__ void big_softmax(const PaArgs &a, const PagedPiece &p, BigSmem<DP> &sm, uint32_t tmem, int x, int part,
                            Ring<BIG_STAGES> &r, uint32_t &s_ph, Waiter &wait) {
    constexpr int NB = DP / 64, HALF = BIG_TILE / 2;
    const int n = big_steps(p), lim_min = first_masked(p);
    if (x == 1 && p.n_tok <= a.tile_tok) {  // this tile is empty
        r.advance(2 * n);
        return;
    }
    const int quarter = threadIdx.x / 32 % 4, lane = threadIdx.x % 32, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t ts = tmem_s(tmem, x) + lanes, to = tmem_o<DP>(tmem, x) + lanes + part * (DP / 2);
    const int tt = x * a.tile_tok + row / a.rep, lim = p.pos0 + tt + 1;
    // a negative scale negates Q in the first product; a zero one must still leave masked scores at -infinity
    const float c = fmaxf(fabsf(a.scale_log2), 1e-30f);
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    for (int j = 0; j < n; j++) {
        r.next();
        const Ring<BIG_STAGES> rv = r;
        r.next();
        const int t0 = p.kv0 + j * BIG_TILE;
        const bool masked = t0 + BIG_TILE > lim_min;
        wait(&sm.s_full[x], s_ph & 1);
        s_ph ^= 1;
        __syncwarp();
        tc_fence_after();
        bool slow = false;
        unsigned char *v = sm.ring + (size_t)rv.s * BIG_STAGE;
        if (masked) {  // V past the item's end becomes zero; rows only some tokens see are checked
            wait(&sm.full[rv.s], rv.ph);
            __syncwarp();
            const int end = min(BIG_TILE, p.kv_end - t0), check = max(0, lim_min - t0);
            for (int i = row + part * 128; i < NB * BIG_TILE * 8; i += 256) {
                uint4 *chunk = reinterpret_cast<uint4 *>(v) + i;
                const int t = i / 8 % BIG_TILE;
                if (t >= end) *chunk = make_uint4(0, 0, 0, 0);
                else if (t >= check) slow |= not_finite8(*chunk);
            }
            fence_proxy_async();
            slow = any_at<256>(9 + x, slow);
        }
        if (masked && row == 0 && part == 0) sm.slow[x] = slow;
        // P is taken against the reference as it stands, its maximum found on the way. Only if a row outgrew its
        // reference (always in the first step) is the reference moved, what was summed against it rescaled, and P
        // taken again; S is still in tensor memory, for P is stored after the row's two threads have agreed.
        const uint32_t sv = ts + HALF * part;
        const int seen = lim - t0 - HALF * part, pairs = 1 + x * 4 + quarter;
        uint32_t pk[32];
        float top, more;
        auto take = [&]() {
            const float base = m == -INFINITY ? 0.0f : -m;
            more = masked ? exp64<true>(sv, seen, pair(c, c), pair(base, base), pk, top)
                          : exp64<false>(sv, 0, pair(c, c), pair(base, base), pk, top);
        };
        take();
        if (any_at<64>(pairs, top * c > m + GROW || (m == -INFINITY && top > m))) {
            sm.stat[x][part][row] = top;
            bar_sync(pairs, 64);
            const float both = fmaxf(top, sm.stat[x][part ^ 1][row]) * c;
            const bool grow = both > m + GROW || (m == -INFINITY && both > m);
            const float f = !grow ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - both);
            if (grow) m = both;
            l *= f;
            if (j > 0) {  // O is at rest: the product of j - 1 came before these scores
#pragma unroll 1
                for (int i = 0; i < DP / 32; i++) {
                    uint32_t o[16];
                    tmem_ld8(to + 16 * i, reinterpret_cast<float *>(o));
                    tmem_ld8(to + 16 * i + 8, reinterpret_cast<float *>(o) + 8);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st16(to + 16 * i, o);
                }
                tmem_wait_st();
            }
            bar_sync(pairs, 64);  // both have read the maxima
            take();
        }
        if (!slow) {
            l += more;
            tmem_st16(sv, pk);
            tmem_st16(sv + 16, pk + 16);
            tmem_wait_st();
        } else {
            // on the CUDA cores, 16 columns of O at a time, over the positions this row sees
#pragma unroll 1
            for (int d = 0; d < DP / 32; d++) {
                const int dd = part * (DP / 32) + d;
                float acc[16];
                const float base = m == -INFINITY ? 0.0f : -m;
                if (j > 0) {
                    tmem_ld8(to + 16 * d, acc);
                    tmem_ld8(to + 16 * d + 8, acc + 8);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[e] = 0.0f;
                }
#pragma unroll 1
                for (int t8 = 0; t8 < BIG_TILE; t8 += 8) {
                    float sc[8];
                    __syncwarp();
                    tmem_ld8(ts + t8, sc);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int t = t8 + e;
                        if (t0 + t >= lim || t0 + t >= p.kv_end) continue;
                        const float w = ex2(__fmaf_rn(sc[e], c, base));
                        if (d == 0 && t / HALF == part) l += w;
#pragma unroll
                        for (int g = 0; g < 2; g++) {
                            const uint4 q4 = *reinterpret_cast<const uint4 *>(v + dd / 4 * BOX64 + t * 128 + (((dd % 4 * 2 + g) ^ (t & 7)) << 4));
                            const __nv_bfloat162 *w2 = reinterpret_cast<const __nv_bfloat162 *>(&q4);
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const float2 vv = __bfloat1622float2(w2[q]);
                                acc[8 * g + 2 * q] += w * vv.x;
                                acc[8 * g + 2 * q + 1] += w * vv.y;
                            }
                        }
                    }
                }
                __syncwarp();
                tmem_st16(to + 16 * d, reinterpret_cast<const uint32_t *>(acc));
            }
            tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[x]);
    }
    sm.stat[x][part][row] = l;
    bar_sync(1 + x * 4 + quarter, 64);
    l += sm.stat[x][part ^ 1][row];
    wait(&sm.o_full[x], s_ph >> 1);
    s_ph ^= 2;
    __syncwarp();
    tc_fence_after();
    const bool valid = row / a.rep < a.tile_tok && tt < p.n_tok;
    const int head = p.kvh * a.rep + row % a.rep;
    const size_t at = (size_t)x * BIG_TILE + row;  // this row in a scratch slot
    if (p.part >= 0) {
#pragma unroll
        for (int i = 0; i < DP / 64; i++) {
            uint32_t o[32];
            tmem_ld32(to + 32 * i, o);
            tmem_wait_ld();
            if (valid) {
                uint4 *dst = reinterpret_cast<uint4 *>(big_part<DP>(a, p.part, part * (DP / 2) + 32 * i, at));
#pragma unroll
                for (int e = 0; e < 8; e++)
                    __stcg(dst + e * (2 * BIG_TILE), make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
            }
        }
        if (valid && part == 0) __stcg(a.big_ml + (size_t)p.part * (2 * BIG_TILE) + at, make_float2(m, l));
    } else {
        const float inv = 1.0f / l;
        bf16 *dst = a.out + (p.tok0 + tt) * a.out_stride + (long long)head * a.head_dim;
#pragma unroll
        for (int i = 0; i < DP / 64; i++) {
            uint32_t o[32];
            tmem_ld32(to + 32 * i, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t w[4];
#pragma unroll
                for (int q = 0; q < 4; q++)
                    w[q] = pack_bf16(__uint_as_float(o[8 * e + 2 * q]) * inv, __uint_as_float(o[8 * e + 2 * q + 1]) * inv);
                const int d = part * (DP / 2) + 32 * i + 8 * e;
                if (valid && d < a.head_dim)  // a row without positions is zero
                    *reinterpret_cast<uint4 *>(dst + d) = lim <= 0 ? make_uint4(0, 0, 0, 0) : make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    tc_fence_before();
    bar_sync(1 + x * 4 + quarter, 64);  // the sums have been read
}

template <int DP>
__global__ void __launch_bounds__(BIG_THREADS, 1)
    paged_big_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ PaArgs a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // no room to align by hand; the declaration's alignment holds for the shared window
    BigSmem<DP> &sm = *reinterpret_cast<BigSmem<DP> *>(smem_raw);
    if (smem_u32(smem_raw) % 1024 != 0) {
        pdl_wait();
        if (threadIdx.x == 0) {
            atomicOr(&g_dev_error, DEV_ERR_TMEM);
            give_ready(a.ready + blockIdx.x);
        }
        return;
    }
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        for (int i = 0; i < BIG_STAGES; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        mbar_init(&sm.q_full, 1);
        mbar_init(&sm.q_empty, 1);
        for (int x = 0; x < 2; x++) {
            mbar_init(&sm.s_full[x], 1);
            mbar_init(&sm.o_full[x], 1);
            mbar_init(&sm.p_full[x], 9);
        }
        fence_barrier_init();
        sm.down = 0;
        prefetch_tmap(&mq);
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    // The next kernel may start once this one's predecessors are done (the kernel for few rows takes that over) and
    // every CTA has its tensor memory: a dependent's CTA that took it first would wait for this kernel while
    // this CTA waits for its memory.
    pdl_wait();
    if (threadIdx.x == 0) give_ready(a.ready + blockIdx.x);
    pdl_trigger();
    const int2 work = a.ctas[PAGED_MAX_CTAS + blockIdx.x];
    if (work.y < 0) zero_rows(a);
    Ring<BIG_STAGES> r;
    Waiter wait(&g_dev_error, &sm.down);
    if (warp < 4) {
        uint32_t q_ph = 0, p_ph = 0;
        const bool first = threadIdx.x % 32 == 0;
        for (int i = 0; i < work.y; i++) {
            const PagedPiece p = a.pieces[work.x + i];
            if (warp % 2 == 0) big_produce<DP>(a, &mq, &mk, &mv, p, sm, r, q_ph, warp / 2, wait);
            else if (warp == 1) big_multiply<DP>(a, p, sm, tmem, r, q_ph, p_ph, wait);
            else if (first) big_ready<DP>(a, p, sm, r, p_ph, wait);
        }
        __syncwarp();
        if (warp == 0) {  // the products' release of the ring arrives asynchronously: before the CTA ends
            for (int i = 0; i < BIG_STAGES; i++) {
                wait(&sm.empty[r.s], r.ph ^ 1);
                r.next();
            }
            wait(&sm.q_empty, q_ph ^ 1);
        }
    } else {
        const int group = warp / 4 - 1;
        uint32_t s_ph = 0;
        for (int i = 0; i < work.y; i++) {
            const PagedPiece p = a.pieces[work.x + i];
            big_softmax<DP>(a, p, sm, tmem, group / 2, group % 2, r, s_ph, wait);
        }
    }
    if (__syncthreads_or(wait.dead)) settle();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------- host

// K or V pages as a 4-D map (column, slot, kv head, page) with a box of `rows` slots of 64 columns.
bool make_page_map(CUtensorMap *map, const void *base, const PagedAttnCall &c, int rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.shape.head_dim, (cuuint64_t)c.shape.page_size, (cuuint64_t)c.shape.n_kv_heads,
                                (cuuint64_t)c.shape.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.cache.pos_stride * 2, (cuuint64_t)c.cache.head_stride * 2,
                                   (cuuint64_t)c.cache.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query rows as a 3-D map (column, head, token): a box is all heads of a kv head for a tile's tokens.
bool make_query_map(CUtensorMap *map, const PagedAttnCall &c, const PaArgs &a) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)c.shape.head_dim, (cuuint64_t)c.shape.n_heads, (cuuint64_t)c.shape.n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)c.shape.head_dim * 2, (cuuint64_t)c.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.rep, (cuuint32_t)a.tile_tok}, estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16 *>(c.q), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int NQ, bool AFTER_BIG = false>
cudaError_t launch_small(const CUtensorMap &mk, const CUtensorMap &mv, const PaArgs &a, cudaStream_t s) {
    const size_t smem = sizeof(SmallSmem<DP, NQ>) + 1024;
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(paged_small_kernel<DP, NQ, AFTER_BIG>), smem);
    if (e != cudaSuccess) return e;
    return launch(paged_small_kernel<DP, NQ, AFTER_BIG>, dim3(paged_ctas()), dim3((SMALL_PRODUCERS + SMALL_WARPS) * 32), smem, s, 1, mk, mv, a);
}

template <int DP>
int run(const PagedAttnCall &c, PaArgs &a, cudaStream_t s) {
    CUtensorMap mk, mv;
    const int small_step = paged_small_step(c.shape), loads = small_step * SMALL_PRODUCERS;
    a.small_box = std::min(a.small_box, small_step);
    a.small_step_pages = loads / a.page_size;
    a.small_step_slots = loads % a.page_size;
    a.big_step_pages = BIG_TILE / a.page_size;
    a.big_step_slots = BIG_TILE % a.page_size;
    if (!make_page_map(&mk, c.cache.key_pages, c, a.small_box) || !make_page_map(&mv, c.cache.value_pages, c, a.small_box))
        return Q3_ERR_SHAPE;
    if (paged_has_big(c.shape)) {
        CUtensorMap mq, mk_big, mv_big;
        if (!make_page_map(&mk_big, c.cache.key_pages, c, a.big_box) || !make_page_map(&mv_big, c.cache.value_pages, c, a.big_box) ||
            !make_query_map(&mq, c, a))
            return Q3_ERR_SHAPE;
        // f32 accumulator, bf16 operands; second product: B = V with its columns contiguous
        const uint32_t kinds = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BIG_TILE >> 4) << 24);
        a.idesc_qk = kinds | ((uint32_t)(BIG_TILE >> 3) << 17) | (c.scale < 0.0f ? 1u << 13 : 0u);
        a.idesc_pv = kinds | ((uint32_t)(DP >> 3) << 17) | (1u << 16);
        const size_t big_smem = sizeof(BigSmem<DP>);
        Q3_TRY_LAUNCH(allow_smem(reinterpret_cast<const void *>(paged_big_kernel<DP>), big_smem));
        Q3_TRY_LAUNCH(launch(paged_big_kernel<DP>, dim3(paged_ctas()), dim3(BIG_THREADS), big_smem, s, 1, mq, mk_big, mv_big, a));
        Q3_TRY_LAUNCH((launch_small<DP, 1, true>(mk, mv, a, s)));  // eight rows (paged_small_rows)
        return Q3_OK;
    }
    const int tiles = paged_small_rows(c.shape) / 8;
    if (tiles == 1) Q3_TRY_LAUNCH((launch_small<DP, 1>(mk, mv, a, s)));
    if (tiles == 2) Q3_TRY_LAUNCH((launch_small<DP, 2>(mk, mv, a, s)));
    if constexpr (DP == 64)
        if (tiles == 3) Q3_TRY_LAUNCH((launch_small<DP, 3>(mk, mv, a, s)));
    return Q3_OK;
}

}  // namespace

unsigned take_error_paged_attn() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v)) != cudaSuccess) return 0;
    if (v) cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return v;
}

int paged_attention(const PagedAttnCall &c, cudaStream_t s) {
    const PagedPlanLayout l = paged_plan_layout(c.shape);
    const PagedScratchLayout x = paged_scratch_layout(c.shape);
    PaArgs a = {};
    a.out = c.out;
    a.q = c.q;
    a.out_stride = c.out_stride;
    a.q_stride = c.q_stride;
    a.table = reinterpret_cast<const int *>(c.plan + l.table);
    a.ctas = reinterpret_cast<const int2 *>(c.plan + l.ctas);
    a.pieces = reinterpret_cast<const PagedPiece *>(c.plan + l.pieces);
    a.splits = reinterpret_cast<const PagedPiece *>(c.plan + l.splits);
    a.counters = reinterpret_cast<int *>(c.plan + l.counters);
    a.ready = reinterpret_cast<int *>(c.plan + l.ready);
    a.small_o = reinterpret_cast<float *>(c.scratch + x.small_o);
    a.small_ml = reinterpret_cast<float2 *>(c.scratch + x.small_ml);
    a.big_o = reinterpret_cast<float *>(c.scratch + x.big_o);
    a.big_ml = reinterpret_cast<float2 *>(c.scratch + x.big_ml);
    a.rep = c.shape.n_heads / c.shape.n_kv_heads;
    a.tile_tok = BIG_TILE / a.rep;
    a.head_dim = c.shape.head_dim;
    a.page_size = c.shape.page_size;
    a.max_pages = c.shape.max_pages;
    a.n_tokens = c.shape.n_tokens;
    a.row_elems = c.shape.n_heads * c.shape.head_dim;
    a.small_box = a.big_box = std::min(c.shape.page_size & -c.shape.page_size, BIG_TILE);
    a.scale_log2 = c.scale * 1.4426950408889634f;
    return a.head_dim <= 64 ? run<64>(c, a, s) : run<128>(c, a, s);
}

}  // namespace q3
