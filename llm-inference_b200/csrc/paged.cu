// Paged serving (include/qwen3_b200.h): the step plan, the append of new tokens with rotary positions, the rotary
// frequencies, and the C entries of these and of the attention over the pages, whose kernels are in paged_attn.cu.
#include <math.h>

#include <algorithm>

#include "paged.cuh"

namespace q3 {
int check_device();

namespace {

__device__ unsigned g_dev_error;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------------------ plan
// One CTA. The description is checked here once, so that the kernels of every layer can use the
// plan's copy of the page table and the token map without checks of their own. Latency bounds it: 10 us for one sequence,
// 17 for 32 of 64 pages, 28 for four chunks of 2048 tokens, 83 for 256 sequences with tables of 2560 pages, once per step.
constexpr int PLAN_THREADS = 1024;

struct PlanArgs {
    char *plan;
    PagedPlanLayout l;
    q3_paged_shape s;
    const int *q_start, *kv_len, *page_table;
    int n_ctas, small_shift, small_rows;  // a small item's step is 1 << small_shift positions
    bool has_big;
};

// Costs, in units of a kind's own: a step of a small item is one, the 16 KB load that it waits for; a 128-position step of
// one or two tensor-core tiles COST_BIG_ONE or COST_BIG_TWO; an item's start and end (queries, merge, output) COST_ITEM or
// COST_BIG_ITEM.
// Items are cut only while each CTA still gets MIN_SHARE or BIG_MIN_SHARE. A unit of the big kind takes BIG_WEIGHT / 2 of the small one's
// time where the two share the SMs: with 31 decodes and a chunk of 333 tokens, 1 to 4 and 5.5 gave 178, 107, 89, 88, 96 us
// (105 one after the other), with 32 decodes at 4096 and a chunk of 2048 at 8192 425, 370, 334, 400, 480 (376).
constexpr int COST_ITEM = 3, COST_BIG_ITEM = 6, COST_BIG_ONE = 2, COST_BIG_TWO = 3, MIN_SHARE = 10, BIG_MIN_SHARE = 6, BIG_WEIGHT = 6;

// The items of sequence q: a big one has n_q per kv head.
struct SeqItems {
    bool big;
    int n_q, span;  // items per kv head, tokens of each
    __device__ __forceinline__ int ends() const { return big ? COST_BIG_ITEM : COST_ITEM; }
};

// A step without the kernel for many rows may still describe a sequence with more of them than it may have. It
// has no positions then, but its rows are written: as items of what a small one holds.
__device__ __forceinline__ SeqItems seq_items(const PagedSeq &q, int rep, const PlanArgs &a) {
    SeqItems s;
    s.big = a.has_big && (long long)q.q_len * rep > a.small_rows;
    s.span = s.big ? 2 * (BIG_TILE / rep) : max(1, a.small_rows / rep);
    s.n_q = q.q_len == 0 ? 0 : (q.q_len + s.span - 1) / s.span;
    return s;
}

// Item i's positions end here, it has this many steps, and each costs this much.
__device__ __forceinline__ void item_steps(const PagedSeq &q, const SeqItems &s, int i, int shift, int *end, int *n, int *cost) {
    const int last = min((i + 1) * s.span, q.q_len);
    *end = max(0, q.kv_len - q.q_len + last);
    *n = max(1, (*end + (1 << shift) - 1) >> shift);
    *cost = !s.big ? 1 : last - i * s.span > s.span / 2 ? COST_BIG_TWO : COST_BIG_ONE;
}

// Steps of an item that lie before cost r of it; its ends come first.
__device__ __forceinline__ int steps_before(long long r, int ends, int n, int cost) {
    return (int)max(0ll, min((long long)n, (r - ends + cost - 1) / cost));
}

// Exclusive prefix sum of v[0 .. n) in place by the whole CTA; returns the total.
__device__ long long scan(long long *v, int n, long long *warp_sums) {
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS;
    long long mine = 0;
    for (int i = tid * per; i < min(n, (tid + 1) * per); i++) mine += v[i];
    long long sum = mine;
    for (int off = 1; off < 32; off *= 2) {
        const long long o = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += o;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    long long before = 0, total = 0;
    for (int w = 0; w < PLAN_THREADS / 32; w++) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    before += sum - mine;
    for (int i = tid * per; i < min(n, (tid + 1) * per); i++) {
        const long long x = v[i];
        v[i] = before;
        before += x;
    }
    __syncthreads();
    return total;
}

__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ __align__(16) unsigned char plan_smem[];
    long long *big_s = reinterpret_cast<long long *>(plan_smem);  // cost before each sequence's big items
    long long *small_s = big_s + a.s.n_seqs + 1;                  // and before its small ones
    long long *item_s = small_s + a.s.n_seqs + 1;                 // items before: big ones << 32 | small ones
    int *start_s = reinterpret_cast<int *>(item_s + a.s.n_seqs + 1);
    int *kv_s = start_s + a.s.n_seqs + 1;
    __shared__ long long sums_s[PLAN_THREADS / 32];
    pdl_trigger();
    pdl_wait();
    const int n = a.s.n_seqs, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    int *table = reinterpret_cast<int *>(a.plan + a.l.table);
    int4 *toks = reinterpret_cast<int4 *>(a.plan + a.l.toks);

    for (int i = tid; i <= n; i += PLAN_THREADS) start_s[i] = a.q_start[i];
    __syncthreads();
    bool falls = false;
    for (int i = tid; i <= n; i += PLAN_THREADS)
        falls |= start_s[i] < 0 || start_s[i] > a.s.n_tokens || (i > 0 && start_s[i] < start_s[i - 1]);
    const bool bad_starts = __syncthreads_or(falls);

    for (int b = warp; b < n; b += PLAN_THREADS / 32) {  // a warp checks a sequence's pages
        const int q0 = start_s[b], q_len = start_s[b + 1] - q0, kv = a.kv_len[b];
        const int used = (int)min(((long long)kv + a.s.page_size - 1) / a.s.page_size, (long long)a.s.max_pages);
        bool bad = bad_starts || q_len > a.s.max_q_len || kv < 0 || kv > (long long)a.s.max_pages * a.s.page_size;
        for (int i = lane; i < a.s.max_pages; i += 32) {
            int page = -1;
            if (i < used && !bad) {
                page = a.page_table[(size_t)b * a.s.max_pages + i];
                if (page < 0 || page >= a.s.n_pages) {
                    bad = true;
                    page = -1;
                }
            }
            table[(size_t)b * a.s.max_pages + i] = page;
        }
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) {
            if (bad) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
            kv_s[b] = bad ? 0 : kv;
        }
    }
    __syncthreads();
    auto seq = [&](int b) -> PagedSeq {
        return bad_starts ? PagedSeq{0, 0, 0} : PagedSeq{start_s[b], start_s[b + 1] - start_s[b], kv_s[b]};
    };
    for (int t = tid; t < a.s.n_tokens; t += PLAN_THREADS) {
        int4 tok = make_int4(-1, bad_starts ? PAGED_PADDING : PAGED_OUTSIDE, -1, -1);
        if (!bad_starts && n > 0 && t >= start_s[0] && t < start_s[n]) {
            int lo = 0, hi = n - 1;  // the last sequence that starts at or before t and is not empty there
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (start_s[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const PagedSeq q = seq(lo);
            const int pos = q.kv_len - q.q_len + (t - q.q0);
            tok.x = lo;
            tok.y = pos < 0 ? PAGED_PADDING : pos + 1;
            if (pos >= 0) {
                tok.z = table[(size_t)lo * a.s.max_pages + pos / a.s.page_size];
                tok.w = pos % a.s.page_size;
            }
        }
        toks[t] = tok;
    }

    // ---- work
    const int rep = a.s.n_heads / a.s.n_kv_heads, kvh = a.s.n_kv_heads;
    constexpr int BIG_SHIFT = 7;
    static_assert(1 << BIG_SHIFT == BIG_TILE, "a step of a big item");
    for (int b = tid; b < n; b += PLAN_THREADS) {
        const PagedSeq q = seq(b);
        const SeqItems s = seq_items(q, rep, a);
        long long cost = 0;
        for (int i = 0; i < s.n_q; i++) {
            int end, steps, c;
            item_steps(q, s, i, s.big ? BIG_SHIFT : a.small_shift, &end, &steps, &c);
            cost += s.ends() + (long long)steps * c;
        }
        big_s[b] = s.big ? cost * kvh : 0;
        small_s[b] = s.big ? 0 : cost * kvh;
        item_s[b] = (long long)s.n_q * kvh << (s.big ? 32 : 0);
    }
    __syncthreads();
    const long long items = scan(item_s, n, sums_s);
    const int n_items[2] = {(int)(items & 0xffffffff), (int)(items >> 32)};
    const long long total_big = scan(big_s, n, sums_s), total_small = scan(small_s, n, sums_s);
    if (tid == 0) {
        big_s[n] = total_big;
        small_s[n] = total_small;
    }
    __syncthreads();
    int2 *ctas = reinterpret_cast<int2 *>(a.plan + a.l.ctas);
    PagedPiece *pieces = reinterpret_cast<PagedPiece *>(a.plan + a.l.pieces);
    PagedPiece *splits = reinterpret_cast<PagedPiece *>(a.plan + a.l.splits);
    int *counters = reinterpret_cast<int *>(a.plan + a.l.counters), *ready = reinterpret_cast<int *>(a.plan + a.l.ready);
    // The two kernels of a step with items of both kinds run side by side: the big one's CTAs first, the small
    // one's on the SMs that those leave: tensor-core work beside loads, and memory bandwidth is not for want of SMs.
    const long long weight = total_big * BIG_WEIGHT / 2;
    const int share = total_big > 0 && total_small > 0
                          ? (int)max(1ll, min((long long)a.n_ctas - 1, a.n_ctas * weight / (weight + total_small)))
                          : a.n_ctas;
    // Items are cut where there are CTAs to spare and every piece still gets its least share; in equal numbers of pieces, if
    // that leaves no more than a tenth of the CTAs without work (32 sequences' decodes with 532 tokens at 1389: 28 us, 39
    // otherwise; the geometric mean of 36 random batches is 1 % less). Least shares of 6, 8, 10, 12 and 16 for big items: 17.2,
    // 18.2, 18.7, 20 and 21 us for 14 decodes with 31 tokens at 3995; of 8, 10 and 16 for small ones: 16.2, 11.5 and 11.7 us
    // for 3 draft tokens of 4 sequences at 1000, 10.1, 9.7 and 11.5 for one token of one sequence in the thousands.
    auto ctas_used = [&](int most, bool big) {
        const int n_of = max(1, n_items[big]);
        const long long shares = big ? total_big / BIG_MIN_SHARE : total_small / MIN_SHARE;
        if (shares < 2 * n_of) return min(most, n_of);
        const int used = (int)min((long long)most, shares), even = used / n_of * n_of;
        return 10 * even >= 9 * used ? even : used;
    };
    const int used_big = ctas_used(share, true);
    const int used_small = ctas_used(total_big > 0 ? max(1, a.n_ctas - used_big) : a.n_ctas, false);
    // A CTA's pieces start at (items before its first) + (CTAs before it): every cut adds one piece at most.
    for (int id = tid; id < 2 * a.n_ctas; id += PLAN_THREADS) {
        const bool big = id >= a.n_ctas;
        const int c = big ? id - a.n_ctas : id, shift = big ? BIG_SHIFT : a.small_shift;
        const long long total = big ? total_big : total_small;
        const long long *pre = big ? big_s : small_s;
        const int used = big ? used_big : used_small;
        auto bound = [&](int i) { return total * i / used; };
        const long long u0 = c < used ? bound(c) : total, u1 = c < used ? bound(c + 1) : total;
        int count = 0, first_piece = -1;
        PagedPiece split = {};
        long long u = u0, start = u0;  // of the item
        int lo = 0, head = 0, i = 0;
        PagedSeq q = {};
        SeqItems s = {};
        if (u < u1) {  // the item that holds u0; then one after the other
            int hi = n - 1;  // the last sequence that starts at or before u
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (pre[mid] <= u) lo = mid;
                else hi = mid - 1;
            }
            q = seq(lo);
            s = seq_items(q, rep, a);
            const long long per_head = (pre[lo + 1] - pre[lo]) / kvh;
            head = (int)((u - pre[lo]) / per_head);
            start = pre[lo] + head * per_head;
        }
        while (u < u1) {
            int end, steps, cost;
            long long len;
            for (;;) {  // all lanes look first, then all write
                item_steps(q, s, i, shift, &end, &steps, &cost);
                len = s.ends() + (long long)steps * cost;
                if (u < start + len) break;
                start += len;
                if (++i < s.n_q) continue;
                i = 0;
                if (++head < kvh) continue;
                head = 0;
                do lo++;
                while (pre[lo + 1] == pre[lo]);  // u < total: there is one
                q = seq(lo);
                s = seq_items(q, rep, a);
            }
            const int t0 = steps_before(u - start, s.ends(), steps, cost);
            const int t1 = u1 >= start + len ? steps : steps_before(u1 - start, s.ends(), steps, cost);
            if (t1 > t0) {
                PagedPiece p;
                p.seq = lo;
                p.kvh = head;
                p.tok0 = q.q0 + i * s.span;
                p.n_tok = min(s.span, q.q_len - i * s.span);
                p.kv0 = t0 << shift;
                p.kv1 = t1 == steps ? end : t1 << shift;
                p.kv_end = end;
                p.pos0 = q.kv_len - q.q_len + i * s.span;
                p.part = -1;
                p.first = c;
                p.n_parts = 1;
                if (t0 > 0 || t1 < steps) {
                    int f = c;
                    while (steps_before(bound(f) - start, s.ends(), steps, cost) > 0) f--;
                    p.first = f;
                    while (f + 1 < used && bound(f + 1) < start + len && steps_before(bound(f + 1) - start, s.ends(), steps, cost) < steps) f++;
                    p.n_parts = f - p.first + 1;
                    p.part = part_slot(p.first, c - p.first);
                    if (t0 == 0 && p.n_parts > 1) split = p;
                }
                if (first_piece < 0)
                    first_piece = (big ? n_items[0] + a.n_ctas + (int)(item_s[lo] >> 32) : (int)(item_s[lo] & 0xffffffff)) +
                                  head * s.n_q + i + c;
                pieces[first_piece + count] = p;
                count++;
            }
            u = start + len;
        }
        ctas[(big ? PAGED_MAX_CTAS : 0) + c] = make_int2(max(first_piece, 0), bad_starts ? -1 : count);
        if (big) splits[c] = split;
        else counters[c] = ready[c] = 0;
    }
}

// ------------------------------------------------------------------ append
// One CTA per token: 128 threads that take the heads in rounds where tokens are many, a group of lanes for every head
// (up to 512 threads) where they are few. A unit is two 8-element chunks of a head that one lane holds in
// registers: for half-split pairs chunk u and its partner u + rope_dim/16, so a pair's two elements sit in one
// lane; otherwise u and u + lph. A head is a group of `lph` lanes (a power of two), so the sum of squares is a few
// shuffles. The angles depend on the token alone: the CTA computes them once, into shared memory, where lanes read
// theirs for every head (held in registers they cost occupancy: 44 us against 40.5). A lane's first query head is
// asked for before that.
//
// With many tokens the instructions bound it about as much as the bytes: 8192 tokens of 48 heads of 128 take 37.5 us
// (5.4 TB/s, 0.83 of the measured copy bandwidth), interleaved 39 to 40 (61 with angles in the pairs' order, whose reads
// met in a few banks); without packed arithmetic and a loop per kind of head it was 43. With few, the chain plan ->
// angle -> heads: 2.4 us for one token.
//
// The angle is reduced in fp64: pos * inv_freq reaches 10^5 rad and more, where an fp32 product is
// off by up to 2^-25 of itself, more than a bf16 result may be. turns = pos * inv_freq / 2 pi, its
// nearest integer dropped, goes to sincospif.
constexpr int APPEND_MAX_THREADS = 512, APPEND_THREADS = 128;
constexpr int APPEND_ODD_THREADS = 128;

struct AppendArgs {
    bf16 *q_out;
    const bf16 *q, *k, *v;
    const bf16 *q_norm_w, *k_norm_w;
    const float *inv_freq;
    bf16 *key_pages, *value_pages;
    long long q_out_stride, q_stride, k_stride, v_stride, page_stride, head_stride, pos_stride;
    const int4 *toks;
    int n_heads, n_kv_heads, head_dim, rope_dim, lph;
    float eps, amplitude;
};

// eight bf16 as four pairs of floats, and back
__device__ __forceinline__ void unpack8(const uint4 &u, uint64_t *f) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}

__device__ __forceinline__ uint4 pack8(const uint64_t *f) {
    uint4 u;
    __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 v = unpair(f[i]);
        h[i] = __floats2bfloat162_rn(v.x, v.y);
    }
    return u;
}

__device__ __forceinline__ void rope_angle(int pos, float inv_freq, float amplitude, float *c, float *s) {
    const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;  // 1 / 2 pi
    float cs, sn;
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
    *c = cs * amplitude;
    *s = sn * amplitude;
}

template <bool INTERLEAVED>
__global__ void __launch_bounds__(APPEND_MAX_THREADS, 2) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    // cos and sin of pair j: (cos, cos) and (-sin, sin) interleaved; half split cos and sin, for two pairs at a time.
    // Laid out so that the lanes of a group read 16 bytes each side by side: a lane's first 16 bytes of all lanes,
    // then the second ones.
    __shared__ __align__(16) float cos_s[PAGED_MAX_HEAD_DIM], sin_s[PAGED_MAX_HEAD_DIM];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, groups = blockDim.x / a.lph, first = threadIdx.x / a.lph, step = groups * a.head_dim;
    const int u = threadIdx.x % a.lph, half = a.rope_dim / 2, nc = a.head_dim / 8, hc = INTERLEAVED ? 0 : half / 8;
    const int c0 = INTERLEAVED || u < hc ? u : 2 * u;  // half split, units past the rotated pairs: chunks 2u, 2u + 1
    const int c1 = INTERLEAVED ? u + a.lph : u < hc ? u + hc : c0 + 1;
    const bool in0 = c0 < nc, in1 = c1 < nc;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto load = [&](const bf16 *src, bool on, uint4 &r0, uint4 &r1) {
        r0 = on && in0 ? reinterpret_cast<const uint4 *>(src)[c0] : zero;
        r1 = on && in1 ? reinterpret_cast<const uint4 *>(src)[c1] : zero;
    };
    auto store = [&](bf16 *dst, const uint4 &r0, const uint4 &r1) {
        if (in0) reinterpret_cast<uint4 *>(dst)[c0] = r0;
        if (in1) reinterpret_cast<uint4 *>(dst)[c1] = r1;
    };
    const bf16 *src = a.q + t * a.q_stride + first * a.head_dim;
    uint4 n0, n1;
    load(src, first < a.n_heads, n0, n1);
    const int4 tok = a.toks[t];
    const int pos = tok.y - 1;
    if (tok.y == PAGED_OUTSIDE) return;
    bf16 *dst = a.q_out + t * a.q_out_stride + first * a.head_dim;
    if (pos < 0) {  // padding: zero query rows, nothing stored
        for (int h = first; h < a.n_heads; h += groups, dst += step) store(dst, zero, zero);
        return;
    }
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        float cs, sn;
        rope_angle(pos, a.inv_freq[j], a.amplitude, &cs, &sn);
        if (INTERLEAVED) {
            const int at = (j % 4 / 2 * 16 + j / 4) * 2 + j % 2;
            reinterpret_cast<float2 *>(cos_s)[at] = make_float2(cs, cs);
            reinterpret_cast<float2 *>(sin_s)[at] = make_float2(-sn, sn);
        } else {
            const int at = (j % 8 / 4 * 8 + j / 8) * 4 + j % 4;
            cos_s[at] = cs;
            sin_s[at] = sn;
        }
    }
    __syncthreads();
    const unsigned group = ((1u << a.lph) - 1) << (threadIdx.x % 32 / a.lph * a.lph);
    const float inv_dim = 1.0f / a.head_dim;
    // one head: norm with weights w (if there are any), rotation, one rounding
    auto turn = [&](uint4 &r0, uint4 &r1, const bf16 *w) {
        uint64_t x[8];
        unpack8(r0, x);
        unpack8(r1, x + 4);
        if (w != nullptr) {  // uniform over q heads and over k heads, whose groups of lanes may share a warp
            uint64_t sq = mul2(x[0], x[0]);
#pragma unroll
            for (int i = 1; i < 8; i++) sq = fma2(x[i], x[i], sq);
            float sum = unpair(sq).x + unpair(sq).y;
            for (int off = a.lph / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(group, sum, off);
            const float inv = rsqrtf(sum * inv_dim + a.eps);
            uint4 g0, g1;
            load(w, true, g0, g1);
            uint64_t g[4];
            unpack8(g0, g);
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = mul2(mul2(x[i], pair(inv, inv)), g[i]);
            unpack8(g1, g);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 + i] = mul2(mul2(x[4 + i], pair(inv, inv)), g[i]);
        }
        if (INTERLEAVED) {
            const ulonglong2 *c = reinterpret_cast<const ulonglong2 *>(cos_s), *s = reinterpret_cast<const ulonglong2 *>(sin_s);
#pragma unroll
            for (int i = 0; i < 4; i++) {  // chunk c0's two pairs of pairs, then c1's
                const int at = i % 2 * 16 + (i < 2 ? c0 : c1);
                if (i < 2 ? !in0 : !in1) continue;
                const ulonglong2 cc = c[at], ss = s[at];
                const float2 v = unpair(x[2 * i]), w = unpair(x[2 * i + 1]);
                const int at_pair = 4 * (i < 2 ? c0 : c1) + i % 2 * 2;  // pairs from `half` on stay as they are, NaN or not
                if (at_pair < half) x[2 * i] = fma2(pair(v.y, v.x), ss.x, mul2(x[2 * i], cc.x));
                if (at_pair + 1 < half) x[2 * i + 1] = fma2(pair(w.y, w.x), ss.y, mul2(x[2 * i + 1], cc.y));
            }
        } else if (u < hc) {
            const ulonglong2 *c = reinterpret_cast<const ulonglong2 *>(cos_s) + u, *s = reinterpret_cast<const ulonglong2 *>(sin_s) + u;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const ulonglong2 cc = c[8 * i], ss = s[8 * i];
                constexpr unsigned long long SIGNS = 0x8000000080000000ull;
                const ulonglong2 nn = make_ulonglong2(ss.x ^ SIGNS, ss.y ^ SIGNS);
                const uint64_t e0 = x[2 * i], o0 = x[4 + 2 * i], e1 = x[2 * i + 1], o1 = x[5 + 2 * i];
                x[2 * i] = fma2(o0, nn.x, mul2(e0, cc.x));
                x[4 + 2 * i] = fma2(e0, ss.x, mul2(o0, cc.x));
                x[2 * i + 1] = fma2(o1, nn.y, mul2(e1, cc.y));
                x[5 + 2 * i] = fma2(e1, ss.y, mul2(o1, cc.y));
            }
        }
        r0 = pack8(x);
        r1 = pack8(x + 4);
    };
    // key and value heads go to the groups from the other end, so that none has two heads more than another
    int kv = groups - 1 - first;
    auto kv_load = [&](int i) {
        load(i < a.n_kv_heads ? a.k + t * a.k_stride + i * a.head_dim : a.v + t * a.v_stride + (i - a.n_kv_heads) * a.head_dim,
             i < 2 * a.n_kv_heads, n0, n1);
    };
    if (first >= a.n_heads) kv_load(kv);
    for (int h = first; h < a.n_heads; h += groups) {
        uint4 r0 = n0, r1 = n1;
        src += step;
        if (h + groups < a.n_heads) load(src, true, n0, n1);
        else kv_load(kv);
        turn(r0, r1, a.q_norm_w);
        store(dst, r0, r1);
        dst += step;
    }
    const long long slot = tok.z * a.page_stride + tok.w * a.pos_stride;
    for (; kv < 2 * a.n_kv_heads; kv += groups) {
        uint4 r0 = n0, r1 = n1;
        if (kv + groups < 2 * a.n_kv_heads) kv_load(kv + groups);
        if (kv < a.n_kv_heads) {
            turn(r0, r1, a.k_norm_w);
            store(a.key_pages + slot + kv * a.head_stride, r0, r1);
        } else {
            store(a.value_pages + slot + (kv - a.n_kv_heads) * a.head_stride, r0, r1);
        }
    }
}

// Half-split pairs whose distance is not a multiple of 8 elements: one warp per head, the head's
// fp32 values in the warp's shared memory. Two-byte accesses, and no head's loads ahead of the one before: 8192 tokens
// of 48 heads of 128, 40 elements rotated, take 107 us where the kernel above takes 39 with 48 of them.
__global__ void __launch_bounds__(APPEND_ODD_THREADS) paged_append_odd_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ float cos_s[PAGED_MAX_HEAD_DIM / 2], sin_s[PAGED_MAX_HEAD_DIM / 2];
    __shared__ float head_s[APPEND_ODD_THREADS / 32][PAGED_MAX_HEAD_DIM];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, lane = threadIdx.x % 32;
    const int4 tok = a.toks[t];
    const int pos = tok.y - 1, D = a.head_dim, half = a.rope_dim / 2;
    if (tok.y == PAGED_OUTSIDE) return;
    for (int j = threadIdx.x; j < half; j += APPEND_ODD_THREADS)
        if (pos >= 0) rope_angle(pos, a.inv_freq[j], a.amplitude, &cos_s[j], &sin_s[j]);
    __syncthreads();
    float *x = head_s[threadIdx.x / 32];
    for (int h = threadIdx.x / 32; h < a.n_heads + 2 * a.n_kv_heads; h += APPEND_ODD_THREADS / 32) {
        const int kh = h - a.n_heads, vh = kh - a.n_kv_heads;
        if (pos < 0) {
            if (kh < 0)
                for (int d = lane; d < D; d += 32)
                    a.q_out[t * a.q_out_stride + (long long)h * D + d] = __float2bfloat16(0.0f);
            continue;
        }
        const long long slot = tok.z * a.page_stride + tok.w * a.pos_stride;
        if (vh >= 0) {
            for (int d = lane; d < D; d += 32)
                a.value_pages[slot + vh * a.head_stride + d] = a.v[t * a.v_stride + (long long)vh * D + d];
            continue;
        }
        const bf16 *src = kh < 0 ? a.q + t * a.q_stride + (long long)h * D : a.k + t * a.k_stride + (long long)kh * D;
        bf16 *dst = kh < 0 ? a.q_out + t * a.q_out_stride + (long long)h * D : a.key_pages + slot + kh * a.head_stride;
        const bf16 *w = kh < 0 ? a.q_norm_w : a.k_norm_w;
        float sum = 0.0f;
        for (int d = lane; d < D; d += 32) {
            const float v = __bfloat162float(src[d]);
            x[d] = v;
            sum = __fmaf_rn(v, v, sum);
        }
        if (w != nullptr) {
            for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            const float inv = rsqrtf(sum / D + a.eps);
            for (int d = lane; d < D; d += 32) x[d] = x[d] * inv * __bfloat162float(w[d]);
        }
        __syncwarp();
        for (int d = lane; d < D; d += 32) {
            float y = x[d];
            if (d < half) y = x[d] * cos_s[d] - x[d + half] * sin_s[d];
            else if (d < 2 * half) y = x[d] * cos_s[d - half] + x[d - half] * sin_s[d - half];
            dst[d] = __float2bfloat16(y);
        }
        __syncwarp();
    }
}

}  // namespace

unsigned take_error_paged_attn();

unsigned take_error_paged() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v)) != cudaSuccess) return 0;
    if (v) cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return v | take_error_paged_attn();
}

int paged_shape_check(const q3_paged_shape *s) {
    if (!s) return Q3_ERR_ARG;
    if (s->n_seqs < 0 || s->n_seqs > PAGED_MAX_SEQS || s->n_tokens < 0 || s->max_q_len < 0) return Q3_ERR_SHAPE;
    if (s->n_heads <= 0 || s->n_kv_heads <= 0 || s->n_heads % s->n_kv_heads != 0 || s->n_heads / s->n_kv_heads > 128)
        return Q3_ERR_SHAPE;
    if (s->head_dim <= 0 || s->head_dim % 8 != 0 || s->head_dim > PAGED_MAX_HEAD_DIM) return Q3_ERR_SHAPE;
    if (s->page_size <= 0 || s->page_size % 8 != 0 || s->n_pages <= 0 || s->max_pages <= 0) return Q3_ERR_SHAPE;
    // a position, and the index of a page-table entry, fit an int
    if ((long long)s->max_pages * s->page_size > (1ll << 30) || (long long)s->n_seqs * s->max_pages > (1ll << 30))
        return Q3_ERR_SHAPE;
    return Q3_OK;
}

namespace {
int cache_check(const q3_paged_cache *c) {
    if (!c || !c->key_pages || !c->value_pages) return Q3_ERR_ARG;
    if (c->page_stride <= 0 || c->head_stride <= 0 || c->pos_stride <= 0) return Q3_ERR_SHAPE;
    if (!aligned16(c->key_pages) || !aligned16(c->value_pages) || c->page_stride % 8 || c->head_stride % 8 || c->pos_stride % 8)
        return Q3_ERR_ALIGN;
    return Q3_OK;
}

// a row tensor: 16-byte aligned rows, at least `width` elements apart
int rows_check(const void *p, long long stride, long long width) {
    if (!p) return Q3_ERR_ARG;
    if (stride < width) return Q3_ERR_SHAPE;
    return !aligned16(p) || stride % 8 ? Q3_ERR_ALIGN : Q3_OK;
}
}  // namespace

}  // namespace q3

using namespace q3;

#define TRY(expr)                     \
    do {                              \
        int st_ = (expr);             \
        if (st_ != Q3_OK) return st_; \
    } while (0)

extern "C" {

size_t q3_paged_plan_bytes(const q3_paged_shape *shape) {
    return paged_shape_check(shape) == Q3_OK ? std::max<size_t>(paged_plan_layout(*shape).bytes, 256) : 0;
}

size_t q3_paged_attention_scratch_bytes(const q3_paged_shape *shape) {
    return paged_shape_check(shape) == Q3_OK ? paged_scratch_layout(*shape).bytes : 0;
}

int q3_paged_plan(void *plan, const q3_paged_shape *shape, const int *q_start, const int *kv_len,
                  const int *page_table, void *stream) {
    TRY(paged_shape_check(shape));
    if (!plan || !q_start || (shape->n_seqs > 0 && (!kv_len || !page_table))) return Q3_ERR_ARG;
    if (!aligned16(plan)) return Q3_ERR_ALIGN;
    TRY(check_device());
    PlanArgs a = {static_cast<char *>(plan), paged_plan_layout(*shape), *shape, q_start, kv_len, page_table,
                  paged_ctas(), __builtin_ctz(paged_small_step(*shape)), paged_small_rows(*shape), paged_has_big(*shape)};
    const size_t smem = (size_t)(shape->n_seqs + 1) * (3 * sizeof(long long) + 2 * sizeof(int));
    Q3_TRY_LAUNCH(allow_smem(reinterpret_cast<const void *>(paged_plan_kernel), smem));
    Q3_TRY_LAUNCH(launch(paged_plan_kernel, dim3(1), dim3(PLAN_THREADS), smem, (cudaStream_t)stream, 1, a));
    return Q3_OK;
}

int q3_paged_rope_append(q3_bf16 *q_out, long long q_out_stride, const q3_bf16 *q, long long q_stride,
                         const q3_bf16 *k, long long k_stride, const q3_bf16 *v, long long v_stride,
                         const q3_bf16 *q_norm_w, const q3_bf16 *k_norm_w, float eps, const float *inv_freq,
                         int rope_dim, int interleaved, float amplitude, const q3_paged_cache *cache,
                         const q3_paged_shape *shape, const void *plan, void *stream) {
    TRY(paged_shape_check(shape));
    const q3_paged_shape &s = *shape;
    const long long qd = (long long)s.n_heads * s.head_dim, kd = (long long)s.n_kv_heads * s.head_dim;
    if (s.n_tokens == 0) return Q3_OK;  // before the pointers: tensors of no elements have none
    if (!plan) return Q3_ERR_ARG;
    TRY(rows_check(q_out, q_out_stride, qd));
    TRY(rows_check(q, q_stride, qd));
    TRY(rows_check(k, k_stride, kd));
    TRY(rows_check(v, v_stride, kd));
    TRY(cache_check(cache));
    if (rope_dim < 0 || rope_dim > s.head_dim || rope_dim % 2 != 0) return Q3_ERR_SHAPE;
    if (rope_dim > 0 && !inv_freq) return Q3_ERR_ARG;
    if (q_out == q && q_out_stride != q_stride) return Q3_ERR_SHAPE;
    if (!aligned16(q_norm_w) || !aligned16(k_norm_w) || !aligned16(plan)) return Q3_ERR_ALIGN;
    TRY(check_device());
    AppendArgs a;
    a.q_out = (bf16 *)q_out;
    a.q = (const bf16 *)q;
    a.k = (const bf16 *)k;
    a.v = (const bf16 *)v;
    a.q_norm_w = (const bf16 *)q_norm_w;
    a.k_norm_w = (const bf16 *)k_norm_w;
    a.inv_freq = inv_freq;
    a.key_pages = (bf16 *)cache->key_pages;
    a.value_pages = (bf16 *)cache->value_pages;
    a.q_out_stride = q_out_stride;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.page_stride = cache->page_stride;
    a.head_stride = cache->head_stride;
    a.pos_stride = cache->pos_stride;
    a.toks = reinterpret_cast<const int4 *>(static_cast<const char *>(plan) + paged_plan_layout(s).toks);
    a.n_heads = s.n_heads;
    a.n_kv_heads = s.n_kv_heads;
    a.head_dim = s.head_dim;
    a.rope_dim = rope_dim;
    a.eps = eps;
    a.amplitude = amplitude;
    const int chunks = s.head_dim / 8, hc = interleaved ? 0 : rope_dim / 16;
    const int units = hc + (chunks - 2 * hc + 1) / 2;
    for (a.lph = 1; a.lph < units;) a.lph *= 2;
    cudaStream_t st = (cudaStream_t)stream;
    const int most = s.n_tokens >= 2 * num_sms() ? APPEND_THREADS : APPEND_MAX_THREADS;
    const int heads = s.n_heads + 2 * s.n_kv_heads, rounds = (heads * a.lph + most - 1) / most;
    const dim3 grid(s.n_tokens), block(((heads + rounds - 1) / rounds * a.lph + 31) / 32 * 32);
    if (interleaved) Q3_TRY_LAUNCH(launch(paged_append_kernel<true>, grid, block, 0, st, 1, a));
    else if (rope_dim % 16 == 0) Q3_TRY_LAUNCH(launch(paged_append_kernel<false>, grid, block, 0, st, 1, a));
    else Q3_TRY_LAUNCH(launch(paged_append_odd_kernel, dim3(s.n_tokens), dim3(APPEND_ODD_THREADS), 0, st, 1, a));
    return Q3_OK;
}

int q3_paged_attention(q3_bf16 *out, long long out_stride, const q3_bf16 *q, long long q_stride,
                       const q3_paged_cache *cache, float scale, const q3_paged_shape *shape, void *plan,
                       void *scratch, void *stream) {
    TRY(paged_shape_check(shape));
    const q3_paged_shape &s = *shape;
    const long long qd = (long long)s.n_heads * s.head_dim;
    if (s.n_tokens == 0 || s.n_seqs == 0) return Q3_OK;  // before the pointers: tensors of no elements have none
    if (!plan || !scratch) return Q3_ERR_ARG;
    TRY(rows_check(out, out_stride, qd));
    TRY(rows_check(q, q_stride, qd));
    TRY(cache_check(cache));
    if (!aligned16(plan) || !aligned16(scratch)) return Q3_ERR_ALIGN;
    TRY(check_device());
    const PagedAttnCall c = {(bf16 *)out, (const bf16 *)q, out_stride, q_stride, *cache, scale, s,
                             static_cast<char *>(plan), static_cast<char *>(scratch)};
    return paged_attention(c, (cudaStream_t)stream);
}

int q3_rope_inv_freq(float *inv_freq, float *amplitude, int rope_dim, float theta, const q3_rope_scaling *scaling) {
    if (!inv_freq || !amplitude) return Q3_ERR_ARG;
    if (rope_dim <= 0 || rope_dim % 2 != 0 || !(theta > 1.0f)) return Q3_ERR_SHAPE;
    q3_rope_scaling sc = {};
    if (scaling) sc = *scaling;
    const double pi = 3.14159265358979323846;
    const bool parts = sc.kind == Q3_ROPE_BY_PARTS, yarn = sc.kind == Q3_ROPE_YARN;
    if (sc.kind < Q3_ROPE_PLAIN || sc.kind > Q3_ROPE_YARN) return Q3_ERR_ARG;
    if (sc.kind != Q3_ROPE_PLAIN && !(sc.factor >= 1.0f && std::isfinite(sc.factor))) return Q3_ERR_SHAPE;
    if ((parts || yarn) && sc.original_max <= 0) return Q3_ERR_SHAPE;
    if (parts && !(sc.low_freq_factor > 0 && sc.high_freq_factor > sc.low_freq_factor)) return Q3_ERR_SHAPE;
    if (yarn && !(sc.beta_slow > 0 && sc.beta_fast > sc.beta_slow && sc.attention_factor >= 0)) return Q3_ERR_SHAPE;
    // YaRN: pair j turns original_max * theta^(-2j/d) / 2 pi times; the j that turns beta times
    auto pair_of = [&](double beta) {
        return rope_dim * log(sc.original_max / (beta * 2 * pi)) / (2 * log((double)theta));
    };
    const double low = yarn ? std::max(floor(pair_of(sc.beta_fast)), 0.0) : 0.0;
    const double high = yarn ? std::min(ceil(pair_of(sc.beta_slow)), (double)(rope_dim - 1)) : 1.0;
    for (int j = 0; j < rope_dim / 2; j++) {
        double f = pow((double)theta, -2.0 * j / rope_dim);
        double keep = 1.0;  // share of the unscaled frequency
        if (sc.kind == Q3_ROPE_LINEAR) keep = 0.0;
        if (parts)
            keep = std::min(1.0, std::max(0.0, (sc.original_max * f / (2 * pi) - sc.low_freq_factor) /
                                                   ((double)sc.high_freq_factor - sc.low_freq_factor)));
        if (yarn) keep = 1.0 - std::min(1.0, std::max(0.0, (j - low) / std::max(high - low, 0.001)));
        if (sc.kind != Q3_ROPE_PLAIN) f = keep * f + (1.0 - keep) * f / sc.factor;
        inv_freq[j] = (float)f;
    }
    *amplitude = !yarn ? 1.0f : sc.attention_factor > 0 ? sc.attention_factor : (float)(0.1 * log((double)sc.factor) + 1.0);
    return Q3_OK;
}

}  // extern "C"
