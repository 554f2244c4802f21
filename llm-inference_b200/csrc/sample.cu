// The next token of each row from given random numbers: temperature, top-k, top-p, min-p and draft tokens
// (q3_sample_logits).
//
// A row's tokens are ordered by logit, largest first, ties by index; token i weighs w_i = 2^((x_i - max) log2 e / T). What
// top-k, top-p and min-p keep are beginnings of that order, so the kept tokens are known by their mass M, the smallest of
// the three, and the token drawn is the one where the running mass passes u M. Top-k's end is the token where the running
// count passes k - 1, top-p's the one where the mass passes p times that: all three are the same search for a crossing.
// A draft token takes the first place of the order for the draw: it comes out with its own probability, the
// others with theirs.
//
// Weights are whole numbers, round(2^41 w), from exponentials in fp64: their sums are the same in any order, so neither the
// atomics below nor the way the row is cut change a result, and a draw is decided as in 64 bits.
//
// A cluster of CTAs shares a row. Two ways to find a crossing:
//   - bf16 logits have few values: one pass counts each value between 2^-32 and 2^8 of either sign, and zeros (one shared-memory
//     atomic a token, the exponentials once per value that occurs). Equal tokens weigh the same, so a running sum over
//     the values says which value and which of its tokens; one more pass, by the CTA that has it, finds its index.
//   - fp32 logits, and bf16 rows in which a value outside those weighs anything: a pass for the largest, one for a
//     histogram of mass (and for top-k of count) over the logits, and per crossing one that gathers the tokens of its bin, which are
//     ranked by comparing each with each. A bin of too many tokens is cut finer by the bits of its logits; as many equal ones are
//     told apart by counting them in the order of their index.
// CTAs write what others need into their shared memory before a cluster barrier: loads after it that wait for one another
// cost more than all the arithmetic. The counts of values are added up by all CTAs, each for a share of the groups of values
// that any has tokens of, and the sums go to the first CTA, which then needs no more barriers.
//
// Bound by the chain of these steps for few rows (one of 151936 bf16 12.5 us, 32 with all settings 17.6), for many half by
// shared-memory atomics and half by phases in which most warps wait (256 rows 45 us, 1.7 TB/s), and by instructions for fp32 rows
// (100 of 32003 35 us, the pass for the histogram half of it).
#include <math.h>

#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace q3 {
int check_device();

namespace {

constexpr int SL_THREADS = 512;
constexpr int SL_WARPS = SL_THREADS / 32;
constexpr int SL_MAX_CLUSTER = 8;
constexpr int SL_BITS = 41;        // the largest weight is 2^41: those of a whole row add up to less than 2^62
constexpr int SL_SLICE = 1 << 18;  // tokens of a CTA at most: the upper halves of their weights, up to 2^9 each, add up within 32 bits
constexpr int SL_VOCAB = 1 << 20;

typedef unsigned long long u64;

struct SampleArgs {
    int *out;
    float *prob;
    const void *logits;
    long long stride;
    int vocab, slice;  // slice: tokens of a CTA, a multiple of 8
    const float *u, *temperature, *top_p, *min_p;
    const int *top_k, *draft;
};

// What a CTA tells the others.
struct Told {
    u64 above, before_draft;  // its mass above min-p's limit and before the draft
    unsigned first;           // key of its largest logit, 0: none
    unsigned count, low, high;
};

// Where a running sum passes a target: the token's weight, what comes before it, and which token it is.
struct Crossing {
    u64 before, w;
    int index;     // of the token
    int pos;       // or its value's place, and which token of that value it is
    unsigned nth;
};

__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// Unsigned numbers in the order of the floats; both zeros are one.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Weights of a row's logits.
struct Weigher {
    float peak;
    double c;  // log2 e / T
    // round(2^SL_BITS * 2^((x - peak) c)): the power's whole part goes to the exponent, the rest f in [-1/2, 1/2] through the
    // Chebyshev series of 2^f there, cut after the tenth term: off by 3.2e-16, a thousandth of a unit (the Taylor polynomial of as many
    // terms by 3e-13, and weights by nearly a whole unit). No branches, so that a thread's weights overlap: one chain of these
    // operations is 200 cycles.
    __device__ __forceinline__ u64 operator()(float x) const {
        const double t = ((double)x - (double)peak) * c;
        const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number, kept in the low bits
        const double shifted = t + magic;
        const int n = __double2loint(shifted);
        const double f = t - (shifted - magic);
        double y = 7.074194562613105e-09;  // the series as a polynomial in f, the tenth power first
        y = fma(y, f, 1.020869083593037e-07);
        y = fma(y, f, 1.3215432534254118e-06);
        y = fma(y, f, 1.5252657257186041e-05);
        y = fma(y, f, 0.00015403530463727982);
        y = fma(y, f, 0.0013333558230170627);
        y = fma(y, f, 0.009618129107587253);
        y = fma(y, f, 0.05550410866444768);
        y = fma(y, f, 0.24022650695910158);
        y = fma(y, f, 0.69314718055995);
        y = fma(y, f, 1.0);
        y = __hiloint2double(__double2hiint(y) + ((n + SL_BITS) << 20), __double2loint(y));
        const u64 w = (u64)__double_as_longlong(y + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: the sum's fraction bits
        return x == peak ? 1ull << SL_BITS : t > -44.0 ? w : 0;
    }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct ScanShared {
    u64 mass[SL_WARPS];
    unsigned count[SL_WARPS];
};

// Exclusive running sums over the CTA's threads in place of m and n; the CTA's sums go to mass and count.
__device__ void block_scan(ScanShared &s, u64 &m, unsigned &n, u64 &mass, unsigned &count) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    auto scan = [&](u64 &rm, unsigned &rn) {  // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 ym = __shfl_up_sync(0xffffffffu, rm, o);
            const unsigned yn = __shfl_up_sync(0xffffffffu, rn, o);
            rm += lane >= o ? ym : 0;
            rn += lane >= o ? yn : 0;
        }
    };
    u64 rm = m;
    unsigned rn = n;
    scan(rm, rn);
    __syncthreads();  // earlier readers of s
    if (lane == 31) {
        s.mass[warp] = rm;
        s.count[warp] = rn;
    }
    __syncthreads();
    u64 wm = lane < SL_WARPS ? s.mass[lane] : 0;
    unsigned wn = lane < SL_WARPS ? s.count[lane] : 0;
    scan(wm, wn);
    mass = __shfl_sync(0xffffffffu, wm, SL_WARPS - 1);
    count = __shfl_sync(0xffffffffu, wn, SL_WARPS - 1);
    wm = __shfl_sync(0xffffffffu, wm, max(warp - 1, 0));
    wn = __shfl_sync(0xffffffffu, wn, max(warp - 1, 0));
    m = rm - m + (warp ? wm : 0);
    n = rn - n + (warp ? wn : 0);
}

// The last of N entries whose running sum (what comes before it) is not above the target, by all lanes of a warp. Entries of
// no weight begin where the next one does, so the target lies in the entry that is found.
template <int N>
__device__ __forceinline__ int search(const u64 *mass, const unsigned *count, u64 target, bool by_count) {
    constexpr int EACH = N / 32;
    const int lane = threadIdx.x % 32;
    auto before = [&](int e) { return by_count ? (u64)count[e] : mass[e]; };
    int e = EACH * (31 - __clz(__ballot_sync(0xffffffffu, before(lane * EACH) <= target)));
    e += 31 - __clz(__ballot_sync(0xffffffffu, lane < EACH && before(e + lane % EACH) <= target));
    return e;
}

// A row as the CTAs of a cluster see it.
template <typename T>
struct Row {
    static constexpr int PER = 16 / sizeof(T);
    cg::cluster_group cluster;
    int C, rank;
    const T *in;
    int vocab, i0, slice;  // i0: index of the slice's first place, where a 16-byte line begins; it may lie before the row

    __device__ __forceinline__ void sync() {
        arrive();
        wait();
    }
    // the two halves of a barrier
    __device__ __forceinline__ void arrive() {
        if (C > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    }
    __device__ __forceinline__ void wait() {
        if (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        else __syncthreads();
    }
    template <typename V>
    __device__ __forceinline__ V *of(V *p, int r) { return C > 1 ? cluster.map_shared_rank(p, r) : p; }

    // A line of the row; places outside it hold -infinity.
    __device__ __forceinline__ uint4 line(int i) const {
        if (i >= 0 && i + PER <= vocab) return __ldg(reinterpret_cast<const uint4 *>(in + i));
        return edge(in, vocab, i);
    }
    static __device__ __noinline__ uint4 edge(const T *in, int vocab, int i) {
        alignas(16) T x[PER];
#pragma unroll 1
        for (int e = 0; e < PER; e++) x[e] = i + e >= 0 && i + e < vocab ? in[i + e] : T(-INFINITY);
        return *reinterpret_cast<const uint4 *>(x);
    }
    // f(line, index of its first place) over the slice, with LOADS loads in flight and f's code only once: most of these
    // kernels' code runs once or a few times, and waiting for it is what costs
    template <int LOADS, typename F>
    __device__ __forceinline__ void each_line(F f) const {
        constexpr int STEP = SL_THREADS * PER;
        uint4 next[LOADS];
        int v = threadIdx.x * PER;
#pragma unroll
        for (int l = 0; l < LOADS; l++)
            if (v + l * STEP < slice) next[l] = line(i0 + v + l * STEP);
#pragma unroll 1
        for (; v < slice; v += STEP) {
            const uint4 raw = next[0];
#pragma unroll
            for (int l = 1; l < LOADS; l++) next[l - 1] = next[l];
            if (v + LOADS * STEP < slice) next[LOADS - 1] = line(i0 + v + LOADS * STEP);
            f(raw, i0 + v);
        }
    }
    // f(x, index)
    template <int LOADS, typename F>
    __device__ __forceinline__ void each(F f) const {
        each_line<LOADS>([&](const uint4 &raw, int i) {
            const T *x = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int e = 0; e < PER; e++) f(to_f32(x[e]), i + e);
        });
    }
};

// ------------------------------------------------------------------ any logits: histogram and gathered bins

constexpr int SL_BINS = 1024;
constexpr int SL_CAND = 256;  // tokens of a bin that are ranked directly

struct alignas(16) Candidate {
    u64 order;  // key in the upper half, complement of the index below: larger comes earlier
    u64 w;
};

struct BinsShared {
    alignas(16) unsigned part[3][SL_BINS];  // this CTA's histogram: lower and upper halves of the masses, and counts
    u64 sum_mass[2][SL_BINS];   // what comes before each bin in the row; [1]: of a bin that was cut finer
    unsigned sum_count[2][SL_BINS];
    Candidate list[2][SL_CAND];  // this CTA's tokens of the bin in question; finds take turns
    Candidate all[SL_CAND];      // and the cluster's
    unsigned n_list, key_lo, key_hi;
    Told told[4][SL_MAX_CLUSTER];  // the first pass's, the second's, and the lists' (by turns)
    int bin, tie;
    Crossing found;
    ScanShared scan;
};

template <typename T>
struct Bins {
    BinsShared &s;
    Row<T> &row;
    Weigher weigh;
    float per_bin;
    unsigned least_key;  // no logit below it weighs anything
    bool counting;       // tokens, too
    int turn = 0;

    // by adding 2^23, which leaves the nearest whole number in the low bits
    __device__ __forceinline__ float place_of(float x) const { return fminf((weigh.peak - x) * per_bin, SL_BINS - 1.0f) + 8388608.0f; }
    __device__ __forceinline__ int bin_of(float x) const { return __float_as_int(place_of(x)) & (SL_BINS - 1); }
    static __device__ __forceinline__ float bin_place(int bin) { return 8388608.0f + bin; }

    __device__ __forceinline__ void zero() {
        for (int b = threadIdx.x; b < SL_BINS; b += SL_THREADS) s.part[0][b] = s.part[1][b] = s.part[2][b] = 0;
    }
    // N tokens. 64-bit atomics in shared memory are loops, so the lower halves' own overflow says what to carry to the upper ones;
    // most weights have no upper half, and only top-k asks for counts.
    template <int N>
    __device__ __forceinline__ void add(const int (&b)[N], const u64 (&w)[N]) {
        unsigned up[N];
#pragma unroll
        for (int e = 0; e < N; e++) {
            const unsigned low = (unsigned)w[e];
            up[e] = (unsigned)(w[e] >> 32);
            if (low) up[e] += atomicAdd(&s.part[0][b[e]], low) + low < low;
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            if (up[e]) atomicAdd(&s.part[1][b[e]], up[e]);
            if (counting && w[e]) atomicAdd(&s.part[2][b[e]], 1u);
        }
    }

    // Running sums of the CTAs' histograms into sum_*[level]; each CTA adds up a share of the bins for all.
    __device__ void merge(int level, u64 base_mass, unsigned base_count, u64 &mass, unsigned &count) {
        row.sync();
        // four bins a thread: remote shared memory gives and takes 16 bytes as fast as 4
        const int share = (SL_BINS / 4 + row.C - 1) / row.C, b = 4 * (row.rank * share + threadIdx.x);
        if (threadIdx.x < share && b < SL_BINS) {
            u64 m[4] = {};
            uint4 n = {};
#pragma unroll 1
            for (int r = 0; r < row.C; r++) {
                uint4 p[3];
#pragma unroll
                for (int k = 0; k < 3; k++) p[k] = *reinterpret_cast<const uint4 *>(row.of(s.part[k], r) + b);
                m[0] += p[0].x + ((u64)p[1].x << 32);
                m[1] += p[0].y + ((u64)p[1].y << 32);
                m[2] += p[0].z + ((u64)p[1].z << 32);
                m[3] += p[0].w + ((u64)p[1].w << 32);
                n.x += p[2].x;
                n.y += p[2].y;
                n.z += p[2].z;
                n.w += p[2].w;
            }
#pragma unroll 1
            for (int r = 0; r < row.C; r++) {
                ulonglong2 *to = reinterpret_cast<ulonglong2 *>(row.of(s.sum_mass[level], r) + b);
                to[0] = make_ulonglong2(m[0], m[1]);
                to[1] = make_ulonglong2(m[2], m[3]);
                *reinterpret_cast<uint4 *>(row.of(s.sum_count[level], r) + b) = n;
            }
        }
        row.sync();
        static_assert(SL_BINS == 2 * SL_THREADS, "two bins a thread");
        const int at = 2 * threadIdx.x;
        const u64 m0 = s.sum_mass[level][at];
        const unsigned n0 = s.sum_count[level][at];
        u64 sm = m0 + s.sum_mass[level][at + 1];
        unsigned sn = n0 + s.sum_count[level][at + 1];
        block_scan(s.scan, sm, sn, mass, count);
        s.sum_mass[level][at] = base_mass + sm;
        s.sum_mass[level][at + 1] = base_mass + sm + m0;
        s.sum_count[level][at] = base_count + sn;
        s.sum_count[level][at + 1] = base_count + sn + n0;
        __syncthreads();
    }

    // The token where the running mass (or count) of the row passes `target`, which lies in the row.
    __device__ Crossing find(u64 target, bool by_count) {
        unsigned lo = 0, hi = 0;  // keys of the tokens in question, once the first bin is cut
        bool cut = false;
        int bin = search<SL_BINS>(s.sum_mass[0], s.sum_count[0], target, by_count);
        u64 mass = s.sum_mass[0][bin];
        unsigned count = s.sum_count[0][bin];
        while (true) {
            // this CTA's tokens of the bin
            const int at_turn = turn;
            turn ^= 1;
            Candidate *list = s.list[at_turn];
            if (threadIdx.x == 0) {
                s.n_list = 0;
                s.key_lo = 0xffffffffu;
                s.key_hi = 0;
            }
            __syncthreads();
            const float least = of_key(cut ? lo : least_key), most = cut ? of_key(hi) : INFINITY, its = bin_place(bin);
            row.template each<2>([&](float x, int i) {
                if (!(x >= least && x <= most && (cut || place_of(x) == its))) return;
                const unsigned key = key_of(x);
                const unsigned at = atomicAdd(&s.n_list, 1u);
                if (at < SL_CAND) list[at].order = (u64)key << 32 | (unsigned)~i;
                atomicMin(&s.key_lo, key);
                atomicMax(&s.key_hi, key);
            });
            __syncthreads();
            if (threadIdx.x < SL_CAND && threadIdx.x < s.n_list) list[threadIdx.x].w = weigh(of_key((unsigned)(list[threadIdx.x].order >> 32)));
            if (threadIdx.x < row.C) {
                Told *t = row.of(&s.told[2 + at_turn][row.rank], threadIdx.x);
                t->count = s.n_list;
                t->low = s.key_lo;
                t->high = s.key_hi;
            }
            row.sync();
            const Told *told = s.told[2 + at_turn];
            unsigned n = 0;
            lo = 0xffffffffu;
            hi = 0;
            for (int r = 0; r < row.C; r++) {
                n += told[r].count;
                lo = min(lo, told[r].low);
                hi = max(hi, told[r].high);
            }
            if (n <= SL_CAND) return rank_all(at_turn, n, target, by_count, mass, count);
            if (lo == hi) return nth_tie(told, lo, target, by_count, mass, count);
            // cut the bin by the bits of its keys
            cut = true;
            const int shift = 32 - __clz((hi - lo) / SL_BINS);
            zero();
            __syncthreads();
            row.template each<1>([&](float x, int) {
                const unsigned key = key_of(x);
                if (x == x && key >= lo && key <= hi) add<1>({(int)((hi - key) >> shift)}, {weigh(x)});
            });
            u64 all_mass;
            unsigned all_count;
            merge(1, mass, count, all_mass, all_count);
            bin = search<SL_BINS>(s.sum_mass[1], s.sum_count[1], target, by_count);
            mass = s.sum_mass[1][bin];
            count = s.sum_count[1][bin];
            const unsigned span = (1u << shift) - 1;
            hi -= (unsigned)bin << shift;
            lo = hi - lo > span ? hi - span : lo;
            if (hi == key_of(0.0f) - 1) hi--;  // the key of -0, which no logit has: compared as a float it would take the zeros in
        }
    }

    // Among the n tokens that the CTAs listed.
    __device__ Crossing rank_all(int at_turn, unsigned n, u64 target, bool by_count, u64 mass, unsigned count) {
        unsigned at = 0;
        for (int r = 0; r < row.C; r++) {
            const unsigned k = s.told[2 + at_turn][r].count;
            const Candidate *from = row.of(s.list[at_turn], r);
            for (unsigned j = threadIdx.x; j < k; j += SL_THREADS) s.all[at + j] = from[j];
            at += k;
        }
        __syncthreads();
        // `sub` neighbouring threads compare one token with all
        int sub = 32;
        while ((unsigned)(SL_THREADS / sub) < n) sub /= 2;
        const unsigned mine = threadIdx.x / sub, from = threadIdx.x % sub;
        const Candidate own = mine < n ? s.all[mine] : Candidate{~0ull, 0};
        u64 before = 0;
        unsigned places = 0;
#pragma unroll 4
        for (unsigned j = from; j < n; j += sub) {
            const Candidate c = s.all[j];
            const bool ahead = c.order > own.order;
            before += ahead ? c.w : 0;
            places += ahead;
        }
        for (int o = sub / 2; o > 0; o /= 2) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            places += __shfl_xor_sync(0xffffffffu, places, o);
        }
        before += mass;
        places += count;
        if (mine < n && from == 0 && (by_count ? places == target : before <= target && target < before + own.w))
            s.found = {before, own.w, (int)~(unsigned)own.order, 0, 0};
        __syncthreads();
        const Crossing f = s.found;
        __syncthreads();  // all, found: read
        return f;
    }

    // Among tokens of one logit, more than are ranked directly: by their index.
    __device__ Crossing nth_tie(const Told *told, unsigned key, u64 target, bool by_count, u64 mass, unsigned count) {
        const u64 w = weigh(of_key(key));
        const u64 nth = by_count ? target - count : (target - mass) / w;
        u64 left = nth;
        int owner = 0;
        for (; owner < row.C - 1; owner++) {
            if (left < told[owner].count) break;
            left -= told[owner].count;
        }
        if (row.rank == owner) {
            for (int v0 = 0; v0 < row.slice; v0 += SL_THREADS) {
                const int i = row.i0 + v0 + threadIdx.x;
                const bool is = v0 + (int)threadIdx.x < row.slice && i >= 0 && i < row.vocab && key_of(to_f32(row.in[i])) == key;
                u64 none = 0, sum;
                unsigned before = is, here;
                block_scan(s.scan, none, before, sum, here);
                if (is && before == left)
                    for (int r = 0; r < row.C; r++) *row.of(&s.tie, r) = i;
                if (left < here) break;
                left -= here;
            }
        }
        row.sync();
        return {mass + nth * w, w, s.tie, 0, 0};
    }

    __device__ __forceinline__ int index(const Crossing &f) { return f.index; }
};

// ------------------------------------------------------------------ bf16 logits: counts of their values

// Magnitudes that are counted, from 2^-32 to below 2^8. From 2^-24 on, one row in 300 of 151936 normal logits had one below
// and went the other way, which its whole batch waited for.
constexpr int SL_LOW = (127 - 32) << 7, SL_HIGH = (127 + 8) << 7;
constexpr float SL_TINY = 0x1p-32f;
constexpr int SL_SIGN = SL_HIGH - SL_LOW;
// Places in the order of the values: positive ones, zero, which has a group of its own, negative ones; in groups of neighbouring
// ones, which a warp takes side by side. Counters lie in another order, that of the values' bits: positive ones, negative ones, zero,
// so that a token's counter takes few instructions to find.
constexpr int SL_GROUP = 32;
constexpr int SL_PLACES = 2 * SL_SIGN + SL_GROUP;
constexpr int SL_USED = SL_PLACES / SL_GROUP;
constexpr int SL_GROUPS = SL_THREADS;  // searched before the values themselves; the last ones are empty
static_assert(SL_SIGN % SL_GROUP == 0 && SL_USED <= SL_GROUPS, "whole groups");

struct ValuesShared {
    alignas(16) unsigned count[SL_PLACES];  // this CTA's
    Told told[SL_MAX_CLUSTER];
    unsigned occupied[SL_MAX_CLUSTER][SL_WARPS];  // which groups each CTA has tokens of
    unsigned short list[SL_GROUPS];               // its share of those that any has
    unsigned tiny, equal;  // a low magnitude but zero; the draft's equals before it in its CTA
    unsigned outer;               // key of the largest of high magnitude, 0: none
    unsigned top;
    // in the cluster's first CTA:
    u64 group_mass[SL_GROUPS];  // then what comes before each group
    unsigned group_count[SL_GROUPS];
    unsigned equals[SL_MAX_CLUSTER];
    Crossing at;
    float prob;
    bool is_draft;
    ScanShared scan;
    unsigned warps[2][2 * SL_WARPS];
};

__device__ __forceinline__ bf16 value_of(int pos) {
    const int m = pos < SL_SIGN ? SL_HIGH - 1 - pos : pos < SL_SIGN + SL_GROUP ? 0 : SL_LOW + (pos - SL_SIGN - SL_GROUP) + 0x8000;
    return __ushort_as_bfloat16((unsigned short)m);
}
// The value's place, -1 if it is not counted.
__device__ __forceinline__ int pos_of(unsigned h) {
    const int m = h & 0x7fff;
    if (m == 0) return SL_SIGN;
    if (m < SL_LOW || m >= SL_HIGH) return -1;
    return h & 0x8000 ? SL_SIGN + SL_GROUP + (m - SL_LOW) : SL_HIGH - 1 - m;
}
// The counter of a place, and the first of a group.
__device__ __forceinline__ int counter_of(int pos) { return pos < SL_SIGN ? SL_SIGN - 1 - pos : pos < SL_SIGN + SL_GROUP ? pos + SL_SIGN : pos - SL_GROUP; }
__device__ __forceinline__ int counters_of(int g) {
    return SL_GROUP * (g < SL_SIGN / SL_GROUP ? SL_SIGN / SL_GROUP - 1 - g : g == SL_SIGN / SL_GROUP ? 2 * SL_SIGN / SL_GROUP : g - 1);
}
// f(value) is true for the first values, down to some place: the number of them, by all lanes of a warp.
template <typename F>
__device__ __forceinline__ int first_values(F f) {
    int lo = 0, hi = SL_PLACES;  // true before lo, false from hi on
    const int lane = threadIdx.x % 32;
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && f(to_f32(value_of(at)))));
        if (n == 0) return lo;
        hi = min(hi, lo + n * step);
        lo += (n - 1) * step + 1;
    }
    return lo;
}

struct Values {
    ValuesShared &s;
    Row<bf16> &row;
    unsigned *sum;  // the cluster's counts, in a CTA for its share of the groups, in the first one all that are not empty
    Weigher weigh;

    // Bits of a line's places that hold the value; both zeros are one.
    static __device__ __forceinline__ unsigned equals(const uint4 &raw, bf16 value) {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&raw), v = __halves2bfloat162(value, value);
        unsigned n = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) n |= (__heq2_mask(h[e], v) & 0x20001u) << 2 * e;
        return (n | n >> 16) & 0xffu;
    }

    __device__ __forceinline__ void zero() {
        for (int v = 4 * threadIdx.x; v < SL_PLACES; v += 4 * SL_THREADS) *reinterpret_cast<uint4 *>(s.count + v) = make_uint4(0, 0, 0, 0);
        if (threadIdx.x == 0) s.tiny = s.outer = s.equal = s.top = 0;
    }

    // A value that is not counted one by one, and not -infinity.
    __device__ __noinline__ static void odd(ValuesShared &s, unsigned v) {
        const unsigned m = v & 0x7fff;
        if (m == 0) atomicAdd(&s.count[2 * SL_SIGN], 1u);
        else if (m < SL_LOW) s.tiny = 1;
        else if (m <= 0x7f80) atomicMax(&s.outer, key_of(__uint_as_float(v << 16)));  // else NaN
    }

    // One pass over the slice: counts, and the largest value.
    __device__ void stream() {
        __nv_bfloat162 top = __floats2bfloat162_rn(-INFINITY, -INFINITY);
        const __nv_bfloat162 least = __floats2bfloat162_rn(SL_TINY, SL_TINY), most = __floats2bfloat162_rn(256.0f, 256.0f);
        row.each_line<4>([&](const uint4 &raw, int) {
            const unsigned *h = reinterpret_cast<const unsigned *>(&raw);
            unsigned m2[4];
            bool all = true;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                top = __hmax2(top, *reinterpret_cast<const __nv_bfloat162 *>(&h[e]));  // not NaN, if either is not
                m2[e] = h[e] & 0x7fff7fffu;
                const __nv_bfloat162 mag = *reinterpret_cast<const __nv_bfloat162 *>(&m2[e]);
                all = all && __hbge2(mag, least) && __hblt2(mag, most);
            }
            if (all) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    atomicAdd(&s.count[(m2[e] & 0xffffu) + ((unsigned)((int)(h[e] << 16) >> 31) & SL_SIGN) - SL_LOW], 1u);
                    atomicAdd(&s.count[(m2[e] >> 16) + ((unsigned)((int)h[e] >> 31) & SL_SIGN) - SL_LOW], 1u);
                }
                return;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const unsigned v = e % 2 ? h[e / 2] >> 16 : h[e / 2] & 0xffff, off = (v & 0x7fff) - SL_LOW;
                if (off < (unsigned)SL_SIGN) atomicAdd(&s.count[off + (v & 0x8000 ? SL_SIGN : 0)], 1u);
                else if (v != 0xff80) odd(s, v);
            }
        });
        float t = fmaxf(__low2float(top), __high2float(top));
        t = t == t ? t : -INFINITY;
        const unsigned best = __reduce_max_sync(0xffffffffu, t > -INFINITY ? key_of(t) : 0);
        if (threadIdx.x % 32 == 0) atomicMax(&s.top, best);
        __syncthreads();
        unsigned any = 0;
        if (threadIdx.x < SL_USED) {
#pragma unroll
            for (int k = 0; k < SL_GROUP / 4; k++) {  // each lane from another bank on
                const uint4 n = *reinterpret_cast<const uint4 *>(s.count + counters_of(threadIdx.x) + 4 * ((k + threadIdx.x) % (SL_GROUP / 4)));
                any |= n.x | n.y | n.z | n.w;
            }
        }
        any = __ballot_sync(0xffffffffu, any != 0);
        if ((int)threadIdx.x % 32 < row.C) *row.of(&s.occupied[row.rank][threadIdx.x / 32], threadIdx.x % 32) = any;
    }

    // The CTAs' counts to the first one, each CTA the sums of its share of the groups. draft: index, or -1.
    __device__ void merge(int draft, float xd) {
        // Two thirds of the groups are empty in a row of normal logits; the others are dealt out to the CTAs in turn.
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
        unsigned some = 0;  // lane j: the 32 groups of warp j that any CTA has tokens of
        if (lane < SL_WARPS)
            for (int r = 0; r < row.C; r++) some |= s.occupied[r][lane];
        unsigned run = __popc(some);
#pragma unroll
        for (int o = 1; o < SL_WARPS; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, run, o);
            run += lane >= o ? y : 0;
        }
        const unsigned own = __shfl_sync(0xffffffffu, some, warp), all = __shfl_sync(0xffffffffu, run, SL_WARPS - 1);
        const unsigned before = __shfl_sync(0xffffffffu, run - __popc(some), warp) + __popc(own & ((1u << lane) - 1));
        if (own >> lane & 1) {
            if ((int)(before % row.C) == row.rank) s.list[before / row.C] = (unsigned short)threadIdx.x;
        } else if (row.rank == 0) {
            s.group_mass[threadIdx.x] = s.group_count[threadIdx.x] = 0;
        }
        const int n_list = ((int)all + row.C - 1 - row.rank) / row.C;
        __syncthreads();
        if (row.C > 1) {  // remote shared memory gives and takes 16 bytes as fast as 4
#pragma unroll 1
            for (int i = threadIdx.x; i < n_list * (SL_GROUP / 4); i += SL_THREADS) {
                const int v = counters_of(s.list[i / (SL_GROUP / 4)]) + i % (SL_GROUP / 4) * 4;
                uint4 n = *reinterpret_cast<const uint4 *>(s.count + v);
#pragma unroll 1
                for (int r0 = 1; r0 < row.C; r0 += 4) {
                    uint4 of[4];  // all loads before the first sum
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int rank = row.rank + r0 + r;
                        of[r] = r0 + r < row.C ? *reinterpret_cast<const uint4 *>(row.of(s.count, rank < row.C ? rank : rank - row.C) + v)
                                               : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        n.x += of[r].x;
                        n.y += of[r].y;
                        n.z += of[r].z;
                        n.w += of[r].w;
                    }
                }
                *reinterpret_cast<uint4 *>(sum + v) = n;
                if (row.rank != 0) *reinterpret_cast<uint4 *>(row.of(sum, 0) + v) = n;
            }
            __syncthreads();
        }
        const int sub = n_list <= SL_THREADS / 8 ? 8 : n_list <= SL_THREADS / 4 ? 4 : n_list <= SL_THREADS / 2 ? 2 : 1;
        const bool mine = (int)threadIdx.x / sub < n_list;  // `sub` neighbouring threads share a group
        const int g = mine ? s.list[threadIdx.x / sub] : 0;
        u64 mass = 0;
        unsigned count = 0;
        // a warp's lanes stay together
#pragma unroll 1
        for (int e = 0; e < SL_GROUP; e += sub) {
            const int pos = g * SL_GROUP + (e + threadIdx.x) % SL_GROUP;  // from another bank in each group
            const unsigned n = mine ? sum[counter_of(pos)] : 0;
            if (__any_sync(0xffffffffu, n != 0)) {
                const u64 w = weigh(to_f32(value_of(n ? pos : 0)));
                mass += n * w;
                count += w ? n : 0;
            }
        }
        for (int o = sub / 2; o > 0; o /= 2) {
            mass += __shfl_xor_sync(0xffffffffu, mass, o);
            count += __shfl_xor_sync(0xffffffffu, count, o);
        }
        if (mine && threadIdx.x % sub == 0) {
            *row.of(&s.group_mass[g], 0) = mass;
            *row.of(&s.group_count[g], 0) = count;
        }
        if (draft >= 0) {  // the draft's equals with a smaller index
            const bf16 value = __float2bfloat16(xd);
            const int pos = pos_of(__bfloat16_as_ushort(value));
            const unsigned here = pos < 0 ? 0 : s.count[counter_of(pos)];
            if (here > 0 && row.i0 + row.slice <= draft) {
                if (threadIdx.x == 0) s.equal = here;
            } else if (here > 1 && row.i0 < draft) {
                unsigned n = 0;
                row.each_line<2>([&](const uint4 &raw, int i) {
                    const unsigned is = equals(raw, value);
                    n += __popc(i + Row<bf16>::PER <= draft ? is : i < draft ? is & ((1u << (draft - i)) - 1) : 0);
                });
                n = __reduce_add_sync(0xffffffffu, n);
                if (threadIdx.x % 32 == 0) atomicAdd(&s.equal, n);
            }
            __syncthreads();
            if (threadIdx.x == 0) *row.of(&s.equals[row.rank], 0) = s.equal;
        }
        row.sync();
    }

    // What follows is the first CTA's. Running sums of the groups, and the row's.
    __device__ void scan(u64 &mass, unsigned &count) {
        const int g = threadIdx.x;
        u64 m = s.group_mass[g];
        unsigned n = s.group_count[g];
        block_scan(s.scan, m, n, mass, count);
        s.group_mass[g] = m;
        s.group_count[g] = n;
        __syncthreads();
    }

    // The token where the running mass (or count) of the row passes `target`, which lies in the row: which one of which value.
    // By all lanes of a warp.
    __device__ Crossing find(u64 target, bool by_count) {
        __syncwarp();
        const int lane = threadIdx.x % 32;
        const int g = search<SL_GROUPS>(s.group_mass, s.group_count, target, by_count);
        const int pos = g * SL_GROUP + lane;
        const u64 w = weigh(to_f32(value_of(pos)));
        const unsigned n = w ? sum[counter_of(pos)] : 0;
        const u64 m = n * w;
        u64 bm = m;
        unsigned bn = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 ym = __shfl_up_sync(0xffffffffu, bm, o);
            const unsigned yn = __shfl_up_sync(0xffffffffu, bn, o);
            if (lane >= o) {
                bm += ym;
                bn += yn;
            }
        }
        bm += s.group_mass[g] - m;
        bn += s.group_count[g] - n;
        const int src = 31 - __clz(__ballot_sync(0xffffffffu, n > 0 && (by_count ? bn <= target : bm <= target)));
        bm = __shfl_sync(0xffffffffu, bm, src);
        bn = __shfl_sync(0xffffffffu, bn, src);
        const u64 ws = __shfl_sync(0xffffffffu, w, src);
        const unsigned nth = by_count ? (unsigned)target - bn : (unsigned)((target - bm) / ws);
        return {bm + nth * ws, ws, -1, g * SL_GROUP + src, nth};
    }
    // The mass before a value, by all lanes of a warp.
    __device__ u64 before(int pos) {
        const int g = pos / SL_GROUP, at = g * SL_GROUP + threadIdx.x % 32;
        const bool some = g + 1 < SL_GROUPS && s.group_count[g + 1] > s.group_count[g];  // of an empty group there are no sums
        return s.group_mass[g] + warp_sum(some && at < pos ? sum[counter_of(at)] * weigh(to_f32(value_of(at))) : 0);
    }

    // The index of a value's nth token.
    __device__ int index(const Crossing &f) {
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
        const unsigned here = lane < row.C ? row.of(s.count, lane)[counter_of(f.pos)] : 0;
        unsigned run = here;
#pragma unroll
        for (int o = 1; o < SL_MAX_CLUSTER; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
        }
        const int owner = __popc(__ballot_sync(0xffffffffu, lane < row.C && run <= f.nth));
        unsigned left = f.nth - __shfl_sync(0xffffffffu, run - here, owner);
        const int i0 = row.i0 + owner * row.slice;
        // 1024 lines a step, until the step that has it; the next step's lines are on their way meanwhile
        const bf16 value = value_of(f.pos);
        const int lines = row.slice / 8;
        const uint4 none = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);  // NaN equals nothing
        auto load = [&](int l) { return l < lines ? row.line(i0 + 8 * l) : none; };
        uint4 next[2] = {load(threadIdx.x), load(SL_THREADS + threadIdx.x)};
#pragma unroll 1
        for (int l0 = 0, odd = 0; l0 < lines; l0 += 2 * SL_THREADS, odd ^= 1) {
            const unsigned is[2] = {equals(next[0], value), equals(next[1], value)};
            next[0] = load(l0 + 2 * SL_THREADS + threadIdx.x);
            next[1] = load(l0 + 3 * SL_THREADS + threadIdx.x);
            // counts of the warps for the first 512 lines, then for the others: an entry a lane
            static_assert(2 * SL_WARPS == 32, "an entry a lane");
            const unsigned n0 = __reduce_add_sync(0xffffffffu, __popc(is[0])), n1 = __reduce_add_sync(0xffffffffu, __popc(is[1]));
            if (lane < 2) s.warps[odd][lane * SL_WARPS + warp] = lane ? n1 : n0;
            __syncthreads();
            const unsigned n = s.warps[odd][lane], all = __reduce_add_sync(0xffffffffu, n);
            if (left >= all) {
                left -= all;
                continue;
            }
            auto scan = [&](unsigned v) {
                unsigned r = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned y = __shfl_up_sync(0xffffffffu, r, o);
                    r += lane >= o ? y : 0;
                }
                return r - v;
            };
            const unsigned b = scan(n);
            const int e = __ffs(__ballot_sync(0xffffffffu, left >= b && left < b + n)) - 1;
            left -= __shfl_sync(0xffffffffu, b, e);
            if (e % SL_WARPS == warp) {
                unsigned mine = e < SL_WARPS ? is[0] : is[1];
                const unsigned before = scan(__popc(mine));
                if (left >= before && left < before + __popc(mine)) {
                    for (unsigned j = left - before; j > 0; j--) mine &= mine - 1;
                    s.at.index = i0 + 8 * (l0 + e / SL_WARPS * SL_THREADS + (int)threadIdx.x) + __ffs(mine) - 1;
                }
            }
            break;
        }
        __syncthreads();
        return s.at.index;
    }
};

// ------------------------------------------------------------------ a row's choices

struct Choice {
    float temperature, p, floor, u, xd;
    int k, draft;
};

// The token that a row takes once its weights can be searched; mass and count: of the whole row.
struct Draw {
    u64 w, mass;
    bool draft;  // the draft, else the crossing's token
    Crossing at;
};
template <typename Finder>
__device__ Draw draw(Finder &finder, const Choice &o, const Weigher &weigh, u64 mass, unsigned count, u64 above, u64 before_draft) {
    Draw d = {};
    const u64 wd = o.draft >= 0 ? weigh(o.xd) : 0;
    int what = o.k > 0 && (unsigned)o.k < count ? 0 : o.p < 1.0f ? 1 : 2;  // top-k's end, top-p's, the token
    while (true) {
        u64 target = o.k - 1;
        if (what == 1) {  // the shortest beginning with at least p of the mass
            const double want = ceil((double)fmaxf(o.p, 0.0f) * (double)mass);
            target = want < 1.0 ? 0 : min((u64)want, mass) - 1;
        } else if (what == 2) {
            if (o.floor > 0.0f) mass = min(mass, above);
            d.mass = mass;
            target = min((u64)((double)o.u * (double)mass), mass - 1);
            if (wd > 0 && before_draft < mass) {
                d.w = wd;
                d.draft = target < wd;
                if (d.draft) return d;
                if (target - wd < before_draft) target -= wd;  // the draft's place in the order is empty
            }
        }
        d.at = finder.find(target, what == 0);
        if (what == 2) break;
        mass = d.at.before + d.at.w;
        what = what == 0 && o.p < 1.0f ? 1 : 2;
    }
    d.w = d.at.w;
    return d;
}

__device__ __forceinline__ Weigher weigher(float peak, float temperature) {
    // an infinite temperature makes all finite logits weigh the same, -infinity still nothing
    return {peak, fmax(1.4426950408889634 / (double)temperature, 1e-300)};
}

template <typename T>
__device__ void sample_bins(BinsShared &s, Row<T> &row, const SampleArgs &a, const Choice &o, int r) {
    const int tid = threadIdx.x;
    // the largest logit, and the smallest finite one
    float top = -INFINITY, low = INFINITY;
    row.template each_line<4>([&](const uint4 &raw, int) {
        const T *x = reinterpret_cast<const T *>(&raw);
        float most = to_f32(x[0]), least = most;
#pragma unroll
        for (int e = 1; e < Row<T>::PER; e++) {  // not NaN, if any is not
            most = fmaxf(most, to_f32(x[e]));
            least = fminf(least, to_f32(x[e]));
        }
        top = fmaxf(top, most);
        if (!(least > -INFINITY)) {
            least = INFINITY;
#pragma unroll
            for (int e = 0; e < Row<T>::PER; e++) least = to_f32(x[e]) > -INFINITY ? fminf(least, to_f32(x[e])) : least;
        }
        low = fminf(low, least);
    });
    const unsigned best = __reduce_max_sync(0xffffffffu, top > -INFINITY ? key_of(top) : 0);
    const unsigned least = __reduce_min_sync(0xffffffffu, key_of(low));
    if (tid % 32 == 0) s.all[tid / 32] = {best, least};
    Bins<T> bins = {s, row, {}, 0.0f, 0, o.k > 0};
    bins.zero();
    if (tid == 0) s.tie = 0x7fffffff;
    __syncthreads();
    if (tid < row.C) {
        unsigned f = 0, l = 0xffffffffu;
        for (int w = 0; w < SL_WARPS; w++) {
            f = max(f, (unsigned)s.all[w].order);
            l = min(l, (unsigned)s.all[w].w);
        }
        Told *t = row.of(&s.told[0][row.rank], tid);
        t->first = f;
        t->low = l;
    }
    row.sync();
    unsigned first = 0, min_key = 0xffffffffu;  // first: the largest one's key, 0: none
    for (int c = 0; c < row.C; c++) {
        first = max(first, s.told[0][c].first);
        min_key = min(min_key, s.told[0][c].low);
    }
    int token = -1;
    float prob = first ? 1.0f : 0.0f;
    if (first && !(o.temperature > 0.0f)) {  // the first of the largest ones
        const float peak = of_key(first);
        row.template each<1>([&](float x, int i) {
            if (x == peak) atomicMin(&s.tie, i);
        });
        __syncthreads();
        if (tid < row.C) row.of(&s.told[1][row.rank], tid)->count = s.tie;
        row.sync();
        unsigned at = 0x7fffffff;
        for (int c = 0; c < row.C; c++) at = min(at, s.told[1][c].count);
        token = (int)at;
    }
    if (first && o.temperature > 0.0f) {
        const Weigher weigh = weigher(of_key(first), o.temperature);
        bins.weigh = weigh;
        const float range = fminf((float)(44.0 / weigh.c), weigh.peak - of_key(min_key));
        bins.per_bin = range > 0.0f ? fminf(SL_BINS / range, 1e30f) : 0.0f;
        // nothing below t = -44 weighs anything, and -infinity does not
        bins.least_key = max(key_of(-3.4028234663852886e38f), key_of(__double2float_rd((double)weigh.peak - 44.0 / weigh.c)));
        const double least_t = o.floor > 0.0f ? log2((double)fminf(o.floor, 1.0f)) : 0.0;
        // the histogram, the mass above min-p's limit, the mass before the draft
        u64 above = 0, before = 0;
        const bool extra = o.floor > 0.0f || o.draft >= 0;
        row.template each_line<2>([&](const uint4 &raw, int i0) {
            const T *in = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int e0 = 0; e0 < Row<T>::PER; e0 += 4) {
                float x[4];
                u64 w[4];
                int b[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {  // side by side, before the branches
                    x[e] = to_f32(in[e0 + e]);
                    w[e] = weigh(x[e]);
                    b[e] = bins.bin_of(x[e]);
                }
                bins.add(b, w);
                if (!extra) continue;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (o.floor > 0.0f && w[e] && (x[e] == weigh.peak || ((double)x[e] - (double)weigh.peak) * weigh.c >= least_t)) above += w[e];
                    if (o.draft >= 0 && (x[e] > o.xd || (x[e] == o.xd && i0 + e0 + e < o.draft))) before += w[e];
                }
            }
        });
        u64 mass, above_all = 0, before_all = 0;
        unsigned count;
        if (extra) {
            unsigned none = 0;
            u64 sum = above;
            block_scan(s.scan, sum, none, above, count);
            sum = before;
            block_scan(s.scan, sum, none, before, count);
            if (tid < row.C) {
                Told *t = row.of(&s.told[1][row.rank], tid);
                t->above = above;
                t->before_draft = before;
            }
        }
        bins.merge(0, 0, 0, mass, count);
        for (int c = 0; c < row.C; c++) {
            above_all += s.told[1][c].above;
            before_all += s.told[1][c].before_draft;
        }
        const Draw d = draw(bins, o, weigh, mass, count, above_all, before_all);
        token = d.draft ? o.draft : d.at.index;
        prob = (float)((double)d.w / (double)d.mass);
    }
    if (row.rank == 0 && tid == 0) {
        a.out[r] = token;
        if (a.prob) a.prob[r] = prob;
    }
}

// False, with nothing written, if a value that is not counted weighs anything.
__device__ bool sample_values(ValuesShared &s, unsigned *sum, Row<bf16> &row, const SampleArgs &a, const Choice &o, int r) {
    const int tid = threadIdx.x;
    Values values = {s, row, row.C > 1 ? sum : s.count};
    values.stream();
    if (tid < row.C) {
        Told *t = row.of(&s.told[row.rank], tid);
        t->first = s.top;
        t->low = s.tiny;
        t->high = s.outer;
    }
    row.arrive();
    Weigher weigh = weigher(0.0f, o.temperature);
    row.wait();
    const Told &told = s.told[min(tid % 32, row.C - 1)];
    const unsigned top = __reduce_max_sync(0xffffffffu, told.first), tiny = __reduce_max_sync(0xffffffffu, told.low),
                   outer = __reduce_max_sync(0xffffffffu, told.high);
    if (top == 0) {  // no tokens
        if (row.rank == 0 && tid == 0) {
            a.out[r] = -1;
            if (a.prob) a.prob[r] = 0.0f;
        }
        return true;
    }
    const float peak = of_key(top);
    const int peak_pos = pos_of(__bfloat16_as_ushort(__float2bfloat16(peak)));
    if (peak_pos < 0) return false;
    Crossing at = {0, 1, -1, peak_pos, 0};
    float prob = 1.0f;
    if (o.temperature > 0.0f) {
        weigh.peak = peak;
        if (outer && weigh(of_key(outer)) > 0) return false;
        if (tiny && (peak < SL_TINY || weigh(SL_TINY) > 0)) return false;
        values.weigh = weigh;
        values.merge(o.draft, o.xd);
        if (row.rank != 0) return true;
        u64 mass;
        unsigned count;
        values.scan(mass, count);
        if (tid < 32) {
            __syncwarp();
            u64 above = 0, before = 0;
            if (o.floor > 0.0f) {
                const double least_t = log2((double)fminf(o.floor, 1.0f));
                above = values.before(first_values([&](float x) {
                    return x >= peak || ((double)x - (double)peak) * weigh.c >= least_t;
                }));
            }
            if (o.draft >= 0) {
                const int pos = pos_of(__bfloat16_as_ushort(__float2bfloat16(o.xd)));
                unsigned ahead = 0;
                for (int c = 0; c < row.C; c++) ahead += s.equals[c];
                if (pos >= 0) before = values.before(pos) + ahead * weigh(o.xd);  // else it weighs nothing
            }
            const Draw d = draw(values, o, weigh, mass, count, above, before);
            if (tid == 0) {
                s.at = d.at;
                s.is_draft = d.draft;
                s.prob = (float)((double)d.w / (double)d.mass);
            }
        }
        __syncthreads();
        at = s.at;
        prob = s.prob;
        if (s.is_draft) {
            if (tid == 0) {
                a.out[r] = o.draft;
                if (a.prob) a.prob[r] = prob;
            }
            return true;
        }
    }
    if (row.rank != 0) return true;
    const int token = values.index(at);
    if (tid == 0) {
        a.out[r] = token;
        if (a.prob) a.prob[r] = prob;
    }
    return true;
}

template <typename T>
__global__ void __launch_bounds__(SL_THREADS, 2) sample_logits_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sl_smem[];
    constexpr bool VALUES = sizeof(T) == 2;
    const cg::cluster_group cluster = cg::this_cluster();
    Row<T> row = {cluster, (int)cluster.num_blocks(), (int)cluster.block_rank(), nullptr, a.vocab, 0, a.slice};
    const int r = blockIdx.x / row.C;
    if constexpr (VALUES) {
        Values values = {*reinterpret_cast<ValuesShared *>(sl_smem), row};
        values.zero();
    }
    pdl_trigger();
    pdl_wait();
    row.sync();  // the others are there to be written to
    row.in = static_cast<const T *>(a.logits) + r * a.stride;
    row.i0 = row.rank * a.slice - (int)((reinterpret_cast<uintptr_t>(row.in) & 15) / sizeof(T));
    Choice o;
    o.temperature = a.temperature ? a.temperature[r] : 1.0f;
    o.k = a.top_k ? a.top_k[r] : 0;
    o.p = a.top_p ? a.top_p[r] : 1.0f;
    o.floor = a.min_p ? a.min_p[r] : 0.0f;
    o.u = fminf(fmaxf(a.u[r], 0.0f), 0x1.fffffep-1f);  // NaN is 0
    o.draft = a.draft ? a.draft[r] : -1;
    o.xd = o.draft >= 0 && o.draft < a.vocab ? to_f32(row.in[o.draft]) : -INFINITY;
    if (!(o.xd > -INFINITY)) o.draft = -1;
    bool done = false;
    if constexpr (VALUES) {
        ValuesShared &s = *reinterpret_cast<ValuesShared *>(sl_smem);
        done = sample_values(s, reinterpret_cast<unsigned *>(sl_smem + (sizeof(ValuesShared) + 15) / 16 * 16), row, a, o, r);
        if (!done) row.sync();  // the same in every CTA; what they have told one another is read
    }
    if (!done) sample_bins(*reinterpret_cast<BinsShared *>(sl_smem), row, a, o, r);
    row.sync();  // the other CTAs have read this one's shared memory
}

}  // namespace

}  // namespace q3

using namespace q3;

extern "C" {

int q3_sample_logits(int *out, float *prob, const void *logits, int dtype, int rows, int vocab, long long stride, const float *u,
                     const float *temperature, const int *top_k, const float *top_p, const float *min_p, const int *draft,
                     void *stream) {
    if (dtype != 0 && dtype != 1) return Q3_ERR_ARG;
    if (rows < 0 || rows > (1 << 24) || vocab <= 0 || vocab > SL_VOCAB || stride < vocab) return Q3_ERR_SHAPE;
    if (rows == 0) return Q3_OK;  // before the pointers: tensors of no elements have none
    if (!out || !logits || !u) return Q3_ERR_ARG;
    const int elt = dtype ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) & (elt - 1)) return Q3_ERR_ALIGN;
    const int st = check_device();
    if (st != Q3_OK) return st;
    // CTAs of a row: two for each SM while a slice has work for its threads
    auto slice_of = [&](int c) { return ((vocab + 16 / elt - 1 + c - 1) / c + 7) / 8 * 8; };
    int c = 1;
    while (c < SL_MAX_CLUSTER && (slice_of(c) > SL_SLICE || ((long long)(c + 1) * rows <= 2 * num_sms() && slice_of(c) > 8 * SL_THREADS)))
        c++;
    SampleArgs a = {out, prob, logits, stride, vocab, slice_of(c), u, temperature, top_p, min_p, top_k, draft};
    size_t smem = sizeof(BinsShared);
    if (dtype == 0) smem = std::max(smem, (sizeof(ValuesShared) + 15) / 16 * 16 + (c > 1 ? SL_PLACES * sizeof(unsigned) : 0));
    auto kernel = dtype == 0 ? sample_logits_kernel<bf16> : sample_logits_kernel<float>;
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(kernel, dim3((unsigned)rows * c), dim3(SL_THREADS), smem, (cudaStream_t)stream, c, a));
    return Q3_OK;
}

}  // extern "C"
