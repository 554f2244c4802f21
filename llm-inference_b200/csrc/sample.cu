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
// Weights are whole numbers, round(2^bits w), from exponentials in fp64: their sums are the same in any order, so neither the
// atomics below nor the way the row is cut change a result, and a draw is decided as in 64 bits.
//
// A cluster of CTAs shares a row. Two ways to find a crossing:
//   - bf16 logits have few values: one pass counts each value between 2^-24 and 2^8 of either sign, and zeros (one shared-memory
//     atomic a token, the exponentials once per value that occurs). Equal tokens weigh the same, so a running sum over
//     the values says which value and which of its tokens; one more pass, by the CTA that has it, finds its index.
//   - fp32 logits, and bf16 rows in which a value outside those weighs anything: a pass for the largest, one for a
//     histogram of mass and count over the logits, and per crossing one that gathers the tokens of its bin, which are ranked by
//     comparing each with each. A bin of too many tokens is cut finer by the bits of its logits; as many equal ones are
//     told apart by counting them in the order of their index.
// CTAs write what all of a cluster need into each other's shared memory before a cluster barrier (reading it after one, C
// loads that wait for one another, cost more than all the arithmetic).
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
constexpr int SL_SLICE = 1 << 17;  // tokens of a CTA at most: 15-bit parts of their weights add up within 32 bits
constexpr int SL_VOCAB = SL_MAX_CLUSTER * (SL_SLICE - 64);
constexpr int SL_LOADS = 4;  // 16-byte loads that a thread has in flight

typedef unsigned long long u64;

struct SampleArgs {
    int *out;
    float *prob;
    const void *logits;
    long long stride;
    int vocab, slice, bits;  // slice: tokens of a CTA, a multiple of 8
    const float *u, *temperature, *top_p, *min_p;
    const int *top_k, *draft;
};

// What a CTA tells the others.
struct Told {
    u64 mass, above, before_draft;  // of its share of the bins; its mass above min-p's limit and before the draft
    u64 first;                      // its largest token: key in the upper half, complement of the index below
    unsigned count, low, high;
};

// Where a running sum passes a target: the token's weight, what comes before it, and which token it is.
struct Crossing {
    u64 before, w;
    int index;  // of the token; of a value: -1
    int pos, owner;
    unsigned nth;  // the value's place, the CTA that has the token and which of its tokens of that value it is
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
    int bits;
    // round(2^bits * 2^((x - peak) c)): the power's whole part goes to the exponent, the rest f in [-1/2, 1/2] through the
    // Taylor polynomial of e^(f ln 2) (the first term left out is below 3e-13). No branches, so that a thread's
    // weights overlap: one chain of these operations is 200 cycles.
    __device__ __forceinline__ u64 operator()(float x) const {
        const double t = ((double)x - (double)peak) * c;
        const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number, kept in the low bits
        const double shifted = t + magic;
        const int n = __double2loint(shifted);
        const double f = t - (shifted - magic);
        double y = 7.054911620801121e-09;  // (ln 2)^k / k!, k = 10 down
        y = fma(y, f, 1.0178086009239696e-07);
        y = fma(y, f, 1.3215486790144305e-06);
        y = fma(y, f, 1.5252733804059838e-05);
        y = fma(y, f, 0.00015403530393381606);
        y = fma(y, f, 0.0013333558146428441);
        y = fma(y, f, 0.009618129107628477);
        y = fma(y, f, 0.055504108664821576);
        y = fma(y, f, 0.2402265069591007);
        y = fma(y, f, 0.6931471805599453);
        y = fma(y, f, 1.0);
        y = __hiloint2double(__double2hiint(y) + ((n + bits) << 20), __double2loint(y));
        const u64 w = (u64)__double_as_longlong(y + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: the sum's fraction bits
        return x == peak ? 1ull << bits : t > -46.0 ? w : 0;
    }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Exclusive running sum over the CTA's threads; `total` is everyone's sum.
__device__ __forceinline__ u64 block_scan(u64 v, u64 *scan, u64 *total) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    u64 run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
    }
    __syncthreads();  // earlier readers of scan
    if (lane == 31) scan[warp] = run;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < SL_WARPS; w++) {
        if (w < warp) before += scan[w];
        all += scan[w];
    }
    *total = all;
    return before + run - v;
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
        if (C > 1) cluster.sync();
        else __syncthreads();
    }
    template <typename V>
    __device__ __forceinline__ V *of(V *p, int r) { return C > 1 ? cluster.map_shared_rank(p, r) : p; }

    // A line of the row; places outside it hold -infinity.
    __device__ __forceinline__ uint4 line(int i) const {
        if (i >= 0 && i + PER <= vocab) return __ldg(reinterpret_cast<const uint4 *>(in + i));
        uint4 raw;
        T *x = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int e = 0; e < PER; e++) x[e] = i + e >= 0 && i + e < vocab ? in[i + e] : T(-INFINITY);
        return raw;
    }
    // f(line, index of its first place) over the slice, several loads in flight
    template <typename F>
    __device__ __forceinline__ void each_line(F f) const {
        for (int v = threadIdx.x * PER; v < slice; v += SL_LOADS * SL_THREADS * PER) {
            uint4 raw[SL_LOADS];
#pragma unroll
            for (int l = 0; l < SL_LOADS; l++)
                if (v + l * SL_THREADS * PER < slice) raw[l] = line(i0 + v + l * SL_THREADS * PER);
#pragma unroll
            for (int l = 0; l < SL_LOADS; l++)
                if (v + l * SL_THREADS * PER < slice) f(raw[l], i0 + v + l * SL_THREADS * PER);
        }
    }
    // f(x, index); NaN comes as -infinity
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each_line([&](const uint4 &raw, int i) {
            const T *x = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const float v = to_f32(x[e]);
                f(v == v ? v : -INFINITY, i + e);
            }
        });
    }
};

// ------------------------------------------------------------------ any logits: histogram and gathered bins

constexpr int SL_BINS = 1024;
constexpr int SL_CAND = 256;  // tokens of a bin that are ranked directly

struct Candidate {
    u64 order;  // key in the upper half, complement of the index below: larger comes earlier
    u64 w;
};

struct BinsShared {
    unsigned part[3][SL_BINS];  // this CTA's histogram: 15-bit parts of the weights
    unsigned count[SL_BINS];
    u64 sum_mass[2][SL_BINS];   // the cluster's, this CTA's share of the bins; [1]: of a bin that was cut finer
    unsigned sum_count[2][SL_BINS];
    Candidate list[2][SL_CAND];  // this CTA's tokens of the bin in question; finds take turns
    Candidate all[SL_CAND];      // and the cluster's
    unsigned n_list, key_lo, key_hi;
    Told told[4][SL_MAX_CLUSTER];  // level 0's totals, a cut bin's, and the lists' (by turns)
    u64 bin_mass;                  // before the bin where a find's target lies
    unsigned bin_count;
    int bin, tie;
    Crossing found;
    u64 scan[SL_WARPS];
};

template <typename T>
struct Bins {
    BinsShared &s;
    Row<T> &row;
    Weigher weigh;
    float per_bin;
    int turn = 0;

    // by adding 2^23, which leaves the nearest whole number in the low bits
    __device__ __forceinline__ int bin_of(float x) const {
        return __float_as_int(fminf((weigh.peak - x) * per_bin, SL_BINS - 1.0f) + 8388608.0f) & (SL_BINS - 1);
    }

    __device__ __forceinline__ void zero() {
        for (int b = threadIdx.x; b < SL_BINS; b += SL_THREADS) s.part[0][b] = s.part[1][b] = s.part[2][b] = s.count[b] = 0;
    }
    // 64-bit atomics in shared memory are loops; most weights have few parts
    __device__ __forceinline__ void add(int b, u64 w) {
        const unsigned p0 = (unsigned)w & 0x7fff, p1 = (unsigned)(w >> 15) & 0x7fff, p2 = (unsigned)(w >> 30);
        if (p0) atomicAdd(&s.part[0][b], p0);
        if (p1) atomicAdd(&s.part[1][b], p1);
        if (p2) atomicAdd(&s.part[2][b], p2);
        if (w) atomicAdd(&s.count[b], 1u);
    }

    // The CTAs' histograms into sum_*[level], each CTA its share of the bins; everyone learns the shares' totals, and what
    // else each CTA has to tell.
    __device__ void merge(int level, u64 above, u64 before_draft) {
        row.sync();
        const int share = (SL_BINS + row.C - 1) / row.C, first = row.rank * share, n_own = min(share, SL_BINS - first);
        u64 m = 0, n = 0;
        for (int b = threadIdx.x; b < n_own; b += SL_THREADS) {
            u64 mass = 0;
            unsigned count = 0;
#pragma unroll
            for (int r = 0; r < SL_MAX_CLUSTER; r++)
                if (r < row.C) {
                    const unsigned p0 = row.of(s.part[0], r)[first + b], p1 = row.of(s.part[1], r)[first + b],
                                   p2 = row.of(s.part[2], r)[first + b];
                    mass += p0 + ((u64)p1 << 15) + ((u64)p2 << 30);
                    count += row.of(s.count, r)[first + b];
                }
            s.sum_mass[level][b] = mass;
            s.sum_count[level][b] = count;
            m += mass;
            n += count;
        }
        u64 mass, count;
        block_scan(m, s.scan, &mass);
        block_scan(n, s.scan, &count);
        if (threadIdx.x < row.C) {
            Told *t = row.of(&s.told[level][row.rank], threadIdx.x);
            t->mass = mass;
            t->count = (unsigned)count;
            t->above = above;
            t->before_draft = before_draft;
        }
        row.sync();
    }

    // The bin where the running mass (or count) passes `target`, and mass and count before it; the target lies in a bin.
    __device__ void find_bin(int level, u64 target, bool by_count, u64 &mass, unsigned &count, int &bin) {
        int owner = 0;
        for (; owner < row.C - 1; owner++) {
            const u64 m = s.told[level][owner].mass;
            const unsigned n = s.told[level][owner].count;
            if ((by_count ? count + n : mass + m) > target) break;
            mass += m;
            count += n;
        }
        const int share = (SL_BINS + row.C - 1) / row.C, first = owner * share, n_own = min(share, SL_BINS - first);
        if (row.rank == owner) {
            constexpr int EACH = SL_BINS / SL_THREADS;
            u64 m[EACH], n[EACH], tm = 0, tn = 0, total;
            const int b0 = threadIdx.x * EACH;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                m[e] = b0 + e < n_own ? s.sum_mass[level][b0 + e] : 0;
                n[e] = b0 + e < n_own ? s.sum_count[level][b0 + e] : 0;
                tm += m[e];
                tn += n[e];
            }
            u64 bm = mass + block_scan(tm, s.scan, &total), bn = count + block_scan(tn, s.scan, &total);
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const u64 lo = by_count ? bn : bm, hi = lo + (by_count ? n[e] : m[e]);
                if (lo <= target && target < hi)
                    for (int r = 0; r < row.C; r++) {
                        *row.of(&s.bin, r) = first + b0 + e;
                        *row.of(&s.bin_mass, r) = bm;
                        *row.of(&s.bin_count, r) = (unsigned)bn;
                    }
                bm += m[e];
                bn += n[e];
            }
        }
        row.sync();
        bin = s.bin;
        mass = s.bin_mass;
        count = s.bin_count;
    }

    // The token where the running mass (or count) of the row passes `target`, which lies in the row.
    __device__ Crossing find(u64 target, bool by_count) {
        u64 mass = 0;
        unsigned count = 0, lo = 0, hi = 0;  // lo, hi: keys of the tokens in question, once the first bin is cut
        int bin = 0;
        bool cut = false;
        find_bin(0, target, by_count, mass, count, bin);
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
            row.each([&](float x, int i) {
                const unsigned key = key_of(x);
                if (cut ? key < lo || key > hi : bin_of(x) != bin) return;
                const u64 w = weigh(x);
                if (w == 0) return;
                const unsigned at = atomicAdd(&s.n_list, 1u);
                if (at < SL_CAND) list[at] = {(u64)key << 32 | (unsigned)~i, w};
                atomicMin(&s.key_lo, key);
                atomicMax(&s.key_hi, key);
            });
            __syncthreads();
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
            row.each([&](float x, int) {
                const unsigned key = key_of(x);
                if (key >= lo && key <= hi) add((hi - key) >> shift, weigh(x));
            });
            merge(1, 0, 0);
            find_bin(1, target, by_count, mass, count, bin);
            const unsigned span = (1u << shift) - 1;
            hi -= (unsigned)bin << shift;
            lo = hi - lo > span ? hi - span : lo;
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
        for (unsigned j = from; j < n; j += sub)
            if (s.all[j].order > own.order) {
                before += s.all[j].w;
                places++;
            }
        for (int o = sub / 2; o > 0; o /= 2) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            places += __shfl_xor_sync(0xffffffffu, places, o);
        }
        before += mass;
        places += count;
        if (mine < n && from == 0 && (by_count ? places == target : before <= target && target < before + own.w))
            s.found = {before, own.w, (int)~(unsigned)own.order, 0, 0, 0};
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
                u64 here;
                const u64 before = block_scan(is, s.scan, &here);
                if (is && before == left)
                    for (int r = 0; r < row.C; r++) *row.of(&s.tie, r) = i;
                if (left < here) break;
                left -= here;
            }
        }
        row.sync();
        return {mass + nth * w, w, s.tie, 0, 0, 0};
    }

    __device__ __forceinline__ int index(const Crossing &f) { return f.index; }
};

// ------------------------------------------------------------------ bf16 logits: counts of their values

constexpr int SL_LOW = (127 - 24) << 7, SL_HIGH = (127 + 8) << 7;  // magnitudes that are counted, from 2^-24 to below 2^8
constexpr int SL_SIGN = SL_HIGH - SL_LOW;
constexpr int SL_VALUES = 2 * SL_SIGN + 1;  // in the order of the values: positive ones, zero, negative ones

struct ValuesShared {
    unsigned count[SL_VALUES + 3];  // this CTA's
    Told told[SL_MAX_CLUSTER], told_first[SL_MAX_CLUSTER];
    Crossing found[2];  // finds take turns, so that the next one's writer does not meet the readers of this one
    unsigned tiny, zeros, equal;  // low magnitudes but zero; the draft's equals before it in its CTA
    unsigned outer;               // key of the largest of high magnitude, 0: none
    int index;
    u64 sums[2];
    unsigned top;
    u64 scan[SL_WARPS];
    unsigned warps[SL_WARPS];
};

__device__ __forceinline__ bf16 value_of(int pos) {
    const int m = pos < SL_SIGN ? SL_HIGH - 1 - pos : pos == SL_SIGN ? 0 : SL_LOW + (pos - SL_SIGN - 1) + 0x8000;
    return __ushort_as_bfloat16((unsigned short)m);
}
// The value's place, -1 if it is not counted.
__device__ __forceinline__ int pos_of(unsigned h) {
    const unsigned m = h & 0x7fff;
    if (m == 0) return SL_SIGN;
    if (m - SL_LOW >= SL_SIGN) return -1;
    return h & 0x8000 ? SL_SIGN + 1 + (m - SL_LOW) : SL_HIGH - 1 - m;
}

struct Values {
    ValuesShared &s;
    Row<bf16> &row;
    unsigned *sum;  // this CTA's share of the cluster's counts
    Weigher weigh;
    int share, each, base;  // values of a CTA's share and of a thread; the thread's first one
    u64 before_mass, mass;  // of the thread's values
    unsigned before_count, count;
    int turn = 0;

    // bits of a line's places that hold the value; zeros are one
    static __device__ __forceinline__ unsigned equals(const uint4 &raw, unsigned value) {
        unsigned n = 0;
        const unsigned *h = reinterpret_cast<const unsigned *>(&raw);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            unsigned a = h[e] & 0xffff, b = h[e] >> 16;
            if (a == 0x8000) a = 0;
            if (b == 0x8000) b = 0;
            n |= (a == value ? 1u : 0u) << 2 * e | (b == value ? 2u : 0u) << 2 * e;
        }
        return n;
    }

    __device__ __forceinline__ void zero() {
        for (int v = threadIdx.x; v < SL_VALUES; v += SL_THREADS) s.count[v] = 0;
        if (threadIdx.x == 0) s.tiny = s.zeros = s.outer = s.equal = s.top = 0;
    }

    // One pass over the slice: counts, and the largest value.
    __device__ void stream() {
        __nv_bfloat162 top = __floats2bfloat162_rn(-INFINITY, -INFINITY);
        unsigned zeros = 0, tiny = 0, outer = 0;
        row.each_line([&](const uint4 &raw, int) {
            const unsigned *h = reinterpret_cast<const unsigned *>(&raw);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                top = __hmax2(top, *reinterpret_cast<const __nv_bfloat162 *>(&h[e]));  // not NaN, if either is not
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const unsigned v = k ? h[e] >> 16 : h[e] & 0xffff, m = v & 0x7fff, off = m - SL_LOW;
                    if (off < (unsigned)SL_SIGN) atomicAdd(&s.count[v & 0x8000 ? SL_SIGN + 1 + off : SL_SIGN - 1 - off], 1u);
                    else if (m == 0) zeros++;
                    else if (m < SL_LOW) tiny = 1;
                    else if (m <= 0x7f80 && v != 0xff80) outer = max(outer, key_of(__uint_as_float(v << 16)));
                }
            }
        });
        float t = fmaxf(__low2float(top), __high2float(top));
        t = t == t ? t : -INFINITY;
        const unsigned best = __reduce_max_sync(0xffffffffu, t > -INFINITY ? key_of(t) : 0);
        zeros = __reduce_add_sync(0xffffffffu, zeros);
        tiny = __reduce_or_sync(0xffffffffu, tiny);
        outer = __reduce_max_sync(0xffffffffu, outer);
        if (threadIdx.x % 32 == 0) {
            atomicMax(&s.top, best);
            if (zeros) atomicAdd(&s.count[SL_SIGN], zeros);
            if (tiny) s.tiny = 1;
            if (outer) atomicMax(&s.outer, outer);
        }
        __syncthreads();
    }

    // The CTAs' counts, each CTA its share; everyone learns the shares' totals. draft: index, or -1.
    __device__ void merge(bool has_floor, double least_t, int draft, float xd) {
        share = (SL_VALUES + row.C - 1) / row.C;
        const int first = row.rank * share, n_own = max(0, min(share, SL_VALUES - first));
        if (row.C > 1) {
#pragma unroll 4
            for (int b = threadIdx.x; b < n_own; b += SL_THREADS) {
                unsigned n = 0;
#pragma unroll
                for (int r = 0; r < SL_MAX_CLUSTER; r++)
                    if (r < row.C) n += row.of(s.count, r)[first + b];
                sum[b] = n;
            }
            __syncthreads();
        }
        const unsigned value = draft < 0 || xd == 0.0f ? 0 : (unsigned)__bfloat16_as_ushort(__float2bfloat16(xd));
        const int draft_pos = draft < 0 ? 0 : pos_of(value);  // -1: it weighs nothing
        const u64 wd = draft < 0 ? 0 : weigh(xd);
        each = (share + SL_THREADS - 1) / SL_THREADS;
        base = threadIdx.x * each;
        mass = 0;
        count = 0;
        u64 above = 0, ahead = 0;
        for (int e = 0; e < each; e++) {
            const unsigned n = base + e < n_own ? sum[base + e] : 0;
            if (n == 0) continue;
            const int pos = first + base + e;
            const float x = to_f32(value_of(pos));
            const u64 w = weigh(x);
            if (w == 0) continue;
            const u64 m = n * w;
            mass += m;
            count += n;
            if (has_floor && (x == weigh.peak || ((double)x - (double)weigh.peak) * weigh.c >= least_t)) above += m;
            if (wd > 0 && pos < draft_pos) ahead += m;
        }
        u64 all_mass, all_count;
        before_mass = block_scan(mass, s.scan, &all_mass);
        before_count = (unsigned)block_scan(count, s.scan, &all_count);
        if (has_floor || wd > 0) {
            above = warp_sum(above);
            ahead = warp_sum(ahead);
            if (threadIdx.x < 2) s.sums[threadIdx.x] = 0;
            __syncthreads();
            if (threadIdx.x % 32 == 0) {
                atomicAdd(&s.sums[0], above);
                atomicAdd(&s.sums[1], ahead);
            }
            if (wd > 0) {  // its equals with a smaller index
                const unsigned here = s.count[draft_pos];
                if (here > 0 && row.i0 + row.slice <= draft) {
                    if (threadIdx.x == 0) s.equal = here;
                } else if (here > 1 && row.i0 < draft) {
                    unsigned n = 0;
                    row.each_line([&](const uint4 &raw, int i) {
                        const unsigned is = equals(raw, value);
                        n += __popc(i + Row<bf16>::PER <= draft ? is : i < draft ? is & ((1u << (draft - i)) - 1) : 0);
                    });
                    n = __reduce_add_sync(0xffffffffu, n);
                    if (threadIdx.x % 32 == 0) atomicAdd(&s.equal, n);
                }
            }
            __syncthreads();
            above = s.sums[0];
            ahead = s.sums[1] + s.equal * wd;
        }
        if (threadIdx.x < row.C) {
            Told *t = row.of(&s.told[row.rank], threadIdx.x);
            t->mass = all_mass;
            t->count = (unsigned)all_count;
            t->above = above;
            t->before_draft = ahead;
        }
        row.sync();
    }

    // The token where the running mass (or count) of the row passes `target`, which lies in the row: which one of which value.
    __device__ Crossing find(u64 target, bool by_count) {
        u64 m0 = 0, n0 = 0;
        int owner = 0;
        for (; owner < row.C - 1; owner++) {
            const u64 m = s.told[owner].mass, n = s.told[owner].count;
            if ((by_count ? n0 + n : m0 + m) > target) break;
            m0 += m;
            n0 += n;
        }
        if (row.rank == owner) {
            const u64 lo = by_count ? n0 + before_count : m0 + before_mass, hi = lo + (by_count ? count : mass);
            const bool mine = lo <= target && target < hi;
            const unsigned who = __ballot_sync(0xffffffffu, mine);
            if (who) {  // the warp where it lies takes the thread's values side by side
                const int src = __ffs(who) - 1, lane = threadIdx.x % 32;
                const int first = owner * share, n_own = min(share, SL_VALUES - first);
                const int b = __shfl_sync(0xffffffffu, base, src) + lane;
                const bool is = lane < each && b < n_own;
                const unsigned n = is ? sum[b] : 0;
                const u64 w = is ? weigh(to_f32(value_of(first + b))) : 0, m = n * w;
                const unsigned k = w ? n : 0;
                u64 bm = m;
                unsigned bn = k;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 ym = __shfl_up_sync(0xffffffffu, bm, o);
                    const unsigned yn = __shfl_up_sync(0xffffffffu, bn, o);
                    if (lane >= o) {
                        bm += ym;
                        bn += yn;
                    }
                }
                bm += m0 + __shfl_sync(0xffffffffu, before_mass, src) - m;
                bn += (unsigned)n0 + __shfl_sync(0xffffffffu, before_count, src) - k;
                if (k > 0 && (by_count ? bn <= target && target < bn + k : bm <= target && target < bm + m)) {
                    const unsigned nth = by_count ? (unsigned)target - bn : (unsigned)((target - bm) / w);
                    const Crossing f = {bm + nth * w, w, -1, first + b, 0, nth};
                    for (int r = 0; r < row.C; r++) *row.of(&s.found[turn], r) = f;
                }
            }
        }
        row.sync();
        const Crossing f = s.found[turn];
        turn ^= 1;
        return f;
    }

    // The index of a value's nth token in the CTA that has it, -1 in the others.
    __device__ int index(const Crossing &f) {
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
        unsigned n = lane < row.C ? row.of(s.count, lane)[f.pos] : 0, run = n;
#pragma unroll
        for (int o = 1; o < SL_MAX_CLUSTER; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += y;
        }
        const unsigned before = __shfl_sync(0xffffffffu, run - n, row.rank), here = __shfl_sync(0xffffffffu, n, row.rank);
        if (f.nth < before || f.nth >= before + here) return -1;
        const unsigned left = f.nth - before;
        // each warp a part of the slice; lane j keeps the count of its j-th 32 lines
        const unsigned value = __bfloat16_as_ushort(value_of(f.pos));
        const int lines = row.slice / 8, per_warp = (lines + SL_WARPS - 1) / SL_WARPS;
        const int first = warp * per_warp, last = min(lines, first + per_warp);
        unsigned mine = 0;
        for (int l0 = first, it = 0; l0 < last; l0 += 32 * SL_LOADS, it += SL_LOADS) {
            unsigned is[SL_LOADS];
#pragma unroll
            for (int l = 0; l < SL_LOADS; l++)
                is[l] = l0 + 32 * l + lane < last ? __popc(equals(row.line(row.i0 + 8 * (l0 + 32 * l + lane)), value)) : 0;
#pragma unroll
            for (int l = 0; l < SL_LOADS; l++) {
                const unsigned all = __reduce_add_sync(0xffffffffu, is[l]);
                if (lane == it + l) mine = all;
            }
        }
        const unsigned all = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) s.warps[warp] = all;
        __syncthreads();
        unsigned ahead = 0;
        for (int w = 0; w < warp; w++) ahead += s.warps[w];
        if (left >= ahead && left < ahead + all) {
            auto scan = [&](unsigned v) {
                unsigned r = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned y = __shfl_up_sync(0xffffffffu, r, o);
                    if (lane >= o) r += y;
                }
                return r - v;
            };
            unsigned b = ahead + scan(mine);
            unsigned who = __ballot_sync(0xffffffffu, left >= b && left < b + mine);
            const int it = __ffs(who) - 1;
            ahead = __shfl_sync(0xffffffffu, b, it);
            const int line = first + 32 * it + lane;
            unsigned is = line < last ? equals(row.line(row.i0 + 8 * line), value) : 0;
            b = ahead + scan(__popc(is));
            if (left >= b && left < b + __popc(is)) {
                for (unsigned k = left - b; k > 0; k--) is &= is - 1;
                s.index = row.i0 + 8 * line + __ffs(is) - 1;
            }
        }
        __syncthreads();
        return s.index;
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
    Draw d;
    if (o.k > 0 && (unsigned)o.k < count) {
        const Crossing f = finder.find((u64)(o.k - 1), true);
        mass = f.before + f.w;
    }
    if (o.p < 1.0f) {  // the shortest beginning with at least p of the mass
        const double want = ceil((double)fmaxf(o.p, 0.0f) * (double)mass);
        const Crossing f = finder.find(want < 1.0 ? 0 : min((u64)want, mass) - 1, false);
        mass = f.before + f.w;
    }
    if (o.floor > 0.0f) mass = min(mass, above);
    d.mass = mass;
    u64 target = min((u64)((double)o.u * (double)mass), mass - 1);
    const u64 wd = o.draft >= 0 ? weigh(o.xd) : 0;
    const bool kept = wd > 0 && before_draft < mass;
    d.draft = kept && target < wd;
    d.w = wd;
    if (!d.draft) {
        if (kept && target - wd < before_draft) target -= wd;  // the draft's place in the order is empty
        d.at = finder.find(target, false);
        d.w = d.at.w;
    }
    return d;
}

__device__ __forceinline__ Weigher weigher(float peak, float temperature, int bits) {
    // an infinite temperature makes all finite logits weigh the same, -infinity still nothing
    return {peak, fmax(1.4426950408889634 / (double)temperature, 1e-300), bits};
}

template <typename T>
__device__ void sample_bins(BinsShared &s, Row<T> &row, const SampleArgs &a, const Choice &o, int r) {
    const int tid = threadIdx.x;
    // the largest token, and the smallest finite logit
    float top = -INFINITY, low = INFINITY;
    int at = 0;
    row.each([&](float x, int i) {
        if (x > top) {
            top = x;
            at = i;
        }
        if (x > -INFINITY) low = fminf(low, x);
    });
    const u64 best = warp_max(top > -INFINITY ? (u64)key_of(top) << 32 | (unsigned)~at : 0);
    const unsigned least = __reduce_min_sync(0xffffffffu, key_of(low));
    if (tid % 32 == 0) {
        s.scan[tid / 32] = best;
        s.all[tid / 32].order = least;
    }
    Bins<T> bins = {s, row, {}, 0.0f};
    bins.zero();
    __syncthreads();
    if (tid < row.C) {
        u64 f = 0, l = 0xffffffffu;
        for (int w = 0; w < SL_WARPS; w++) {
            f = max(f, s.scan[w]);
            l = min(l, s.all[w].order);
        }
        Told *t = row.of(&s.told[1][row.rank], tid);
        t->first = f;
        t->low = (unsigned)l;
    }
    row.sync();
    u64 first = 0;
    unsigned min_key = 0xffffffffu;
    for (int c = 0; c < row.C; c++) {
        first = max(first, s.told[1][c].first);
        min_key = min(min_key, s.told[1][c].low);
    }
    int token = first ? (int)~(unsigned)first : -1;
    float prob = first ? 1.0f : 0.0f;
    if (first && o.temperature > 0.0f) {
        const Weigher weigh = weigher(of_key((unsigned)(first >> 32)), o.temperature, a.bits);
        bins.weigh = weigh;
        const float range = fminf((float)(46.0 / weigh.c), weigh.peak - of_key(min_key));
        bins.per_bin = range > 0.0f ? fminf(SL_BINS / range, 1e30f) : 0.0f;
        const double least_t = o.floor > 0.0f ? log2((double)fminf(o.floor, 1.0f)) : 0.0;
        // the histogram, the mass above min-p's limit, the mass before the draft
        u64 above = 0, before = 0;
        row.each([&](float x, int i) {
            const u64 w = weigh(x);
            bins.add(bins.bin_of(x), w);
            if (o.floor > 0.0f && w && (x == weigh.peak || ((double)x - (double)weigh.peak) * weigh.c >= least_t)) above += w;
            if (o.draft >= 0 && (x > o.xd || (x == o.xd && i < o.draft))) before += w;
        });
        if (o.floor > 0.0f || o.draft >= 0) {
            u64 sum;
            block_scan(above, s.scan, &sum);
            above = sum;
            block_scan(before, s.scan, &sum);
            before = sum;
        }
        bins.merge(0, above, before);
        u64 mass = 0, above_all = 0, before_all = 0;
        unsigned count = 0;
        for (int c = 0; c < row.C; c++) {
            mass += s.told[0][c].mass;
            count += s.told[0][c].count;
            above_all += s.told[0][c].above;
            before_all += s.told[0][c].before_draft;
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
        Told *t = row.of(&s.told_first[row.rank], tid);
        t->first = s.top;
        t->low = s.tiny;
        t->high = s.outer;
    }
    row.sync();
    unsigned top = 0, tiny = 0, outer = 0;
    for (int c = 0; c < row.C; c++) {
        top = max(top, (unsigned)s.told_first[c].first);
        tiny |= s.told_first[c].low;
        outer = max(outer, s.told_first[c].high);
    }
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
    const bool greedy = !(o.temperature > 0.0f);
    const Weigher weigh = weigher(peak, greedy ? 1.0f : o.temperature, a.bits);
    values.weigh = weigh;
    Crossing at = {0, 1, -1, peak_pos, 0, 0};
    bool is_draft = false;
    float prob = 1.0f;
    if (!greedy) {
        if (outer && weigh(of_key(outer)) > 0) return false;
        if (tiny && (peak < 0x1p-24f || weigh(0x1p-24f) > 0)) return false;
        const double least_t = o.floor > 0.0f ? log2((double)fminf(o.floor, 1.0f)) : 0.0;
        values.merge(o.floor > 0.0f, least_t, o.draft, o.xd);
        u64 mass = 0, above = 0, before = 0;
        unsigned count = 0;
        for (int c = 0; c < row.C; c++) {
            mass += s.told[c].mass;
            count += s.told[c].count;
            above += s.told[c].above;
            before += s.told[c].before_draft;
        }
        const Draw d = draw(values, o, weigh, mass, count, above, before);
        prob = (float)((double)d.w / (double)d.mass);
        is_draft = d.draft;
        at = d.at;
    }
    const int token = is_draft ? (row.rank == 0 ? o.draft : -1) : values.index(at);
    if (token >= 0 && tid == 0) {
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
    const int bits = vocab <= (1 << 18) ? 44 : 42;  // the whole row's mass stays below 2^62
    SampleArgs a = {out, prob, logits, stride, vocab, slice_of(c), bits, u, temperature, top_p, min_p, top_k, draft};
    size_t smem = sizeof(BinsShared);
    if (dtype == 0) smem = std::max(smem, (sizeof(ValuesShared) + 15) / 16 * 16 + (c > 1 ? ((SL_VALUES + c - 1) / c) * 4 : 0));
    auto kernel = dtype == 0 ? sample_logits_kernel<bf16> : sample_logits_kernel<float>;
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(kernel, dim3((unsigned)rows * c), dim3(SL_THREADS), smem, (cudaStream_t)stream, c, a));
    return Q3_OK;
}

}  // extern "C"
