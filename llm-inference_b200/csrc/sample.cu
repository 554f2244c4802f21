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
// A cluster of CTAs holds a row in shared memory. It builds one histogram of mass and count over the logits; a crossing is
// looked up in its running sums, and the tokens of the one bin where it lies are gathered and ranked by comparing each
// with each. A bin with too many tokens is cut finer by the bits of its logits; as many equal ones are told apart by
// counting them in the order of their index.
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
constexpr int SL_BINS = 1024;
constexpr int SL_CAND = 512;           // tokens of a bin that are ranked directly
constexpr int SL_MAX_CLUSTER = 8;
constexpr int SL_SLICE_BYTES = 160 * 1024;  // of a row in one CTA

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

struct Candidate {
    u64 order;  // key in the upper half, complement of the index below: larger comes earlier
    u64 w;
};

// Where a running sum passes a target: the token, and what comes before it.
struct Crossing {
    u64 before, w;
    int index;
};

struct SampleShared {
    u64 mass[SL_BINS];      // this CTA's histogram
    unsigned count[SL_BINS];
    u64 sum_mass[2][SL_BINS];  // the cluster's, this CTA's share of the bins; [1]: of a bin that was cut finer
    unsigned sum_count[2][SL_BINS];
    Candidate list[2][SL_CAND];  // this CTA's tokens of the bin in question; finds take turns
    Candidate all[SL_CAND];      // and the cluster's
    u64 part_mass[2];            // of this CTA's share of the bins
    unsigned part_count[2];
    unsigned n_list[2], key_lo[2], key_hi[2];
    u64 first, floor_mass, before_draft;  // this CTA's largest token, its mass above min-p's limit and before the draft
    unsigned min_key;
    u64 bin_mass;  // before the bin where a find's target lies
    unsigned bin_count;
    int bin;
    int tie;
    Crossing found;
    u64 scan[SL_WARPS];
};

__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// Unsigned numbers in the order of the floats; both zeros are one.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// round(2^bits * 2^((x - peak) c)): the power's whole part goes to the exponent, the rest f in [-1/2, 1/2] through the
// Taylor polynomial of e^(f ln 2) (the first term left out is below 3e-13).
__device__ __forceinline__ u64 weight(float x, double peak, double c, int bits) {
    const double t = x == (float)peak ? 0.0 : ((double)x - peak) * c;
    if (!(t > -46.0)) return 0;
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
    return (u64)__double_as_longlong(y + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: the sum's fraction bits
}

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

template <typename T>
struct Sampler {
    SampleShared &s;
    const T *x_s;  // this CTA's slice; what is no token, and NaN, is -infinity there
    cg::cluster_group cluster;
    int C, rank, i0, slice;  // i0: index of the slice's first place
    double peak, c;
    int bits;
    float per_bin;
    int turn = 0;

    __device__ __forceinline__ void sync() {
        if (C > 1) cluster.sync();
        else __syncthreads();
    }

    template <typename V>
    __device__ __forceinline__ V *of(V *p, int r) { return C > 1 ? cluster.map_shared_rank(p, r) : p; }

    __device__ __forceinline__ int bin_of(float x) const { return min(SL_BINS - 1, (int)(((float)peak - x) * per_bin)); }

    // f(x, index) over the slice
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        constexpr int PER = 16 / sizeof(T);
        for (int v = threadIdx.x * PER; v < slice; v += SL_THREADS * PER) {
            const uint4 raw = *reinterpret_cast<const uint4 *>(x_s + v);
            const T *x = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int e = 0; e < PER; e++) f(to_f32(x[e]), i0 + v + e);
        }
    }

    // The CTAs' histograms into sum_*[level], each CTA its share of the bins.
    __device__ void merge(int level) {
        sync();
        const int share = SL_BINS / C;
        u64 m = 0;
        unsigned n = 0;
        for (int b = threadIdx.x; b < share; b += SL_THREADS) {
            u64 mass = 0;
            unsigned count = 0;
            for (int r = 0; r < C; r++) {
                mass += of(s.mass, r)[rank * share + b];
                count += of(s.count, r)[rank * share + b];
            }
            s.sum_mass[level][b] = mass;
            s.sum_count[level][b] = count;
            m += mass;
            n += count;
        }
        u64 total;
        block_scan(m, s.scan, &total);
        if (threadIdx.x == 0) s.part_mass[level] = total;
        block_scan(n, s.scan, &total);
        if (threadIdx.x == 0) s.part_count[level] = (unsigned)total;
        sync();
    }

    // The bin where the running mass (or count) passes `target`, and mass and count before it; the target lies in a bin.
    __device__ void find_bin(int level, u64 target, bool by_count, u64 &mass, unsigned &count, int &bin) {
        int owner = 0;
        for (; owner < C - 1; owner++) {
            const u64 m = *of(&s.part_mass[level], owner);
            const unsigned n = *of(&s.part_count[level], owner);
            if ((by_count ? count + n : mass + m) > target) break;
            mass += m;
            count += n;
        }
        const int share = SL_BINS / C;
        if (rank == owner) {
            constexpr int EACH = SL_BINS / SL_THREADS;
            u64 m[EACH], n[EACH], tm = 0, tn = 0, total;
            const int b0 = threadIdx.x * EACH;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                m[e] = b0 + e < share ? s.sum_mass[level][b0 + e] : 0;
                n[e] = b0 + e < share ? s.sum_count[level][b0 + e] : 0;
                tm += m[e];
                tn += n[e];
            }
            u64 bm = mass + block_scan(tm, s.scan, &total), bn = count + block_scan(tn, s.scan, &total);
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const u64 lo = by_count ? bn : bm, hi = lo + (by_count ? n[e] : m[e]);
                if (lo <= target && target < hi) {
                    s.bin = owner * share + b0 + e;
                    s.bin_mass = bm;
                    s.bin_count = (unsigned)bn;
                }
                bm += m[e];
                bn += n[e];
            }
        }
        sync();
        bin = *of(&s.bin, owner);
        mass = *of(&s.bin_mass, owner);
        count = *of(&s.bin_count, owner);
    }

    // The token where the running mass (or count) of the row passes `target`, which lies in the row.
    __device__ Crossing find(u64 target, bool by_count) {
        u64 mass = 0;
        unsigned count = 0, lo = 0, hi = 0;  // keys of the tokens in question, once the first bin is cut
        int bin = 0;
        bool cut = false;
        int shift = 0;
        find_bin(0, target, by_count, mass, count, bin);
        while (true) {
            // this CTA's tokens of the bin
            const int turn_ = turn;
            turn ^= 1;
            Candidate *list = s.list[turn_];
            if (threadIdx.x == 0) {
                s.n_list[turn_] = 0;
                s.key_lo[turn_] = 0xffffffffu;
                s.key_hi[turn_] = 0;
            }
            __syncthreads();
            const unsigned lo_ = lo, hi_ = hi;
            each([&](float x, int i) {
                const unsigned key = key_of(x);
                const bool in = cut ? key >= lo_ && key <= hi_ : bin_of(x) == bin;
                if (!in) return;
                const u64 w = weight(x, peak, c, bits);
                if (w == 0) return;
                const unsigned at = atomicAdd(&s.n_list[turn_], 1u);
                if (at < SL_CAND) list[at] = {(u64)key << 32 | (unsigned)~i, w};
                atomicMin(&s.key_lo[turn_], key);
                atomicMax(&s.key_hi[turn_], key);
            });
            sync();
            unsigned n = 0;
            lo = 0xffffffffu;
            hi = 0;
            for (int r = 0; r < C; r++) {
                n += *of(&s.n_list[turn_], r);
                lo = min(lo, *of(&s.key_lo[turn_], r));
                hi = max(hi, *of(&s.key_hi[turn_], r));
            }
            if (n <= SL_CAND) return rank_all(turn_, n, target, by_count, mass, count);
            if (lo == hi) return nth_tie(turn_, lo, target, by_count, mass, count);
            // cut the bin by the bits of its keys
            cut = true;
            shift = max(0, 32 - __clz((hi - lo) / SL_BINS));
            zero_bins();
            __syncthreads();
            const unsigned l = lo, h = hi;
            const int sh = shift;
            each([&](float x, int) {
                const unsigned key = key_of(x);
                if (key < l || key > h) return;
                const u64 w = weight(x, peak, c, bits);
                if (w == 0) return;
                atomicAdd(&s.mass[(h - key) >> sh], w);
                atomicAdd(&s.count[(h - key) >> sh], 1u);
            });
            merge(1);
            find_bin(1, target, by_count, mass, count, bin);
            const unsigned top = h - ((unsigned)bin << sh);
            hi = top;
            lo = top - l > (1u << sh) - 1 ? top - ((1u << sh) - 1) : l;
        }
    }

    __device__ __forceinline__ void zero_bins() {
        for (int b = threadIdx.x; b < SL_BINS; b += SL_THREADS) {
            s.mass[b] = 0;
            s.count[b] = 0;
        }
    }

    // Among the n tokens that the CTAs listed.
    __device__ Crossing rank_all(int turn_, unsigned n, u64 target, bool by_count, u64 mass, unsigned count) {
        unsigned at = 0;
        for (int r = 0; r < C; r++) {
            const unsigned k = *of(&s.n_list[turn_], r);
            const Candidate *from = of(s.list[turn_], r);
            for (unsigned j = threadIdx.x; j < k; j += SL_THREADS) s.all[at + j] = from[j];
            at += k;
        }
        __syncthreads();
        // `sub` neighbouring threads compare one token with all
        int sub = 32;
        while (sub > 1 && (unsigned)(SL_THREADS / sub) < n) sub /= 2;
        const unsigned mine = threadIdx.x / sub, from = threadIdx.x % sub;
        const Candidate own = mine < n ? s.all[mine] : Candidate{0, 0};
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
            s.found = {before, own.w, (int)~(unsigned)own.order};
        __syncthreads();
        const Crossing f = s.found;
        __syncthreads();  // all, found: read
        return f;
    }

    // Among tokens of one logit, more than are ranked directly: by their index.
    __device__ Crossing nth_tie(int turn_, unsigned key, u64 target, bool by_count, u64 mass, unsigned count) {
        const u64 w = weight(of_key(key), peak, c, bits);
        const u64 nth = by_count ? target - count : (target - mass) / w;
        u64 left = nth;
        int owner = 0;
        for (; owner < C - 1; owner++) {
            const unsigned k = *of(&s.n_list[turn_], owner);
            if (left < k) break;
            left -= k;
        }
        if (rank == owner) {
            for (int v0 = 0; v0 < slice; v0 += SL_THREADS) {
                const int v = v0 + threadIdx.x;
                const bool is = v < slice && key_of(to_f32(x_s[v])) == key;
                u64 here;
                const u64 before = block_scan(is, s.scan, &here);
                if (is && before == left) s.tie = i0 + v;
                if (left < here) break;
                left -= here;
            }
        }
        sync();
        const int index = *of(&s.tie, owner);
        return {mass + nth * w, w, index};
    }
};

template <typename T>
__global__ void __launch_bounds__(SL_THREADS, 1) sample_logits_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sl_smem[];
    SampleShared &s = *reinterpret_cast<SampleShared *>(sl_smem);
    T *x_s = reinterpret_cast<T *>(sl_smem + (sizeof(SampleShared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / C, tid = threadIdx.x;
    constexpr int PER = 16 / sizeof(T);
    const T ninf = T(-INFINITY);

    pdl_trigger();
    pdl_wait();
    const T *in = static_cast<const T *>(a.logits) + row * a.stride;
    // slices begin `shift` places early, where a 16-byte line does
    const int shift = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    const int i0 = rank * a.slice - shift;
    Sampler<T> m = {s, x_s, cluster, C, rank, i0, a.slice};
    m.bits = a.bits;
    m.zero_bins();

    // the slice into shared memory; its largest token, and its smallest finite logit
    float top = -INFINITY, low = INFINITY;
    int at = 0x7fffffff;
    for (int v = tid * PER; v < a.slice; v += SL_THREADS * PER) {
        const int i = i0 + v;
        T x[PER];
        if (i >= 0 && i + PER <= a.vocab) {
            *reinterpret_cast<uint4 *>(x) = *reinterpret_cast<const uint4 *>(in + i);
        } else {
#pragma unroll
            for (int e = 0; e < PER; e++) x[e] = i + e >= 0 && i + e < a.vocab ? in[i + e] : ninf;
        }
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const float f = to_f32(x[e]);
            if (f != f) x[e] = ninf;
            if (f > top) {
                top = f;
                at = i + e;
            }
            if (f > -INFINITY) low = fminf(low, f);
        }
        *reinterpret_cast<uint4 *>(x_s + v) = *reinterpret_cast<uint4 *>(x);
    }
    if (tid == 0) {
        s.first = 0;
        s.min_key = 0xffffffffu;
        s.floor_mass = s.before_draft = 0;
    }
    __syncthreads();
    const u64 best = warp_max(top > -INFINITY ? (u64)key_of(top) << 32 | (unsigned)~at : 0);
    const unsigned least = __reduce_min_sync(0xffffffffu, key_of(low));
    if (tid % 32 == 0) {
        atomicMax(&s.first, best);
        atomicMin(&s.min_key, least);
    }
    m.sync();
    u64 first = 0;
    unsigned min_key = 0xffffffffu;
    for (int r = 0; r < C; r++) {
        first = max(first, *m.of(&s.first, r));
        min_key = min(min_key, *m.of(&s.min_key, r));
    }
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    int token = first ? (int)~(unsigned)first : -1;
    float prob = first ? 1.0f : 0.0f;
    if (first && temperature > 0.0f) {
        const float max_x = of_key((unsigned)(first >> 32));
        m.peak = max_x;
        m.c = 1.4426950408889634 / (double)temperature;
        const float range = fminf((float)(46.0 / m.c), max_x - of_key(min_key));
        m.per_bin = range > 0.0f ? SL_BINS / range : 0.0f;
        if (!(m.per_bin < 1e30f)) m.per_bin = 1e30f;
        const int k = a.top_k ? a.top_k[row] : 0, draft = a.draft ? a.draft[row] : -1;
        const float p = a.top_p ? a.top_p[row] : 1.0f, floor = a.min_p ? a.min_p[row] : 0.0f;
        const bool has_floor = floor > 0.0f;
        const double least_t = has_floor ? log2((double)fminf(floor, 1.0f)) : 0.0;
        const float xd = draft >= 0 && draft < a.vocab ? to_f32(in[draft]) : -INFINITY;
        const bool has_draft = xd > -INFINITY;
        // one pass: the histogram, the mass above min-p's limit, the mass before the draft
        u64 above = 0, before = 0;
        m.each([&](float x, int i) {
            const u64 w = weight(x, m.peak, m.c, a.bits);
            if (w == 0) return;
            const int b = m.bin_of(x);
            atomicAdd(&s.mass[b], w);
            atomicAdd(&s.count[b], 1u);
            if (has_floor && (x == max_x || ((double)x - m.peak) * m.c >= least_t)) above += w;
            if (has_draft && (x > xd || (x == xd && i < draft))) before += w;
        });
        if (has_floor) {
            above = warp_sum(above);
            if (tid % 32 == 0) atomicAdd(&s.floor_mass, above);
        }
        if (has_draft) {
            before = warp_sum(before);
            if (tid % 32 == 0) atomicAdd(&s.before_draft, before);
        }
        m.merge(0);
        u64 mass = 0, above_all = 0, before_all = 0;
        unsigned count = 0;
        for (int r = 0; r < C; r++) {
            mass += *m.of(&s.part_mass[0], r);
            count += *m.of(&s.part_count[0], r);
            above_all += *m.of(&s.floor_mass, r);
            before_all += *m.of(&s.before_draft, r);
        }
        if (k > 0 && (unsigned)k < count) {
            const Crossing f = m.find((u64)(k - 1), true);
            mass = f.before + f.w;
        }
        if (p < 1.0f) {  // the shortest beginning with at least p of the mass
            const double want = ceil((double)fmaxf(p, 0.0f) * (double)mass);
            const u64 target = want < 1.0 ? 0 : min((u64)want, mass) - 1;
            const Crossing f = m.find(target, false);
            mass = f.before + f.w;
        }
        if (has_floor) mass = min(mass, above_all);
        const float u = fminf(fmaxf(a.u[row], 0.0f), 0x1.fffffep-1f);  // NaN is 0
        u64 target = min((u64)((double)u * (double)mass), mass - 1);
        const u64 wd = has_draft ? weight(xd, m.peak, m.c, a.bits) : 0;
        u64 w;
        if (wd > 0 && before_all < mass && target < wd) {
            token = draft;
            w = wd;
        } else {
            // the draft's place in the order is empty
            if (wd > 0 && before_all < mass && target - wd < before_all) target -= wd;
            const Crossing f = m.find(target, false);
            token = f.index;
            w = f.w;
        }
        prob = (float)((double)w / (double)mass);
    }
    if (rank == 0 && tid == 0) {
        a.out[row] = token;
        if (a.prob) a.prob[row] = prob;
    }
    m.sync();  // the other CTAs have read this one's shared memory
}

}  // namespace

}  // namespace q3

using namespace q3;

extern "C" {

int q3_sample_logits(int *out, float *prob, const void *logits, int dtype, int rows, int vocab, long long stride, const float *u,
                     const float *temperature, const int *top_k, const float *top_p, const float *min_p, const int *draft,
                     void *stream) {
    if (dtype != 0 && dtype != 1) return Q3_ERR_ARG;
    const int elt = dtype ? 4 : 2;
    if (rows < 0 || vocab <= 0 || stride < vocab || (long long)vocab * elt > (long long)SL_MAX_CLUSTER * SL_SLICE_BYTES - 128 ||
        rows > (1 << 24))
        return Q3_ERR_SHAPE;
    if (rows == 0) return Q3_OK;  // before the pointers: tensors of no elements have none
    if (!out || !logits || !u) return Q3_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(logits) & (elt - 1)) return Q3_ERR_ALIGN;
    const int st = check_device();
    if (st != Q3_OK) return st;
    // CTAs of a row: as few as hold it, more while SMs are left
    auto slice_of = [&](int c) { return ((vocab + 16 / elt - 1 + c - 1) / c + 7) / 8 * 8; };
    int c = 1;
    while (c < SL_MAX_CLUSTER &&
           (slice_of(c) * elt > SL_SLICE_BYTES || ((long long)2 * c * rows <= num_sms() && slice_of(c) > 4 * SL_THREADS)))
        c *= 2;
    const int bits = vocab <= (1 << 18) ? 44 : 42;  // the whole row's mass stays below 2^62
    SampleArgs a = {out, prob, logits, stride, vocab, slice_of(c), bits, u, temperature, top_p, min_p, top_k, draft};
    const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 + (size_t)a.slice * elt;
    auto kernel = dtype == 0 ? sample_logits_kernel<bf16> : sample_logits_kernel<float>;
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(kernel, dim3((unsigned)rows * c), dim3(SL_THREADS), smem, (cudaStream_t)stream, c, a));
    return Q3_OK;
}

}  // extern "C"
