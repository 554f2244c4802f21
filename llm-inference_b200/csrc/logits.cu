// Penalties, biases and grammar masks on a step's logits (q3_logits_process, q3_logits_process_bounded).
//
// A CTA owns a slice of one row's vocabulary, eight tokens a thread, whose logits it asks for first. Meanwhile
// it counts the row's history into shared memory (bit 31: the token occurs, low bits: how often it was
// generated; integer adds, so the order of the atomics does not matter) and notes for each biased token the
// largest index of its entries; then one pass over the slice.
//
// Bound by latency: one row by the chain lengths -> ids -> logits, a batch by that chain once for each of the two or
// three CTAs that an SM runs after one another. Each slice reads the row's whole history, from L2 after the
// first, so slices are as large as still leaves two per SM. 32 rows of 151936 bf16 with masks and 2000 ids of history
// each take 13.5 us in a graph (9.0 without the histories: 2.2 TB/s), 100 rows of 32003 floats with 8000 ids 18.5 (8.4).
// Clusters of 8 slices that share the scan and count in one another's shared memory took 22 and 49 us; they
// gain only for a single row of 16000 ids (13.2 -> 6.9).
#include <math.h>

#include <algorithm>
#include <limits>

#include "common.cuh"

namespace q3 {
int check_device();

namespace {

__device__ unsigned g_dev_error;

constexpr int LP_EACH = 8;  // tokens per thread
constexpr unsigned LP_SEEN = 1u << 31;

struct LogitsArgs {
    void *out;
    const void *in;
    int vocab, vec, n_hist, n_bias;  // n_: entries of hist_ids, and of bias_ids and bias
    long long out_stride, stride, mask_stride;
    const int *hist_start, *hist_split, *hist_ids;
    const float *repetition, *frequency, *presence;
    const int *bias_start, *bias_ids;
    const float *bias;
    const unsigned *mask;
};

__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void from_f32(float f, bf16 *o) { *o = __float2bfloat16(f); }
__device__ __forceinline__ void from_f32(float f, float *o) { *o = f; }

__device__ __forceinline__ void unpack(const uint4 *u, float *x, bf16) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __bfloat1622float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const uint4 *u, float *x, float) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float(reinterpret_cast<const uint32_t *>(u)[i]);
}
__device__ __forceinline__ void pack(const float *x, uint4 *u, bf16) {
    __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(u);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
}
__device__ __forceinline__ void pack(const float *x, uint4 *u, float) {
#pragma unroll
    for (int i = 0; i < 8; i++) reinterpret_cast<uint32_t *>(u)[i] = __float_as_uint(x[i]);
}

// f(index, id) for ids[i0 .. i1) by the CTA, four at a time where they are aligned.
template <typename F>
__device__ __forceinline__ void each_id(const int *ids, int i0, int i1, F f) {
    const int lead = min(i1 - i0, (int)((16 - (reinterpret_cast<uintptr_t>(ids + i0) & 15)) & 15) / 4);
    const int quads = (i1 - i0 - lead) / 4, tail = i0 + lead + 4 * quads;
    if ((int)threadIdx.x < lead) f(i0 + threadIdx.x, ids[i0 + threadIdx.x]);
    // the next load is asked for before this one's ids are looked at (100 rows of 8000 ids: 19.5 -> 18.3 us); with three
    // or four in flight, or the first before the caller's barrier, their registers cost an SM its third CTA (20.5 us)
    const int4 *src = reinterpret_cast<const int4 *>(ids + i0 + lead);
    int4 next = threadIdx.x < quads ? __ldg(src + threadIdx.x) : make_int4(0, 0, 0, 0);
#pragma unroll 1
    for (int q = threadIdx.x; q < quads; q += blockDim.x) {
        const int i = i0 + lead + 4 * q;
        const int4 v = next;
        if (q + (int)blockDim.x < quads) next = __ldg(src + q + blockDim.x);
        f(i, v.x);
        f(i + 1, v.y);
        f(i + 2, v.z);
        f(i + 3, v.w);
    }
    if (tail + (int)threadIdx.x < i1) f(tail + threadIdx.x, ids[tail + threadIdx.x]);
}

// A slice starts `shift` tokens early, so that a row whose first logit is not 16-byte aligned is still read in whole
// vectors; a.vec says that input and output rows are aligned alike.
template <typename T>
__global__ void __launch_bounds__(512) logits_process_kernel(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) unsigned lp_smem[];
    constexpr int VECS = LP_EACH * sizeof(T) / 16;
    const int slice = LP_EACH * blockDim.x, r = blockIdx.y, tid = threadIdx.x;
    unsigned *count_s = lp_smem;                                                  // [slice] if there is a history
    int *bias_s = reinterpret_cast<int *>(lp_smem + (a.hist_start ? slice : 0));  // [slice] if there are biases
#pragma unroll
    for (int v = 0; v < LP_EACH / 4; v++) {  // this thread's own tokens
        if (a.hist_start) reinterpret_cast<uint4 *>(count_s)[tid * (LP_EACH / 4) + v] = make_uint4(0, 0, 0, 0);
        if (a.bias_start) reinterpret_cast<int4 *>(bias_s)[tid * (LP_EACH / 4) + v] = make_int4(-1, -1, -1, -1);
    }
    pdl_trigger();
    pdl_wait();
    const T *in = static_cast<const T *>(a.in) + r * a.stride;
    T *out = static_cast<T *>(a.out) + r * a.out_stride;
    const int shift = a.vec ? (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T)) : 0;
    const int s0 = (int)(blockIdx.x * slice) - shift, i0 = s0 + LP_EACH * tid;
    const bool whole = a.vec && i0 >= 0 && i0 + LP_EACH <= a.vocab;
    uint4 raw[VECS];
    if (whole) {
#pragma unroll
        for (int v = 0; v < VECS; v++) raw[v] = reinterpret_cast<const uint4 *>(in + i0)[v];
    }
    uint32_t allowed = 0xff;  // by token, bit 0 first
    if (a.mask && i0 < a.vocab) {
        const unsigned *mask = a.mask + r * a.mask_stride;
        const int from = max(i0, 0), word = from / 32, lastw = (a.vocab - 1) / 32;
        const unsigned bits = __funnelshift_r(mask[word], mask[min(word + 1, lastw)], from % 32);
        allowed = bits << (from - i0);
    }
    int h0 = 0, h1 = 0, hs = 0, b0 = 0, b1 = 0;
    if (a.hist_start) {
        h0 = a.hist_start[r];
        h1 = a.hist_start[r + 1];
        hs = a.hist_split[r];
        if (h0 < 0 || h1 < h0 || hs < h0 || hs > h1 || h1 > a.n_hist) {
            if (tid == 0) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
            h1 = h0;
        }
    }
    if (a.bias_start) {
        b0 = a.bias_start[r];
        b1 = a.bias_start[r + 1];
        if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
            if (tid == 0) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
            b1 = b0;
        }
    }
    const bool hist = h1 > h0, biased = b1 > b0;
    if (hist || biased) {
        __syncthreads();
        const int first = max(s0, 0), n = max(0, min(s0 + slice, a.vocab) - first);  // this slice's ids
        if (hist)
            each_id(a.hist_ids, h0, h1, [&](int i, int id) {
                if ((unsigned)(id - first) < (unsigned)n) {
                    if (i < hs) atomicOr(&count_s[id - s0], LP_SEEN);
                    else atomicAdd(&count_s[id - s0], 1u);
                }
            });
        if (biased)
            each_id(a.bias_ids, b0, b1, [&](int i, int id) {
                if ((unsigned)(id - first) < (unsigned)n) atomicMax(&bias_s[id - s0], i);
            });
        __syncthreads();
    }
    float x[LP_EACH];
    if (whole) {
        unpack(raw, x, T());
    } else {
#pragma unroll
        for (int e = 0; e < LP_EACH; e++) x[e] = i0 + e >= 0 && i0 + e < a.vocab ? to_f32(in[i0 + e]) : 0.0f;
    }
    if (hist) {  // most threads own no token of the history
        const uint4 *own = reinterpret_cast<const uint4 *>(count_s) + tid * (LP_EACH / 4);
        const uint4 ca = own[0], cb = own[1];
        if ((ca.x | ca.y | ca.z | ca.w | cb.x | cb.y | cb.z | cb.w) != 0) {
            const float rep = a.repetition ? a.repetition[r] : 1.0f, freq = a.frequency ? a.frequency[r] : 0.0f,
                        pres = a.presence ? a.presence[r] : 0.0f;
            const unsigned c[LP_EACH] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
#pragma unroll
            for (int e = 0; e < LP_EACH; e++) {
                if (c[e] == 0) continue;
                if (a.repetition) x[e] = x[e] > 0.0f ? x[e] / rep : x[e] * rep;
                const unsigned times = c[e] & ~LP_SEEN;
                if (times != 0) x[e] -= freq * (float)times + pres;
            }
        }
    }
    if (biased) {
        const int4 *own = reinterpret_cast<const int4 *>(bias_s) + tid * (LP_EACH / 4);
        const int4 ba = own[0], bb = own[1];
        if ((ba.x & ba.y & ba.z & ba.w & bb.x & bb.y & bb.z & bb.w) != -1) {
            const int i[LP_EACH] = {ba.x, ba.y, ba.z, ba.w, bb.x, bb.y, bb.z, bb.w};
#pragma unroll
            for (int e = 0; e < LP_EACH; e++)
                if (i[e] >= 0) x[e] += a.bias[i[e]];
        }
    }
#pragma unroll
    for (int e = 0; e < LP_EACH; e++)
        if (!(allowed >> e & 1)) x[e] = -INFINITY;
    if (whole) {
        pack(x, raw, T());
#pragma unroll
        for (int v = 0; v < VECS; v++) reinterpret_cast<uint4 *>(out + i0)[v] = raw[v];
    } else {
#pragma unroll
        for (int e = 0; e < LP_EACH; e++)
            if (i0 + e >= 0 && i0 + e < a.vocab) from_f32(x[e], &out[i0 + e]);
    }
}

}  // namespace

unsigned take_error_logits() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v)) != cudaSuccess) return 0;
    if (v) cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero));
    return v;
}

}  // namespace q3

using namespace q3;

extern "C" {

int q3_logits_process_bounded(void *out, const void *logits, int dtype, int rows, int vocab, long long out_stride,
                              long long stride, const int *hist_start, const int *hist_split, const int *hist_ids,
                              long long n_hist, const float *repetition, const float *frequency, const float *presence,
                              const int *bias_start, const int *bias_ids, const float *bias, long long n_bias,
                              const unsigned *mask, long long mask_stride, void *stream) {
    if (dtype != 0 && dtype != 1) return Q3_ERR_ARG;
    if (rows < 0 || rows > 65535 || vocab <= 0 || stride < vocab || out_stride < vocab) return Q3_ERR_SHAPE;
    if (rows == 0) return Q3_OK;  // before the pointers: tensors of no elements have none
    if (!out || !logits) return Q3_ERR_ARG;
    if (out == logits && out_stride != stride) return Q3_ERR_SHAPE;
    if (hist_start && (!hist_split || !hist_ids)) return Q3_ERR_ARG;
    if (bias_start && (!bias_ids || !bias)) return Q3_ERR_ARG;
    if ((hist_start && n_hist < 0) || (bias_start && n_bias < 0)) return Q3_ERR_SHAPE;
    if (mask && mask_stride < ((long long)vocab + 31) / 32) return Q3_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(logits)) & (dtype ? 3 : 1)) return Q3_ERR_ALIGN;
    const int st = check_device();
    if (st != Q3_OK) return st;
    const int elt = dtype ? 4 : 2;
    // the same place in a 16-byte line for each row's input and output, and whole lines between places of a row
    const bool vec = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(logits)) & 15) == 0 &&
                     (out_stride - stride) * elt % 16 == 0;
    const long long most = std::numeric_limits<int>::max();  // what a start can say
    LogitsArgs a = {out, logits, vocab, vec, (int)std::min(n_hist, most), (int)std::min(n_bias, most), out_stride, stride,
                    mask_stride, hist_start, hist_split, hist_ids, repetition, frequency, presence, bias_start, bias_ids, bias, mask};
    if (!repetition && !frequency && !presence) a.hist_start = nullptr;
    // two slices an SM at least; 128 threads are the smallest that make whole warps busy
    int threads = 512;
    auto slices = [&](int t) { return (vocab + 7 + LP_EACH * t - 1) / (LP_EACH * t); };
    while (threads > 128 && (long long)slices(threads) * rows < 2 * num_sms()) threads /= 2;
    const size_t smem = (size_t)LP_EACH * threads * 4 * ((a.hist_start ? 1 : 0) + (a.bias_start ? 1 : 0));
    const dim3 grid(slices(threads), rows);
    auto kernel = dtype == 0 ? logits_process_kernel<bf16> : logits_process_kernel<float>;
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(kernel, grid, dim3(threads), smem, (cudaStream_t)stream, 1, a));
    return Q3_OK;
}

int q3_logits_process(void *out, const void *logits, int dtype, int rows, int vocab, long long out_stride, long long stride,
                      const int *hist_start, const int *hist_split, const int *hist_ids, const float *repetition,
                      const float *frequency, const float *presence, const int *bias_start, const int *bias_ids,
                      const float *bias, const unsigned *mask, long long mask_stride, void *stream) {
    const long long any = std::numeric_limits<int>::max();
    return q3_logits_process_bounded(out, logits, dtype, rows, vocab, out_stride, stride, hist_start, hist_split, hist_ids, any,
                                     repetition, frequency, presence, bias_start, bias_ids, bias, any, mask, mask_stride, stream);
}

}  // extern "C"
