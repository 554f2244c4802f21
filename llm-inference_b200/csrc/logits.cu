// Penalties, biases and grammar masks on a step's logits (q3_logits_process).
//
// A CTA owns a slice of one row's vocabulary. It counts the row's history into shared memory (bit
// 31: the token occurs, low bits: how often it was generated; integer adds, so the order of the
// atomics does not matter), notes for each biased token the largest index of its entries, and
// then makes one pass over its slice.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace q3 {
int check_device();

namespace {

__device__ unsigned g_dev_error;

constexpr int LP_THREADS = 512;
constexpr int LP_SLICE = 8192;  // tokens per CTA
constexpr unsigned LP_SEEN = 1u << 31;

struct LogitsArgs {
    void *out;
    const void *in;
    int vocab;
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

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logits_process_kernel(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) unsigned lp_smem[];
    unsigned *count_s = lp_smem;                             // [LP_SLICE] if there is a history
    int *bias_s = reinterpret_cast<int *>(lp_smem + (a.hist_start ? LP_SLICE : 0));  // [LP_SLICE] if there are biases
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.y, s0 = blockIdx.x * LP_SLICE, n = min(LP_SLICE, a.vocab - s0), tid = threadIdx.x;
    bool hist = a.hist_start != nullptr, biased = a.bias_start != nullptr;
    int h0 = 0, h1 = 0, hs = 0, b0 = 0, b1 = 0;
    if (hist) {
        h0 = a.hist_start[r];
        h1 = a.hist_start[r + 1];
        hs = a.hist_split[r];
        if (h0 < 0 || h1 < h0 || hs < h0 || hs > h1) {
            if (tid == 0) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
            h1 = h0;
        }
        hist = h1 > h0;
    }
    if (biased) {
        b0 = a.bias_start[r];
        b1 = a.bias_start[r + 1];
        if (b0 < 0 || b1 < b0) {
            if (tid == 0) atomicOr(&g_dev_error, DEV_ERR_POS_RANGE);
            b1 = b0;
        }
        biased = b1 > b0;
    }
    for (int i = tid; i < n; i += LP_THREADS) {
        if (hist) count_s[i] = 0;
        if (biased) bias_s[i] = -1;
    }
    __syncthreads();
    for (int i = h0 + tid; i < h1; i += LP_THREADS) {
        const int t = a.hist_ids[i] - s0;
        if (t >= 0 && t < n) {
            if (i < hs) atomicOr(&count_s[t], LP_SEEN);
            else atomicAdd(&count_s[t], 1);
        }
    }
    for (int i = b0 + tid; i < b1; i += LP_THREADS) {
        const int t = a.bias_ids[i] - s0;
        if (t >= 0 && t < n) atomicMax(&bias_s[t], i);
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[r] : 1.0f;
    const float freq = a.frequency ? a.frequency[r] : 0.0f, pres = a.presence ? a.presence[r] : 0.0f;
    const T *in = static_cast<const T *>(a.in) + r * a.stride + s0;
    T *out = static_cast<T *>(a.out) + r * a.out_stride + s0;
    const unsigned *mask = a.mask ? a.mask + r * a.mask_stride : nullptr;
    for (int i = tid; i < n; i += LP_THREADS) {
        float x = to_f32(in[i]);
        const unsigned c = hist ? count_s[i] : 0u;
        if (c != 0) {
            if (a.repetition) x = x > 0.0f ? x / rep : x * rep;
            const unsigned times = c & ~LP_SEEN;
            if (times != 0) x -= freq * (float)times + pres;
        }
        if (biased && bias_s[i] >= 0) x += a.bias[bias_s[i]];
        if (mask && !(mask[(s0 + i) / 32] >> ((s0 + i) % 32) & 1)) x = -INFINITY;
        from_f32(x, &out[i]);
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

extern "C" int q3_logits_process(void *out, const void *logits, int dtype, int rows, int vocab, long long out_stride,
                                 long long stride, const int *hist_start, const int *hist_split, const int *hist_ids,
                                 const float *repetition, const float *frequency, const float *presence,
                                 const int *bias_start, const int *bias_ids, const float *bias, const unsigned *mask,
                                 long long mask_stride, void *stream) {
    if (!out || !logits || (dtype != 0 && dtype != 1)) return Q3_ERR_ARG;
    if (rows < 0 || rows > 65535 || vocab <= 0 || stride < vocab || out_stride < vocab) return Q3_ERR_SHAPE;
    if (out == logits && out_stride != stride) return Q3_ERR_SHAPE;
    if (hist_start && (!hist_split || !hist_ids)) return Q3_ERR_ARG;
    if (bias_start && (!bias_ids || !bias)) return Q3_ERR_ARG;
    if (mask && mask_stride < ((long long)vocab + 31) / 32) return Q3_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(logits)) & (dtype ? 3 : 1)) return Q3_ERR_ALIGN;
    const int st = check_device();
    if (st != Q3_OK) return st;
    if (rows == 0) return Q3_OK;
    LogitsArgs a = {out,       logits,     vocab,    out_stride, stride,   mask_stride, hist_start, hist_split,
                    hist_ids,  repetition, frequency, presence,  bias_start, bias_ids,  bias,       mask};
    if (!repetition && !frequency && !presence) a.hist_start = nullptr;
    const size_t smem = (size_t)LP_SLICE * 4 * ((a.hist_start ? 1 : 0) + (a.bias_start ? 1 : 0));
    const dim3 grid((vocab + LP_SLICE - 1) / LP_SLICE, rows);
    auto kernel = dtype == 0 ? logits_process_kernel<bf16> : logits_process_kernel<float>;
    cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    Q3_TRY_LAUNCH(launch(kernel, grid, dim3(LP_THREADS), smem, (cudaStream_t)stream, 1, a));
    return Q3_OK;
}
