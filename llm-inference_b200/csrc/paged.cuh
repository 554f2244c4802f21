// Layout of a paged step's plan (paged.cu writes it, the append and attention kernels read it).
#pragma once

#include <algorithm>

#include "common.cuh"

namespace q3 {

constexpr int PAGED_MAX_SEQS = 4096;
constexpr int PAGED_MAX_HEAD_DIM = 128;

// A token's place is its position + 1, or one of these: a row of the batch outside every sequence (never written), or
// padding (its rows are written as zeros). A plan of zeroed memory has neither tokens nor pieces.
constexpr int PAGED_OUTSIDE = 0, PAGED_PADDING = -1;

struct PagedSeq {
    int q0, q_len, kv_len;
};

// Attention work. An item is what one CTA could do alone: the query rows of a (sequence, kv head) that
// attend together. Few rows (q_len * n_heads / n_kv_heads <= paged_small_rows) are one item, fed to warp-level
// matrix instructions; more are cut into items of two 128-row tensor-core tiles. Each kind has its kernel.
// The plan lays a kind's costs end to end and gives each CTA an equal stretch, so an item may be cut along its
// positions into pieces of neighbouring CTAs, which leave partial results in the scratch.
constexpr int BIG_TILE = 128;       // rows of a tensor-core tile, and positions of one of its steps
constexpr int PAGED_MAX_CTAS = 160; // persistent CTAs, one per SM

struct alignas(16) PagedPiece {
    int seq, kvh, tok0, n_tok;   // query rows: tokens tok0 .. tok0 + n_tok of the batch
    int kv0, kv1, kv_end, pos0;  // this piece's positions, the item's end, the first token's position (< 0: padding)
    int part, first, n_parts;    // scratch slot (-1: the item is whole), the item's first CTA, its pieces
};

// Where a piece of CTA c leaves its partial result: an item's first piece is its CTA's last (slot 2c + 1), the
// later ones are the first of theirs (slot 2c).
__host__ __device__ __forceinline__ int part_slot(int first, int i) { return i == 0 ? 2 * first + 1 : 2 * (first + i); }

// Rows of the kernel for few rows: eight for each 8-column tile of its products. Where every sequence fits into a
// few tiles (draft tokens being verified) the step needs no other kernel; where some do not, it is the one for single
// tokens, and all longer sequences go to the kernel for many rows. 32 sequences at 4096, 8 kv heads of 128: 16 rows take
// 92 us here and 128 there (at 1.7 GHz), 24 rows 152 and 128 to 133 (their accumulators spill); 4 kv heads of 64: 16 rows 31
// and 52, 24 rows 37 and 52, 40 rows 64 and 52.
inline int paged_small_rows(const q3_paged_shape &s) {
    const long long most = (long long)s.max_q_len * (s.n_heads / s.n_kv_heads);
    if (most > (s.head_dim <= 64 ? 24 : 16) || most <= 8) return 8;
    return most <= 16 ? 16 : 24;
}
// One query head group alone may be too many; a batch that may bring no tokens at all counts as bringing one.
inline bool paged_has_big(const q3_paged_shape &s) {
    return (long long)std::max(s.max_q_len, 1) * (s.n_heads / s.n_kv_heads) > paged_small_rows(s);
}

// Byte offsets of the plan's parts; the same arithmetic on host and device.
struct PagedPlanLayout {
    size_t table;     // int [n_seqs][max_pages]: checked page ids, -1 past a sequence's last page
    size_t toks;      // int4 [n_tokens]: sequence, place, page, slot
    size_t ctas;      // int2 [2][PAGED_MAX_CTAS], small items' CTAs and big ones': first piece, pieces (-1: zero every row)
    size_t counters;  // int [PAGED_MAX_CTAS]: pieces done of the small item that starts in the CTA; zero at rest
    size_t ready;     // int [PAGED_MAX_CTAS]: the CTA of the kernel for many rows has waited for what came before; zero at rest
    size_t splits;    // PagedPiece [PAGED_MAX_CTAS]: the cut big item that starts in the CTA (n_parts 0: none)
    size_t pieces;    // PagedPiece []
    size_t bytes;
};

inline PagedPlanLayout paged_plan_layout(const q3_paged_shape &s) {
    PagedPlanLayout l = {};
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t o = off;
        off += (bytes + 255) / 256 * 256;
        return o;
    };
    const int rep = s.n_heads / s.n_kv_heads, span = paged_has_big(s) ? 2 * (BIG_TILE / rep) : paged_small_rows(s) / rep;
    const size_t items = (size_t)s.n_kv_heads * ((size_t)s.n_seqs + (size_t)s.n_tokens / span);
    l.table = take((size_t)s.n_seqs * s.max_pages * 4);
    l.toks = take((size_t)s.n_tokens * 16);
    l.ctas = take(2 * PAGED_MAX_CTAS * sizeof(int2));
    l.counters = take(PAGED_MAX_CTAS * sizeof(int));
    l.ready = take(PAGED_MAX_CTAS * sizeof(int));
    l.splits = take(PAGED_MAX_CTAS * sizeof(PagedPiece));
    l.pieces = take((items + 2 * PAGED_MAX_CTAS) * sizeof(PagedPiece));
    l.bytes = off;
    return l;
}

// Scratch of the attention: partial outputs, unnormalized fp32 rows with their maximum (in units of log2) and
// sum, two slots per CTA.
struct PagedScratchLayout {
    size_t small_o, small_ml, big_o, big_ml, bytes;
};

// A step of a small item is one ring stage of K and V; pieces are cut at multiples of it.
constexpr int SMALL_STAGE = 16384;  // bytes
inline int paged_small_step(const q3_paged_shape &s) { return SMALL_STAGE / (4 * (s.head_dim <= 64 ? 64 : 128)); }

inline PagedScratchLayout paged_scratch_layout(const q3_paged_shape &s) {
    PagedScratchLayout l = {};
    const size_t dp = s.head_dim <= 64 ? 64 : 128, slots = 2 * PAGED_MAX_CTAS;
    const size_t big = paged_has_big(s) ? 2 * BIG_TILE : 0;
    l.small_o = 0;
    l.small_ml = l.small_o + slots * paged_small_rows(s) * dp * 4;
    l.big_o = l.small_ml + slots * paged_small_rows(s) * 8;
    l.big_ml = l.big_o + slots * big * dp * 4;
    l.bytes = l.big_ml + slots * big * 8;
    return l;
}

inline int paged_ctas() { return num_sms() < PAGED_MAX_CTAS ? num_sms() : PAGED_MAX_CTAS; }

// two floats as one operand of the packed fp32 instructions
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}

// Q3_OK, or why the shape is not supported.
int paged_shape_check(const q3_paged_shape *s);

// Attention over the pages (paged_attn.cu).
struct PagedAttnCall {
    bf16 *out;
    const bf16 *q;
    long long out_stride, q_stride;
    q3_paged_cache cache;
    float scale;
    q3_paged_shape shape;
    char *plan, *scratch;
};
int paged_attention(const PagedAttnCall &c, cudaStream_t s);

}  // namespace q3
