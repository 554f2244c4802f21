// Layout of a paged step's plan (paged.cu writes it, the append and attention kernels read it).
#pragma once

#include "common.cuh"

namespace q3 {

constexpr int PAGED_MAX_SEQS = 4096;
constexpr int PAGED_MAX_HEAD_DIM = 128;

// A token's sequence and position. pos -1: padding (its rows are written as zeros); PAGED_OUTSIDE:
// a row of the batch outside every sequence (never written).
constexpr int PAGED_OUTSIDE = -2;

struct PagedSeq {
    int q0, q_len, kv_len, pad;
};

// Byte offsets of the plan's parts; the same arithmetic on host and device.
struct PagedPlanLayout {
    size_t seqs;   // PagedSeq [n_seqs]
    size_t table;  // int [n_seqs][max_pages]: checked page ids, -1 past a sequence's last page
    size_t toks;   // int4 [n_tokens]: sequence, position, page, slot
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
    l.seqs = take((size_t)s.n_seqs * sizeof(PagedSeq));
    l.table = take((size_t)s.n_seqs * s.max_pages * 4);
    l.toks = take((size_t)s.n_tokens * 16);
    l.bytes = off;
    return l;
}

// Q3_OK, or why the shape is not supported.
int paged_shape_check(const q3_paged_shape *s);

}  // namespace q3
