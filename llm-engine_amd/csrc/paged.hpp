// What the operators over a paged KV cache share: the batch's description,
// the lookups of a row's sequence and a position's slot, host-side checks.
#pragma once

#include "internal.hpp"
#include "llm_engine_amd.h"

namespace em {

struct PagedArgs {
    int n_heads, n_kv_heads, head_size, group;
    int page_size, n_pages, max_pages;
    int n_seqs, rows;
    long long page_stride, slot_stride, head_stride;
    const int* row_start;
    const int* lengths;
    const int* page_table;
    long long table_stride;
};

inline PagedArgs paged_args(const em_paged_shape& s, const em_paged_batch& b, std::size_t rows) {
    PagedArgs a{};
    a.n_heads = s.n_heads;
    a.n_kv_heads = s.n_kv_heads;
    a.head_size = s.head_size;
    a.group = s.n_heads / s.n_kv_heads;
    a.page_size = s.page_size;
    a.n_pages = s.n_pages;
    a.max_pages = s.max_pages;
    a.n_seqs = b.n_seqs;
    a.rows = static_cast<int>(rows);
    a.page_stride = static_cast<long long>(s.page_stride);
    a.slot_stride = static_cast<long long>(s.slot_stride);
    a.head_stride = static_cast<long long>(s.head_stride);
    a.row_start = b.row_start;
    a.lengths = b.lengths;
    a.page_table = b.page_table;
    a.table_stride = static_cast<long long>(b.table_stride);
    return a;
}

// "" or why the paged operators cannot run the shape / the batch (paged.hip).
std::string paged_reject(const em_paged_shape& s);
std::string paged_batch_reject(const em_paged_shape& s, const em_paged_batch& b,
                               std::size_t rows);

// Whether rows [r0, r1) are a sequence's: all of them the call's. Others' are
// nobody's, in every operator.
__device__ __forceinline__ bool rows_exist(const PagedArgs& a, int r0, int r1) {
    return r0 >= 0 && r1 <= a.rows && r1 > r0;
}

// The sequence that row r belongs to: the last s < n_seqs with row_start[s]
// <= r, or -1 where there is none or its rows do not exist or end before r
// (starts that fall may hide r's, but never give another). All 64 lanes of
// the wave call it with one r; a round reads 64 starts and keeps the span
// between two, so 64 sequences take one memory latency and 4096 two.
__device__ __forceinline__ int row_sequence(const PagedArgs& a, int r) {
    const int lane = threadIdx.x % kWave;
    int lo = 0, span = a.n_seqs;
    while (true) {
        const int step = (span + kWave - 1) / kWave, at = lane * step;
        const bool le = at < span && a.row_start[lo + at] <= r;
        const int n = __popcll(__ballot(le));
        if (n == 0) return -1;
        lo += (n - 1) * step;
        if (step == 1) break;
        span = min(step, span - (n - 1) * step);
    }
    const int r0 = a.row_start[lo], r1 = a.row_start[lo + 1];
    return rows_exist(a, r0, r1) && r0 <= r && r1 > r ? lo : -1;
}

// The first element of position t's slot for kv head 0, or -1 where the
// sequence's table has no page for it. t >= 0 and below 2^31.
__device__ __forceinline__ long long slot_offset(const PagedArgs& a, int seq, int t) {
    const int col = t / a.page_size;
    if (col >= a.max_pages) return -1;
    const int page = a.page_table[seq * a.table_stride + col];
    if (page < 0 || page >= a.n_pages) return -1;
    return page * a.page_stride + (t - col * a.page_size) * a.slot_stride;
}

}  // namespace em
