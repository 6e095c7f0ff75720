// What the operators of the paged 8-bit cache share: the description of a cache and of a ragged batch, and where a row belongs.
#pragma once
#include "hp_common.cuh"
#include "kernels.h"

namespace hp {

// Rows of a batch as the kernels see them. Lengths come from device memory, so nothing they hold is trusted: rows stay inside [0, R), a
// sequence's tokens inside its columns of the table, page numbers inside the pool; what does not is left out and told by the status word.
struct PagedSeq { int s, row0, T, len; };   // sequence, its first row, rows, tokens with these rows (s < 0: none)

__device__ __forceinline__ void paged_bad(int* err) { if (err) *err = HP_EINVAL; }
// rows and tokens of sequence s
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s, int* err) {
    const int a = b.row_start[s], e = b.row_start[s + 1], n = b.kv_len[s];
    PagedSeq q; q.s = s;
    q.row0 = min(max(a, 0), b.R); q.T = min(max(e - a, 0), min(b.max_rows, b.R - q.row0)); q.len = min(max(n, 0), b.max_kv);
    if (q.row0 != a || q.T != e - a || q.len != n) paged_bad(err);
    return q;
}
// The sequence of row r, by one warp: the number of sequences that end at or in front of it. Rows behind the last one: s = -1.
__device__ __forceinline__ PagedSeq paged_find(const PagedBatch& b, int r, int lane, int* err) {
    int s = 0;
    for (int s0 = 0; s0 < b.S; s0 += 32) {
        const bool behind = s0 + lane < b.S && b.row_start[s0 + lane + 1] <= r;
        const int n = __popc(__ballot_sync(0xffffffffu, behind));
        s += n;
        if (n < 32) break;
    }
    if (s >= b.S) return PagedSeq{-1, 0, 0, 0};
    PagedSeq q = paged_seq(b, s, err);
    if (r < q.row0 || r >= q.row0 + q.T) q.s = -1;
    return q;
}
// first row of the page of position pos, counted over the pool's rows of head_dim codes for one head: ((page * n_kv + head) << log2 page_size)
__device__ __forceinline__ uint32_t paged_row(const PagedPool& p, int s, int column, int head, int* err) {
    int id = p.table[(size_t)s * p.table_ld + column];
    if ((unsigned)id >= (unsigned)p.n_pages) { paged_bad(err); return 0xffffffffu; }
    return ((uint32_t)id * (uint32_t)p.n_kv + (uint32_t)head) << p.lg_page;
}

}  // namespace hp
