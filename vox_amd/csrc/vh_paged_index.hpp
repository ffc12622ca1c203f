// vh_paged_index.hpp — where the rows, keys and pages of a ragged batch lie: the index arithmetic of the paged-cache
// kernels, in plain C++ so that the host and a CPU test run the same functions as the device.
//
// A batch: row_start [seqs + 1] (rows row_start[s] .. row_start[s + 1] - 1 belong to sequence s), len [seqs] (keys of s,
// its rows of this call among them), table [seqs][page_ld]. Row i of n stands at position len - n + i. Everything here is
// read from device memory that a caller filled, so every value is brought into range before it addresses anything.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define VH_HD __host__ __device__ __forceinline__
#else
#define VH_HD inline
#endif

namespace vh {

struct PagedKv {
    void *k, *v;
    int64_t page_stride, head_stride, pos_stride;  // elements
    int32_t pages, shift, kv_heads, hd;            // a page holds 1 << shift positions
};
struct PagedBatch {
    const int32_t *row_start, *len, *table;
    int64_t page_ld;
    int32_t seqs, rows;
};
// Groups of neighbouring sequences whose first len keys are the pages of the group's first sequence.
struct PagedGroups {
    const int32_t *seq_start, *len;
    int32_t groups;
};

VH_HD int32_t clamp_i32(int64_t v, int64_t lo, int64_t hi) { return int32_t(v < lo ? lo : v > hi ? hi : v); }

struct SeqRows {
    int32_t first, n, len;
    bool ok;  // the batch's own values were in range
};
VH_HD SeqRows seq_rows(const PagedBatch &b, int32_t shift, int32_t s) {
    const int32_t r0 = b.row_start[s], r1 = b.row_start[s + 1], l = b.len[s];
    SeqRows r;
    r.first = clamp_i32(r0, 0, b.rows);
    r.n = clamp_i32(r1, r.first, b.rows) - r.first;
    r.len = clamp_i32(l, 0, b.page_ld << shift);
    r.ok = r.first == r0 && r.first + r.n == r1 && r.len == l;
    return r;
}

// Keys [begin, end) that the row at position pos sees: causal, the first `prefix` keys by every row, at most `window` back
// (0: all). A row before position 0 sees none.
struct Span {
    int32_t begin, end;
};
VH_HD Span visible(int32_t pos, int32_t len, int32_t prefix, int32_t window) {
    if (pos < 0) return Span{0, 0};
    int32_t end = prefix > pos + 1 ? prefix : pos + 1;
    end = end < len ? end : len;
    const int32_t begin = window > 0 && pos >= window ? pos - window + 1 : 0;
    return Span{begin < end ? begin : end, end};
}

// The page of position pos by its table entry, or -1 when the entry names no page of the pool.
VH_HD int32_t page_of(const PagedKv &c, const int32_t *table, int32_t pos) {
    const int32_t p = table[pos >> c.shift];
    return uint32_t(p) < uint32_t(c.pages) ? p : -1;
}
VH_HD int64_t key_offset(const PagedKv &c, int32_t page, int32_t head, int32_t pos) {
    return int64_t(page) * c.page_stride + int64_t(head) * c.head_stride + int64_t(pos & ((1 << c.shift) - 1)) * c.pos_stride;
}

// The group of sequence s, or -1. A group's bounds are clamped to the batch's sequences.
VH_HD int32_t group_of(const PagedGroups &p, int32_t s) {
    for (int32_t g = 0; g < p.groups; ++g)
        if (s >= p.seq_start[g] && s < p.seq_start[g + 1]) return g;
    return -1;
}

}  // namespace vh
