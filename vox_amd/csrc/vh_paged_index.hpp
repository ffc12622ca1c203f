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

// ------------------------------------------------------------------ the attention's work
// A segment is what meets one run of keys: the rows of a group and its shared keys, or the rows of a sequence and its own
// keys behind the shared ones. Its query rows are (row, head of the kv head's `group` heads), the head fastest; a tile is
// `tile` of them. The keys go in runs (split_of), one per split; a (query row, segment) pair leaves one part per run.
struct Segment {
    int32_t row0, rows;  // rows of the batch
    int32_t seq0, seq1;  // their sequences
    int32_t key0, key1;  // keys, from the page table of seq0
    bool ok;
};
VH_HD Segment group_segment(const PagedBatch &b, const PagedGroups &p, int32_t shift, int32_t g) {
    Segment s;
    s.seq0 = clamp_i32(p.seq_start[g], 0, b.seqs);
    s.seq1 = clamp_i32(p.seq_start[g + 1], s.seq0, b.seqs);
    s.row0 = clamp_i32(b.row_start[s.seq0], 0, b.rows);
    s.rows = clamp_i32(b.row_start[s.seq1], s.row0, b.rows) - s.row0;
    s.key0 = 0;
    s.key1 = clamp_i32(p.len[g], 0, b.page_ld << shift);
    s.ok = s.seq0 == p.seq_start[g] && s.seq1 == p.seq_start[g + 1] && s.key1 == p.len[g];
    return s;
}
// shared: the keys of the sequence's group (0: none).
VH_HD Segment seq_segment(const PagedBatch &b, int32_t shift, int32_t seq, int32_t shared) {
    const SeqRows r = seq_rows(b, shift, seq);
    Segment s;
    s.seq0 = seq;
    s.seq1 = seq + 1;
    s.row0 = r.first;
    s.rows = r.n;
    s.key0 = clamp_i32(shared, 0, r.len);
    s.key1 = r.len;
    s.ok = r.ok;
    return s;
}
// Keys [key0, key1) in at most `splits` runs of a multiple of kKeyTile keys, of at least `least` (a multiple too), whose borders
// but the first and last are multiples of kKeyTile.
constexpr int32_t kKeyTile = 64;
struct Runs {
    int32_t first, step, count;  // run i: keys [max(key0, first + i step), min(key1, first + (i + 1) step))
};
VH_HD Runs runs_of(int32_t key0, int32_t key1, int32_t splits, int32_t least) {
    Runs r;
    r.first = key0 & ~(kKeyTile - 1);
    const int64_t keys = int64_t(key1) - r.first;
    const int64_t even = ((keys + splits - 1) / splits + kKeyTile - 1) & ~int64_t(kKeyTile - 1);
    r.step = int32_t(even > least ? even : least);
    r.count = key1 > key0 ? int32_t((keys + r.step - 1) / r.step) : 0;
    return r;
}
VH_HD Span run_at(const Runs &r, int32_t key0, int32_t key1, int32_t i) {
    const int64_t a = r.first + int64_t(i) * r.step, e = a + r.step;
    return Span{a > key0 ? int32_t(a) : key0, e < key1 ? int32_t(e) : key1};
}
VH_HD int32_t tiles_of(int32_t rows, int32_t group, int32_t tile) { return int32_t((int64_t(rows) * group + tile - 1) / tile); }

}  // namespace vh
