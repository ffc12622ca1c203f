// paged_index_check.cpp — the index arithmetic of the paged-cache kernels (vh_paged_index.hpp) on the host: values that a
// caller got wrong never address anything outside its buffers, and the visible keys are those of the definition.
// Exit status 0 = every check passed.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "vh_paged_index.hpp"

using namespace vh;

static int fails = 0;
#define CHECK(x)                                               \
    do {                                                       \
        if (!(x)) {                                            \
            std::printf("FAIL line %d: %s\n", __LINE__, #x);   \
            ++fails;                                           \
        }                                                      \
    } while (0)

static uint32_t state = 1;
static int rnd(int n) {
    state = state * 1664525u + 1013904223u;
    return int((state >> 8) % uint32_t(n));
}

static void rows_stay_inside() {
    const int32_t wild[] = {INT32_MIN, -7, -1, 0, 1, 5, 6, 7, 100, 112, 113, 1 << 20, INT32_MAX};
    for (int32_t r0 : wild)
        for (int32_t r1 : wild)
            for (int32_t l : wild) {
                const int32_t row_start[2] = {r0, r1}, len[1] = {l};
                const PagedBatch b{row_start, len, nullptr, 7, 1, 6};
                const SeqRows s = seq_rows(b, 4, 0);
                CHECK(s.first >= 0 && s.n >= 0 && s.first + s.n <= 6 && s.len >= 0 && s.len <= 112);
                CHECK(s.ok == (r0 >= 0 && r0 <= r1 && r1 <= 6 && l >= 0 && l <= 112));
                if (s.ok) CHECK(s.first == r0 && s.n == r1 - r0 && s.len == l);
            }
}

static void pages_stay_inside() {
    PagedKv c{};
    c.pages = 10; c.shift = 4; c.page_stride = (int64_t(1) << 33) + 8; c.head_stride = 1024; c.pos_stride = 64; c.kv_heads = 2; c.hd = 64;
    const int32_t table[] = {0, 9, 10, -1, INT32_MIN, INT32_MAX, 3};
    const int32_t want[] = {0, 9, -1, -1, -1, -1, 3};
    for (int p = 0; p < 7 * 16; ++p) CHECK(page_of(c, table, p) == want[p >> 4]);
    CHECK(key_offset(c, 9, 1, 35) == 9 * c.page_stride + 1024 + 3 * 64);  // past 32 bits
}

static void spans() {
    for (int i = 0; i < 20000; ++i) {
        const int len = rnd(40), pos = rnd(45) - 5, prefix = rnd(3) ? 0 : rnd(60), window = rnd(2) ? 0 : rnd(30);
        const Span s = visible(pos, len, prefix, window);
        CHECK(s.begin >= 0 && s.begin <= s.end && s.end <= len);
        for (int j = -2; j < 64; ++j) {
            const bool want = pos >= 0 && j >= 0 && j < len && (j <= pos || j < prefix) && !(window && j <= pos - window);
            CHECK((j >= s.begin && j < s.end) == want);
        }
    }
    const Span far = visible((1 << 30) - 1, 1 << 30, 0, 0);
    CHECK(far.begin == 0 && far.end == 1 << 30);
}

static int group_of(const PagedGroups &p, int s) {
    for (int g = 0; g < p.groups; ++g)
        if (s >= p.seq_start[g] && s < p.seq_start[g + 1]) return g;
    return -1;
}

// Every key of a row belongs to exactly one run of its group or of its sequence, runs start and end on tile borders inside,
// and the tiles cover every query row once.
static void work() {
    for (int it = 0; it < 3000; ++it) {
        const int shift = 3 + rnd(4), seqs = 1 + rnd(12), group = 1 + rnd(9);
        std::vector<int32_t> start(1, 0), len, gs, gl;
        int maxlen = 1;
        for (int s = 0; s < seqs; ++s) {
            const int n = rnd(4) ? rnd(30) : 0;
            start.push_back(start.back() + n);
            len.push_back(rnd(5) ? n + rnd(900) : rnd(3));
            maxlen = len.back() > maxlen ? len.back() : maxlen;
        }
        for (int s = rnd(2); s < seqs; s += 1 + rnd(5)) {
            gs.push_back(s);
            gl.push_back(rnd(4) ? rnd(maxlen) : 0);
        }
        gs.push_back(seqs);
        const PagedBatch b{start.data(), len.data(), nullptr, (maxlen >> shift) + 1, seqs, start.back() + rnd(3)};
        const PagedGroups p{gs.data(), gl.data(), rnd(3) ? int(gl.size()) : 0};
        const int gsplits = 1 + rnd(32), ssplits = 1 + rnd(32), gleast = kKeyTile * (1 + rnd(5)), sleast = kKeyTile * (1 + rnd(5));
        std::vector<int> group_rows(size_t(start.back()), 0);
        for (int g = 0; g < p.groups; ++g) {
            const Segment sg = group_segment(b, p, shift, g);
            CHECK(sg.ok && sg.row0 >= 0 && sg.row0 + sg.rows <= b.rows && sg.key0 == 0 && sg.key1 == gl[size_t(g)]);
            for (int i = 0; i < sg.rows; ++i) ++group_rows[size_t(sg.row0 + i)];
        }
        for (int s = 0; s < seqs; ++s) {
            const int g = group_of(p, s);
            const Segment sg = seq_segment(b, shift, s, g >= 0 ? gl[size_t(g)] : 0);
            CHECK(sg.ok && sg.row0 == start[size_t(s)] && sg.rows == start[size_t(s) + 1] - sg.row0 && sg.key1 == len[size_t(s)]);
            for (int i = 0; i < sg.rows; ++i) CHECK(group_rows[size_t(sg.row0 + i)] == (g >= 0));
            std::vector<int> seen(size_t(len[size_t(s)]), 0);
            auto add = [&](int k0, int k1, int splits, int least) {
                const Runs r = runs_of(k0, k1, splits, least);
                CHECK(r.count >= 0 && r.count <= splits && (r.count > 0) == (k1 > k0));
                for (int i = 0; i < r.count; ++i) {
                    const Span e = run_at(r, k0, k1, i);
                    CHECK(e.begin < e.end && (i == 0 ? e.begin == k0 : e.begin % kKeyTile == 0) && (i == r.count - 1 ? e.end == k1 : e.end % kKeyTile == 0));
                    for (int k = e.begin; k < e.end; ++k)
                        if (k < len[size_t(s)]) ++seen[size_t(k)];  // a group may share more than a short sequence has
                }
            };
            if (g >= 0) add(0, gl[size_t(g)], gsplits, gleast);
            add(sg.key0, sg.key1, ssplits, sleast);
            for (int n : seen) CHECK(n == 1);
            for (int tile : {16, 32, 128}) {
                const int t = tiles_of(sg.rows, group, tile);
                CHECK(t * tile >= sg.rows * group && (t - 1) * tile < sg.rows * group);
            }
        }
    }
    // near the limits nothing overflows
    const Runs r = runs_of((1 << 30) - 5, 1 << 30, 32, 256), all = runs_of(0, 1 << 30, 1, 256);
    CHECK(r.count == 1 && run_at(r, (1 << 30) - 5, 1 << 30, 0).begin == (1 << 30) - 5);
    CHECK(all.count == 1 && run_at(all, 0, 1 << 30, 0).end == 1 << 30);
    // wild group bounds stay inside the batch
    const int32_t wild[] = {INT32_MIN, -1, 0, 2, 3, 4, INT32_MAX};
    const int32_t start[] = {0, 5, 6, 9}, len[] = {5, 1, 40};
    const PagedBatch b{start, len, nullptr, 3, 3, 9};
    for (int32_t a : wild)
        for (int32_t c : wild)
            for (int32_t l : wild) {
                const int32_t gs[] = {a, c};
                const PagedGroups p{gs, &l, 1};
                const Segment s = group_segment(b, p, 4, 0);
                CHECK(s.seq0 >= 0 && s.seq0 <= s.seq1 && s.seq1 <= 3 && s.row0 >= 0 && s.rows >= 0 && s.row0 + s.rows <= 9 && s.key1 >= 0 && s.key1 <= 48);
                for (int q = 0; q < 3; ++q) {
                    const Segment x = seq_segment(b, 4, q, l);
                    CHECK(x.key0 >= 0 && x.key0 <= x.key1 && x.key1 <= 48);
                }
            }
}

int main() {
    rows_stay_inside();
    pages_stay_inside();
    spans();
    work();
    std::printf(fails ? "%d failed\n" : "all passed\n", fails);
    return fails != 0;
}
