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

static void groups() {
    const int32_t start[] = {2, 4, 4, 9}, len[] = {16, 32, 48};
    const PagedGroups p{start, len, 3};
    const int32_t want[] = {-1, -1, 0, 0, 2, 2, 2, 2, 2, -1};
    for (int s = 0; s < 10; ++s) CHECK(group_of(p, s) == want[s]);
}

int main() {
    rows_stay_inside();
    pages_stay_inside();
    spans();
    groups();
    std::printf(fails ? "%d failed\n" : "all passed\n", fails);
    return fails != 0;
}
