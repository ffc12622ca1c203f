// Launchers of the paged-cache kernels.
#include <algorithm>

#include "vh_launch.hpp"
#include "vh_paged.hpp"

namespace vh {

namespace {
template <int N>
using Int = std::integral_constant<int, N>;
// Row type (WT_F32, WT_F16, WT_BF16) and cache type together: f32 and f16 rows read an f16 cache, bf16 rows a bf16 one.
template <class F>
hipError_t by_type(int type, F &&f) {
    if (type == WT_F32) return f(float(), _Float16());
    if (type == WT_F16) return f(_Float16(), _Float16());
    if (type == WT_BF16) return f(__bf16(), __bf16());
    return hipErrorInvalidValue;
}
}  // namespace

hipError_t launch_kv_append(int type, AppendArgs a, hipStream_t s) {
    if (a.c.hd <= 0 || a.c.hd > 128 || a.c.hd % 8 || a.b.rows <= 0 || a.b.seqs <= 0) return hipErrorInvalidValue;
    // 8 values a lane (16 bytes of a 16-bit row) where a lane's pairs are one lane's too
    const bool wide = type != WT_F32 && (!a.rope || a.interleaved || a.rot % 16 == 0);
    const int lph = (a.c.hd <= 64 ? 16 : 32) / (wide ? 2 : 1), per = 256 / lph;
    // Rows that fill the chip by themselves: a wave each. Fewer: a row's turns of heads as blocks of their own up to about 2048
    // blocks (8 a CU).
    const bool many = a.b.rows >= 2048;
    const int64_t turns = (a.heads + 2 * a.c.kv_heads + per - 1) / per;
    a.blocks = int32_t(std::max<int64_t>(1, std::min<int64_t>(turns, 2048 / a.b.rows)));
    const int64_t grid = many ? (int64_t(a.b.rows) + 3) / 4 : int64_t(a.b.rows) * a.blocks;
    a.status = status_word();
    return by_type(type, [&](auto t, auto c) {
        using T = decltype(t);
        using C = decltype(c);
        const dim3 gr{unsigned(grid)}, bl{256};
        auto go = [&](auto lanes, auto n) {
            constexpr int L = decltype(lanes)::value, N = decltype(n)::value;
            return many ? launch(k_kv_append<T, C, L, N, 64>, gr, bl, 0, s, a) : launch(k_kv_append<T, C, L, N, 256>, gr, bl, 0, s, a);
        };
        if constexpr (!std::is_same<T, float>::value)
            if (wide) return lph == 8 ? go(Int<8>(), Int<8>()) : go(Int<16>(), Int<8>());
        return lph == 16 ? go(Int<16>(), Int<4>()) : go(Int<32>(), Int<4>());
    });
}

hipError_t launch_gather_rows(const float *src, int64_t cols, const int32_t *ids, int n, float *out, hipStream_t s) {
    if (n <= 0 || cols <= 0 || cols % 4) return hipErrorInvalidValue;
    return launch(k_gather_rows, dim3(unsigned(n)), dim3(256), 0, s, src, cols, ids, out);
}

// Tiles of 16, 32 or 128 query rows by the most that a segment can have; runs so that the launch has two blocks for each of the
// 256 CUs. A run is at least what the four waves of a small tile read at once (128 keys; 256 instead: a session's step behind
// 512 keys 11.7 instead of 10.4 us, eight behind 1024 15.1 instead of 14.1), of a group's tall tile 256 keys in at most 16 runs
// (64 rows behind 8192 keys: 44 us, in 32 runs 49, whose parts have to be written and read again).
PagedPlan plan_paged_attn(const PagedAttnArgs &a, int32_t max_rows, int32_t max_len, int32_t max_shared) {
    constexpr int32_t kBlocks = 512;
    const int32_t G = a.c.kv_heads, group = a.heads / G;
    auto tile_for = [](int64_t q) { return q <= 16 ? 16 : q <= 32 ? 32 : 128; };
    auto splits_for = [&](int64_t tiles, int32_t keys, int32_t least, int32_t limit) {
        const int64_t want = (kBlocks + tiles * G - 1) / (tiles * G), most = (int64_t(keys) + least - 1) / least;
        return int32_t(std::max<int64_t>(1, std::min<int64_t>({want, most, limit})));
    };
    PagedPlan p{};
    p.sleast = 128;
    const int64_t q = int64_t(a.b.rows) * group;
    p.stile = tile_for(int64_t(max_rows) * group);
    p.direct = int64_t(max_rows) * group <= p.stile;
    p.stiles = int32_t(p.direct ? a.b.seqs : std::min<int64_t>(q / p.stile + a.b.seqs, INT32_MAX));
    p.ssplits = splits_for(p.stiles, max_len, p.sleast, p.stile == 128 ? 16 : 32);
    if (a.p.groups) {
        p.gtile = tile_for(q);
        p.gtiles = int32_t(q / p.gtile + a.p.groups);
        p.gleast = p.gtile == 128 ? 256 : 128;
        p.gsplits = splits_for(std::max<int64_t>(1, q / p.gtile), std::max(max_shared, 1), p.gleast, p.gtile == 128 ? 16 : 32);
    }
    p.slots = p.gsplits + p.ssplits;
    if (p.gsplits || p.ssplits > 1) {
        p.parts = int64_t(a.b.rows) * a.heads * p.slots;
        p.ws_floats = p.parts * (2 + a.c.hd) + a.b.rows;
        p.counts = p.stile <= 32 && p.gtile <= 32 ? int64_t(a.b.rows) * a.heads : 0;
    }
    return p;
}

namespace {
template <class T, class C, int HDP, int GN, int GW, int SN, int SW>
hipError_t attn_launch(const PagedAttnArgs &a, hipStream_t s) {
    constexpr size_t pitch = HDP <= 64 ? 128 : 256, stages = size_t(256) * pitch;  // of either kind of tile
    constexpr size_t nq = GN > SN ? GN : SN, join = (size_t(2) * 4 * nq + size_t(4) * nq * (HDP + 4)) * 4;
    constexpr bool joins = GW == 1 || SW == 1;
    constexpr size_t smem = joins && join > stages ? join : stages;
    const int64_t grid = (int64_t(GN ? a.gtiles : 0) * a.gsplits + int64_t(a.stiles) * a.ssplits) * a.c.kv_heads;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    auto *k = k_paged_attn<T, C, HDP, GN, GW, SN, SW>;
    if (const hipError_t e = ensure_smem(reinterpret_cast<const void *>(k), smem); e != hipSuccess) return e;
    return launch(k, dim3(unsigned(grid)), dim3(256), smem, s, a);
}
template <class T, class C, int HDP>
hipError_t attn_of(const PagedAttnArgs &a, int gtile, int stile, hipStream_t s) {
    if (gtile == 0) {
        if (stile == 16) return attn_launch<T, C, HDP, 0, 0, 16, 1>(a, s);
        if (stile == 32) return attn_launch<T, C, HDP, 0, 0, 32, 1>(a, s);
        return attn_launch<T, C, HDP, 0, 0, 32, 4>(a, s);
    }
    if (gtile == 16) return attn_launch<T, C, HDP, 16, 1, 16, 1>(a, s);
    if (gtile == 32 && stile == 16) return attn_launch<T, C, HDP, 32, 1, 16, 1>(a, s);
    if (gtile == 32) return attn_launch<T, C, HDP, 32, 1, 32, 1>(a, s);
    if (stile == 16) return attn_launch<T, C, HDP, 32, 4, 16, 1>(a, s);
    if (stile == 32) return attn_launch<T, C, HDP, 32, 4, 32, 1>(a, s);
    return attn_launch<T, C, HDP, 32, 4, 32, 4>(a, s);
}
}  // namespace

hipError_t launch_paged_attn(int type, PagedAttnArgs a, const PagedPlan &p, float *ws, int32_t *count, hipStream_t s) {
    if (a.c.hd <= 0 || a.c.hd > 128 || a.c.hd % 8 || a.b.rows <= 0 || a.b.seqs <= 0 || (p.ws_floats && !ws) || (p.counts && !count) || p.slots > 64)
        return hipErrorInvalidValue;
    const int32_t group = a.heads / a.c.kv_heads;
    a.status = status_word();
    a.magic = uint32_t((uint64_t(1) << 32) / uint64_t(group)) + 1;
    a.slots = p.slots; a.gsplits = p.gsplits; a.ssplits = p.ssplits; a.gleast = p.gleast; a.sleast = p.sleast;
    a.gtiles = p.gtiles; a.stiles = p.stiles; a.direct = p.direct;
    a.po = ws;  // 16-byte aligned rows first
    a.ml = ws ? ws + p.parts * a.c.hd : nullptr;
    a.count = p.counts ? count : nullptr;
    a.desc = p.ws_floats && !p.counts ? reinterpret_cast<int32_t *>(a.ml + 2 * p.parts) : nullptr;
    const int64_t join = int64_t(a.b.rows) * ((a.heads + 7) / 8);
    if (join > INT32_MAX) return hipErrorInvalidValue;
    return by_type(type, [&](auto t, auto c) {
        using T = decltype(t);
        using C = decltype(c);
        const hipError_t e = a.c.hd <= 64 ? attn_of<T, C, 64>(a, p.gtile, p.stile, s) : attn_of<T, C, 128>(a, p.gtile, p.stile, s);
        if (e != hipSuccess || !a.desc) return e;
        return launch(k_paged_join<T>, dim3(unsigned(join)), dim3(256), 0, s, a);
    });
}

}  // namespace vh
