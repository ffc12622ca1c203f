// Launchers of the paged-cache kernels.
#include "vh_launch.hpp"
#include "vh_paged.hpp"

namespace vh {

namespace {
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
    const int lph = a.c.hd <= 64 ? 16 : 32, per = 256 / lph;
    a.blocks = (a.heads + 2 * a.c.kv_heads + per - 1) / per;
    const int64_t grid = int64_t(a.b.rows) * a.blocks;
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    a.status = status_word();
    return by_type(type, [&](auto t, auto c) {
        using T = decltype(t);
        using C = decltype(c);
        return lph == 16 ? launch(k_kv_append<T, C, 16>, dim3(unsigned(grid)), dim3(256), 0, s, a)
                         : launch(k_kv_append<T, C, 32>, dim3(unsigned(grid)), dim3(256), 0, s, a);
    });
}

hipError_t launch_paged_attn(int type, PagedAttnArgs a, hipStream_t s) {
    const int64_t grid = int64_t(a.b.rows) * a.heads;
    if (a.c.hd <= 0 || a.c.hd > 128 || a.b.rows <= 0 || a.b.seqs <= 0 || grid > INT32_MAX) return hipErrorInvalidValue;
    a.status = status_word();
    return by_type(type, [&](auto t, auto c) {
        return launch(k_paged_attn_rows<decltype(t), decltype(c)>, dim3(unsigned(grid)), dim3(256), 0, s, a);
    });
}

}  // namespace vh
