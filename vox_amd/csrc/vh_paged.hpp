// vh_paged.hpp — a key/value cache in pages: the append of a step's rows with their rotation, and the attention that
// reads it (gfx950, wave64).
#pragma once
#include "vh_common.hpp"
#include "vh_paged_index.hpp"
#include "vh_types.hpp"

namespace vh {

// The sequence that holds `row`, by 64 (then finer) samples of row_start at once: -1 when the row belongs to none. All
// lanes of a wave call it with one row.
VH_DEV int32_t find_seq(const PagedBatch &b, int32_t row) {
    const int lane = threadIdx.x & 63;
    int32_t lo = 0, n = b.seqs + 1;  // the last s in [lo, lo + n) with row_start[s] <= row
    while (true) {
        const int32_t step = (n + 63) / 64, at = lo + lane * step;
        const bool le = lane * step < n && b.row_start[at] <= row;
        const int cnt = __popcll(__ballot(le));
        if (!cnt) return -1;  // before the first row (row_start never falls)
        lo += (cnt - 1) * step;
        n = min(step, n - (cnt - 1) * step);
        if (step == 1) break;
    }
    return lo < b.seqs ? lo : -1;
}

template <class T>
VH_DEV f32x4 load4(const T *p) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 v = *reinterpret_cast<const t4 *>(p);
    return f32x4{float(v[0]), float(v[1]), float(v[2]), float(v[3])};
}
template <class T>
VH_DEV void store4(T *p, f32x4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<t4 *>(p) = t4{T(v[0]), T(v[1]), T(v[2]), T(v[3])};
}

// One head of one row per LPH lanes, 4 neighbouring values a lane; grid x = rows x a.blocks, block 256 (256 / LPH heads). A
// lane of a rotated head also loads the 4 values its own are paired with (halves: rot / 2 away, in L1 by then;
// interleaved: among its own), so no value crosses lanes but the norm's sum. Rows behind the last sequence, and rows at
// negative positions, write nothing.
template <class T, class C, int LPH>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
    const int row = int(blockIdx.x) / a.blocks;
    const int hh = (int(blockIdx.x) % a.blocks) * (256 / LPH) + int(threadIdx.x) / LPH, e = 4 * (int(threadIdx.x) % LPH);
    const int hd = a.c.hd, G = a.c.kv_heads;
    const int32_t s = find_seq(a.b, row);
    if (s < 0) return;
    const SeqRows sr = seq_rows(a.b, a.c.shift, s);
    raise_status(a.status, !sr.ok, kStatusBadBatch);
    const int32_t pos = sr.len - sr.n + (row - sr.first);
    if (pos < 0) return;
    if (pos >= sr.len || (a.rope && pos >= a.rope_len)) {
        raise_status(a.status, true, kStatusBadBatch);
        return;
    }
    const bool on = hh < a.heads + 2 * G && e < hd;
    const int hc = on ? hh : 0, ec = on ? e : 0;
    const bool is_q = hc < a.heads, is_v = hc >= a.heads + G;
    const T *src = static_cast<const T *>(a.qkv) + int64_t(row) * a.ld_qkv + int64_t(hc) * hd;
    const float *nw = is_v ? nullptr : is_q ? a.qn : a.kn;
    const bool turn = a.rope && !is_v && ec < a.rot;
    const int half = a.rot >> 1;
    const int pe = !turn || a.interleaved ? ec : ec < half ? ec + half : ec - half;
    f32x4 x = load4(src + ec), xp = load4(src + pe);
    // (cos, sin) of this lane's pairs: four pairs of the halves, or two of neighbours
    f32x4 cs0 = {1.f, 0.f, 1.f, 0.f}, cs1 = cs0;
    if (turn) {
        const float *rp = a.rope + int64_t(pos) * a.rot;
        if (a.interleaved) {
            cs0 = *reinterpret_cast<const f32x4 *>(rp + ec);
        } else {
            const float *r = rp + 2 * (ec < half ? ec : ec - half);
            cs0 = *reinterpret_cast<const f32x4 *>(r);
            cs1 = *reinterpret_cast<const f32x4 *>(r + 4);
        }
    }
    if (nw) {  // a head's lanes share the branch; every lane of the wave takes part in the sum below
        const f32x4 w = *reinterpret_cast<const f32x4 *>(nw + ec), wp = *reinterpret_cast<const f32x4 *>(nw + pe);
        const float ss = group_sum<LPH>(on ? x[0] * x[0] + x[1] * x[1] + (x[2] * x[2] + x[3] * x[3]) : 0.f);
        const float inv = 1.0f / sqrtf(ss / float(hd) + a.eps);
        x = w * (x * inv);
        xp = wp * (xp * inv);
    }
    if (!on) return;
    if (turn) {
        if (a.interleaved) {
            x = f32x4{x[0] * cs0[0] - x[1] * cs0[1], x[1] * cs0[0] + x[0] * cs0[1], x[2] * cs0[2] - x[3] * cs0[3],
                      x[3] * cs0[2] + x[2] * cs0[3]};
        } else {
            const f32x4 c = {cs0[0], cs0[2], cs1[0], cs1[2]}, sn = {cs0[1], cs0[3], cs1[1], cs1[3]};
            x = ec < half ? x * c - xp * sn : x * c + xp * sn;
        }
    }
    if (is_q) {
        if (a.q) store4(static_cast<T *>(a.q) + int64_t(row) * a.ld_q + int64_t(hc) * hd + ec, x);
        return;
    }
    const int32_t page = page_of(a.c, a.b.table + int64_t(s) * a.b.page_ld, pos);
    if (page < 0) {
        raise_status(a.status, true, kStatusBadPage);
        return;
    }
    C *dst = static_cast<C *>(is_v ? a.c.v : a.c.k) + key_offset(a.c, page, hc - a.heads - (is_v ? G : 0), pos) + ec;
    store4(dst, x);
}

// One (row, head) per block of 4 waves: wave w takes keys begin + w, + 4, ..., lane l dims l and l + 64, an online softmax
// per wave, the waves merged through LDS.
template <class T, class C>
__global__ __launch_bounds__(256) void k_paged_attn_rows(PagedAttnArgs a) {
    const int row = int(blockIdx.x) / a.heads, h = int(blockIdx.x) % a.heads;
    const int hd = a.c.hd, g = h / (a.heads / a.c.kv_heads), lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int32_t s = find_seq(a.b, row);
    if (s < 0) return;
    const SeqRows sr = seq_rows(a.b, a.c.shift, s);
    raise_status(a.status, !sr.ok, kStatusBadBatch);
    const int32_t pos = sr.len - sr.n + (row - sr.first);
    const Span sp = visible(pos, sr.len, a.prefix ? a.prefix[s] : 0, a.window);
    const int32_t grp = group_of(a.p, s);
    const int32_t shared = grp >= 0 ? a.p.len[grp] : 0;
    const int32_t *tab = a.b.table + int64_t(s) * a.b.page_ld;
    const int32_t *ptab = grp >= 0 ? a.b.table + int64_t(clamp_i32(a.p.seq_start[grp], 0, a.b.seqs - 1)) * a.b.page_ld : tab;
    const bool on0 = lane < hd, on1 = lane + 64 < hd;
    const T *q = static_cast<const T *>(a.q) + int64_t(row) * a.ld_q + int64_t(h) * hd;
    const float q0 = on0 ? float(q[lane]) : 0.f, q1 = on1 ? float(q[lane + 64]) : 0.f;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float mx = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int32_t j = sp.begin + w; j < sp.end; j += 4) {
        const int32_t page = page_of(a.c, j < shared ? ptab : tab, j);
        if (page < 0) {
            raise_status(a.status, lane == 0, kStatusBadPage);
            continue;
        }
        const int64_t off = key_offset(a.c, page, g, j);
        const C *kr = static_cast<const C *>(a.c.k) + off, *vr = static_cast<const C *>(a.c.v) + off;
        float sc = a.scale * wave_sum((on0 ? q0 * float(kr[lane]) : 0.f) + (on1 ? q1 * float(kr[lane + 64]) : 0.f));
        if (a.cap > 0.f) sc = a.cap * tanhf(sc / a.cap);
        sc -= slope * fabsf(float(pos - j));
        const float mn = fmaxf(mx, sc), corr = expf(mx - mn), p = expf(sc - mn);
        o0 = o0 * corr + (on0 ? p * float(vr[lane]) : 0.f);
        o1 = o1 * corr + (on1 ? p * float(vr[lane + 64]) : 0.f);
        l = l * corr + p;
        mx = mn;
    }
    __shared__ float sm_m[4], sm_l[4], sm_o[4][128];
    if (lane == 0) {
        sm_m[w] = mx;
        sm_l[w] = l;
    }
    sm_o[w][lane] = o0;
    sm_o[w][lane + 64] = o1;
    __syncthreads();
    if (int(threadIdx.x) >= hd) return;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int i = 0; i < 4; ++i) M = fmaxf(M, sm_m[i]);
    for (int i = 0; i < 4; ++i) {
        if (sm_m[i] == -INFINITY) continue;
        const float f = expf(sm_m[i] - M);
        L += f * sm_l[i];
        O += f * sm_o[i][threadIdx.x];
    }
    static_cast<T *>(a.out)[int64_t(row) * a.ld_out + int64_t(h) * hd + threadIdx.x] = T(L > 0.f || L != L ? O / L : 0.f);
}

}  // namespace vh
