// vh_paged.hpp — a key/value cache in pages: the append of a step's rows with their rotation, and the attention that
// reads it (gfx950, wave64).
#pragma once
#include <type_traits>

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

template <class T, int N = 4>
VH_DEV void load_n(const T *p, float (&x)[N]) {
    typedef T tn __attribute__((ext_vector_type(N)));
    const tn v = *reinterpret_cast<const tn *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = float(v[i]);
}
template <class T, int N>
VH_DEV void store_n(T *p, const float (&x)[N]) {
    typedef T tn __attribute__((ext_vector_type(N)));
    tn v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = T(x[i]);
    *reinterpret_cast<tn *>(p) = v;
}
template <class T>
VH_DEV void store4(T *p, f32x4 v) {
    const float x[4] = {v[0], v[1], v[2], v[3]};
    store_n(p, x);
}

// One head of one row per LPH lanes, N neighbouring values a lane (16 bytes of a row where halves of the rotation allow it, else 4
// values), TPR / LPH heads at a time. What a row costs is its chain of dependent reads (its sequence, position, page and
// rotation, then its values), so many rows are under way at once. TPR = 256: grid x = rows x a.blocks, block i of a row takes its
// heads in turns i, i + a.blocks, ... (one each for a step's few rows). TPR = 64, for rows that fill the chip by themselves: a
// wave a row, four rows a block, all heads in turns. A lane of a rotated head also loads the N values its own are paired with
// (halves: rot / 2 away, in L1 by then; interleaved: among its own), so no value crosses lanes but the norm's sum. Rows behind
// the last sequence, and rows at negative positions, write nothing. 6354 f32 rows 11.7 us, 4.9 TB/s (a large copy: 4.8); 8325
// bf16 rows 39.8 us, 3.5 TB/s; eight rows 4 us, a launch.
template <class T, class C, int LPH, int N, int TPR>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
    const int row = TPR == 64 ? int(blockIdx.x) * 4 + (int(threadIdx.x) >> 6) : int(blockIdx.x) / a.blocks;
    if (TPR == 64 && row >= a.b.rows) return;
    const int part = TPR == 64 ? 0 : int(blockIdx.x) % a.blocks, blocks = TPR == 64 ? 1 : a.blocks;
    const int e = N * (int(threadIdx.x) % LPH);
    const int hd = a.c.hd, G = a.c.kv_heads, heads = a.heads + 2 * G;
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
    const int32_t page = page_of(a.c, a.b.table + int64_t(s) * a.b.page_ld, pos);
    const T *from = static_cast<const T *>(a.qkv) + int64_t(row) * a.ld_qkv;
    const int half = a.rot >> 1, ec = e < hd ? e : 0;
    const bool inside = a.rope && ec < a.rot, low = ec < half;
    // this lane's cosines and sines: of N pairs of the halves, or of N / 2 of neighbours
    float cs[N], sn[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        cs[i] = 1.f;
        sn[i] = 0.f;
    }
    if (inside) {
        const float *rp = a.rope + int64_t(pos) * a.rot + (a.interleaved ? ec : 2 * (low ? ec : ec - half));
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            if (a.interleaved) {
                cs[i] = cs[i + 1] = rp[i];
                sn[i + 1] = rp[i + 1];
                sn[i] = -sn[i + 1];
            } else {
                cs[i] = rp[2 * i];
                cs[i + 1] = rp[2 * i + 2];
                sn[i] = low ? -rp[2 * i + 1] : rp[2 * i + 1];
                sn[i + 1] = low ? -rp[2 * i + 3] : rp[2 * i + 3];
            }
        }
    }
    const int pe = !inside || a.interleaved ? ec : low ? ec + half : ec - half;
    constexpr int PER = TPR / LPH;
    // the first values of the next turn are loaded during this one
    auto head_of = [&](int turn) { return (part + turn * blocks) * PER + int(threadIdx.x) % TPR / LPH; };
    auto values = [&](int turn, float (&x)[N], float (&xp)[N]) {
        const T *src = from + int64_t(min(head_of(turn), heads - 1)) * hd;
        load_n(src + ec, x);
        load_n(src + pe, xp);
    };
    const int turns = ((heads + PER - 1) / PER + blocks - 1) / blocks;
    float nx[N], np[N];
    values(0, nx, np);
    for (int k = 0; k < turns; ++k) {
        const int hh = head_of(k), hc = min(hh, heads - 1);
        const bool on = hh < heads && e < hd, is_q = hc < a.heads, is_v = hc >= a.heads + G;
        float x[N], xp[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = nx[i];
            xp[i] = np[i];
        }
        if (k + 1 < turns) values(k + 1, nx, np);
        const float *nw = is_v ? nullptr : is_q ? a.qn : a.kn;
        if (nw) {  // a head's lanes share the branch
            float w[N], wp[N], ss = 0.f;
            load_n(nw + ec, w);
            load_n(nw + pe, wp);
#pragma unroll
            for (int i = 0; i < N; ++i) ss = fmaf(x[i], x[i], ss);
            ss = group_sum<LPH>(e < hd ? ss : 0.f);
            const float inv = 1.0f / sqrtf(ss / float(hd) + a.eps);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = w[i] * (x[i] * inv);
                xp[i] = wp[i] * (xp[i] * inv);
            }
        }
        if (!on) continue;
        if (inside && !is_v) {
            float y[N];
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = x[i] * cs[i] + (a.interleaved ? x[i ^ 1] : xp[i]) * sn[i];
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = y[i];
        }
        if (is_q) {
            if (a.q) store_n(static_cast<T *>(a.q) + int64_t(row) * a.ld_q + int64_t(hc) * hd + ec, x);
            continue;
        }
        if (page < 0) {
            raise_status(a.status, true, kStatusBadPage);
            continue;
        }
        store_n(static_cast<C *>(is_v ? a.c.v : a.c.k) + key_offset(a.c, page, hc - a.heads - (is_v ? G : 0), pos) + ec, x);
    }
}

// grid n, block 256: row ids[blockIdx.x] of src to row blockIdx.x of out (the last rows of a ragged batch's sequences).
static __global__ __launch_bounds__(256) void k_gather_rows(const float *src, int64_t cols, const int32_t *ids, float *out) {
    const float *from = src + int64_t(ids[blockIdx.x]) * cols;
    float *to = out + int64_t(blockIdx.x) * cols;
    for (int64_t i = 4 * int64_t(threadIdx.x); i < cols; i += 1024) *reinterpret_cast<f32x4 *>(to + i) = *reinterpret_cast<const f32x4 *>(from + i);
}

// ------------------------------------------------------------------ attention
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Of the cache's type: the sum of 8 values onto c in 32 bits; matrix products: c += a b, columns of b in the lanes' low bits, the K elements of a lane neighbours.
template <class C>
struct Mx;
template <>
struct Mx<_Float16> {
    typedef f16x8 v8;
    static constexpr uint16_t kExp = 0x7C00, kOne = 0x3C00;
    static VH_DEV float sum(v8 a, float c) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 one = {1, 1};
#pragma unroll
        for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2(f16x2{a[i], a[i + 1]}, one, c, false);
        return c;
    }
    static VH_DEV f32x16 mm(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static VH_DEV f32x4 mm(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mx<__bf16> {
    typedef bf16x8 v8;
    static constexpr uint16_t kExp = 0x7F80, kOne = 0x3F80;
    static VH_DEV float sum(v8 a, float c) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 one = {__bf16(1.f), __bf16(1.f)};
#pragma unroll
        for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[i], a[i + 1]}, one, c, false);
        return c;
    }
    static VH_DEV f32x16 mm(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static VH_DEV f32x4 mm(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// What lanes without a key (behind a sequence's last, past head_dim) read instead.
static __device__ __align__(16) uint32_t kZero16[4];

// 16 bytes per lane to LDS lds + 16 lane, from its own address, or from a common one and its own 32-bit offset (s_nop: an
// address that a vector instruction wrote into scalar registers needs 5 cycles); as dma_b128, the waits are the caller's.
VH_DEV void dma_lane16(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
VH_DEV void dma_off16(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
// Every LDS read of this wave has returned, then the block's barrier.
VH_DEV void read_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
VH_DEV void block_barrier() { asm volatile("s_barrier" ::: "memory"); }

VH_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum, sum over the lanes that hold one query row (64 / NQ, NQ apart); every one of them gets it.
template <int NQ>
VH_DEV float rows_max(float v) {
    if (NQ == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int NQ>
VH_DEV float rows_sum(float v) {
    if (NQ == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// c tanh(x) of x2 = 2 x log2 e. 16-bit rows: c - 2 c / (1 + 2^x2), off by about 2^-23 c. FINE: by about 2^-23 of its value
// also near zero, where that cancels: an odd polynomial (Taylor, to x^11) below 0.3. Both are computed and one is taken: no
// branch.
template <bool FINE>
VH_DEV float tanh_f(float x2, float c) {
    float big = fmaf(-2.f * c, __builtin_amdgcn_rcpf(1.f + exp2_fast(x2)), c);
    if constexpr (!FINE) return big;
    const float x = x2 * 0.34657359027997264f, xx = x * x;
    float p = fmaf(xx, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    p = fmaf(xx, p, -17.0f / 315.0f);
    p = fmaf(xx, p, 2.0f / 15.0f);
    p = fmaf(xx, p, -1.0f / 3.0f);
    p = c * fmaf(x * xx, p, x);
    asm volatile("" : "+v"(big), "+v"(p));
    return fabsf(x) < 0.3f ? p : big;
}

// u / d by m = 2^32 / d + 1 (d > 1): at most one too many.
VH_DEV int32_t div_by(int32_t u, int32_t d, uint32_t m) {
    const int32_t q = d == 1 ? u : int32_t(__umulhi(uint32_t(u), m));
    return q - (q * d > u);
}

// 16 and 8 bytes past the caches that other XCDs do not see (agent scope), for parts that another block joins.
VH_DEV void put_far(float *p, float a, float b) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), uint64_t(__float_as_uint(b)) << 32 | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
VH_DEV float2 get_far(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float(uint32_t(v)), __uint_as_float(uint32_t(v >> 32))};
}

// The shared keys of the group that holds sequence s (the first that does; none: 0): 64 groups at a time.
VH_DEV int32_t shared_keys(const PagedGroups &p, int32_t s, int64_t most) {
    const int lane = threadIdx.x & 63;
    for (int32_t base = 0; base < p.groups; base += 64) {
        const int32_t g = min(base + lane, p.groups - 1), n = p.len[g];
        const uint64_t in = __ballot(base + lane < p.groups && s >= p.seq_start[g] && s < p.seq_start[g + 1]);
        if (in) return clamp_i32(__builtin_amdgcn_readlane(n, __ffsll(static_cast<unsigned long long>(in)) - 1), 0, most);
    }
    return 0;
}

// The segment (of n, with rows_of(i) rows each) and the tile in it of the launch's tile t: 64 segments at a time.
template <class F>
VH_DEV bool find_tile(int32_t n, int32_t t, int32_t group, int32_t tile, F rows_of, int32_t *seg, int32_t *local) {
    const int lane = threadIdx.x & 63;
    for (int32_t base = 0; base < n; base += 64) {
        const int32_t mine = base + lane < n ? tiles_of(rows_of(base + lane), group, tile) : 0;
        int32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int32_t up = __shfl_up(sum, o, 64);
            sum += lane >= o ? up : 0;
        }
        const uint64_t past = __ballot(sum > t);
        if (past) {
            const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
            *seg = base + l;
            *local = t - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(mine, l));
            return true;
        }
        t -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// A query row's parts joined by 32 lanes, 4 dims each: M = the largest maximum, sums and outputs scaled by 2^(max - M) and added
// in slot order. gn parts of its group, then (from slot gsplits on) sn of its own keys.
template <class T, bool FAR>
VH_DEV void join_row(const PagedAttnArgs &a, int64_t rh, int32_t gn, int32_t sn) {
    const int l32 = threadIdx.x & 31, e = 4 * l32, n = gn + sn;
    const float *ml = a.ml + 2 * rh * a.slots, *po = a.po + rh * a.slots * a.c.hd + (e < a.c.hd ? e : 0);
    auto slot = [&](int i) { return i < gn ? i : a.gsplits + i - gn; };
    float m[2], l[2], M = -INFINITY, L = 0.f;  // parts l32 and 32 + l32
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        m[k] = -INFINITY;
        l[k] = 0.f;
        if (32 * k + l32 < n) {
            const float *p = ml + 2 * slot(32 * k + l32);
            const float2 v = FAR ? get_far(p) : *reinterpret_cast<const float2 *>(p);
            m[k] = v.x;
            l[k] = v.y;
        }
        M = fmaxf(M, m[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        m[k] = m[k] == -INFINITY ? 0.f : exp2_fast(m[k] - M);
        L += m[k] * l[k];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n; i += 8) {  // 8 parts' outputs in flight
        f32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float *p = po + int64_t(slot(min(i + k, n - 1))) * a.c.hd;
            if constexpr (FAR) {
                const float2 lo = get_far(p), hi = get_far(p + 2);
                v[k] = f32x4{lo.x, lo.y, hi.x, hi.y};
            } else {
                v[k] = *reinterpret_cast<const f32x4 *>(p);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float f = __shfl(i + k < 32 ? m[0] : m[1], (int(threadIdx.x) & 32) + ((i + k) & 31), 64);
            if (i + k < n) x += v[k] * f;
        }
    }
    if (e >= a.c.hd) return;
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    const int64_t row = rh / a.heads;
    store4(static_cast<T *>(a.out) + row * a.ld_out + (rh - row * a.heads) * a.c.hd + e, x * inv);
}

// The same for up to 64 segments, the tiles with the highest index first, whatever their segment: the last tiles of prompts see
// the most keys, and what starts last should not take longest (24 prompts of 1 to 700 rows: 92 us segment by segment). Tiles
// up to 2^23, whose sums are exact in f32.
template <class F>
VH_DEV bool find_tile_down(int32_t n, int32_t t, int32_t group, int32_t tile, F rows_of, int32_t *seg, int32_t *local) {
    const int lane = threadIdx.x & 63;
    const float mine = lane < n ? float(tiles_of(rows_of(lane), group, tile)) : 0.f;
    auto from = [&](int32_t i) { return int32_t(wave_sum(fmaxf(mine - float(i), 0.f))); };  // tiles of index i and more
    if (t >= from(0)) return false;
    int32_t lo = 0, hi = int32_t(wave_max(mine));  // the index: the highest with from(index) > t
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (from(mid) > t) lo = mid;
        else hi = mid;
    }
    const uint64_t with = __ballot(mine > float(lo));
    const int32_t rank = __popcll(with & ((uint64_t(1) << lane) - 1)), want = t - from(lo + 1);
    const uint64_t at = __ballot((with >> lane & 1) && rank == want);
    *seg = __ffsll(static_cast<unsigned long long>(at)) - 1;
    *local = lo;
    return at != 0;
}

// Softmax attention of a tile of query rows over a run of keys, on the matrix cores, transposed: S^T = K Q^T has a query row's
// scores in the registers of one lane (two with 32 x 32 products, four with 16 x 16), so a row's maximum is a few register
// maxima and one or two lane swaps, the rescale of O^T is by a lane's own factor, and P^T is already the operand that O^T +=
// V^T P^T wants: the K index of that product is the order in which S^T's rows lie in registers, and V^T's operand is read in the
// same order by the transposing LDS read (4 keys at a time). Keys and values come to LDS by DMA, in 16-byte pieces at
// piece ^ f(key), so that neither the row-wise reads of K nor the 4 x 16 blocks of V meet in a bank.
//
// NQ query rows per wave, WQ waves beside each other on the same keys, the other 4 / WQ on other keys (tiles of KW keys each,
// every 4 / WQ-th), joined through LDS at the end. WQ = 4 (128 rows, prompts and tall prefixes): keys are read from LDS for
// 128 rows at once, bound by the products and the exponentials beside them. WQ = 1 (16 or 32 rows, steps): every wave streams its
// own keys, no barrier in the loop, bound by the bytes.
//
// f32 rows: q and the weights as two f16 halves, both multiplied (exact products, to about 2^-22). f16 / bf16 rows: the
// weights are rounded to the cache's type, half a step each; sums, maxima and outputs stay in 32 bits. Weights are
// 2^(s - m + kUp) with m within 2^kLag of the running maximum: the running maximum only moves (and O^T is only rescaled) when a
// score passes it by more than kLag, and kUp keeps small f16 weights out of the subnormals.
//
// Measured (calls one after another): 2048 f16 rows of 16 heads behind 30000 keys 630 us, 825 TFLOP/s (a large library product on
// this card: 1200), the matrix cores 41 % busy, the vector units 38 %, LDS 30 % and another 10 % in conflicts of V's reads:
// two waves a SIMD whose phases overlap only in part. 64 sessions of up to 8192 keys 41 us, 4.0 TB/s (a large copy: 4.8).
// One session's step behind 512 keys 10.3 us, of which the launch is 4: a chain of four round trips (the batch, the page
// table, the keys, the join), about 1 us each, and the tiles.
template <class T, class C, int HDP, int NQ, int WQ, bool GROUPS>
VH_DEV void attn_tile(const PagedAttnArgs &a, int id, uint8_t *smem) {
    typedef typename Mx<C>::v8 v8;
    typedef typename std::conditional<NQ == 32, f32x16, f32x4>::type acc;
    constexpr bool kSplit = std::is_same<T, float>::value;
    constexpr int WK = 4 / WQ, KW = WQ == 4 ? 64 : 32, TILE = NQ * WQ;
    constexpr int PITCH = HDP <= 64 ? 128 : 256, CPR = PITCH / 16, R = 64 / CPR;  // bytes of a key in LDS, its pieces, keys a DMA
    constexpr int KB = KW * PITCH, STAGE = 2 * KB, STAGES = WQ == 4 ? 2 : 1;      // K then V of a tile
    constexpr int NI = KW / R / WQ;                                               // DMAs of K (and of V) a wave and tile
    constexpr int KD = NQ == 32 ? 16 : 32;                                        // K of one product
    constexpr int SUB = NQ, NSUB = KW / SUB, AV = NQ == 32 ? 16 : 4;              // keys of one S^T product, values a lane
    constexpr int ND = HDP / NQ;                                                  // O^T products
    constexpr int NC = KW / KD;                                                   // P^T operands
    constexpr float kUp = std::is_same<C, __bf16>::value ? 0.f : 6.f, kLag = 8.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int wq = wave % WQ, wk = wave / WQ, col = lane % NQ, lh = lane / NQ;  // lh: which rows of a product this lane holds
    const int G = a.c.kv_heads, group = a.heads / G, hd = a.c.hd;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((lds_void *)smem));
    const int32_t splits = GROUPS ? a.gsplits : a.ssplits;
    // kv heads are the fastest index: blocks of one kv head (and its keys) meet in few XCDs' L2
    const int g = id % G;
    id /= G;
    const int split = id % splits;
    int32_t t = id / splits, seg_id = t, local = 0, shared = 0;  // shared: of a sequence, the keys of its group
    Segment seg;
    bool whole = false;  // rows whose keys are one run are written here, otherwise the last block of a row joins its parts
    int32_t gruns = 0, pf = 0;
    Runs runs;
    if constexpr (GROUPS) {
        if (a.p.groups == 1) {  // nothing to look for: a round trip less
            seg_id = 0;
            local = t;
        } else if (!find_tile(a.p.groups, t, group, TILE, [&](int32_t i) { return group_segment(a.b, a.p, a.c.shift, i).rows; }, &seg_id, &local)) {
            return;
        }
        seg = group_segment(a.b, a.p, a.c.shift, seg_id);
        runs = runs_of(seg.key0, seg.key1, splits, a.gleast);
    } else {
        auto rows_of = [&](int32_t i) {
            const int32_t r0 = clamp_i32(a.b.row_start[i], 0, a.b.rows);
            return clamp_i32(a.b.row_start[i + 1], r0, a.b.rows) - r0;
        };
        if (!a.direct && a.b.seqs == 1) {
            seg_id = 0;
            local = a.stiles - 1 - t;
        } else if (!a.direct && !(a.b.seqs <= 64 && a.stiles <= 1 << 23 ? find_tile_down(a.b.seqs, t, group, TILE, rows_of, &seg_id, &local)
                                                                 : find_tile(a.b.seqs, t, group, TILE, rows_of, &seg_id, &local)))
            return;
        pf = a.prefix ? a.prefix[seg_id] : 0;
        shared = shared_keys(a.p, seg_id, a.b.page_ld << a.c.shift);
        seg = seq_segment(a.b, a.c.shift, seg_id, shared);
        runs = runs_of(seg.key0, seg.key1, splits, a.sleast);
    }
    const int32_t qrows = seg.rows * group;
    raise_status(a.status, threadIdx.x == 0 && (!seg.ok || (!GROUPS && a.direct && qrows > TILE)), kStatusBadBatch);
    if (local * TILE >= qrows) return;
    if constexpr (!GROUPS) {
        gruns = runs_of(0, shared, a.gsplits, a.gleast).count;
        whole = gruns == 0 && runs.count <= 1;
        if (a.desc && split == 0 && g == 0) {  // what k_paged_join will find
            const int32_t i = div_by(local * TILE, group, a.magic) + int(threadIdx.x);
            if (i < seg.rows && i * group < local * TILE + TILE) a.desc[seg.row0 + i] = whole ? 0 : gruns | runs.count << 16;
        }
    }
    if (split >= runs.count && !(whole && split == 0)) return;
    const Span run = runs.count ? run_at(runs, seg.key0, seg.key1, split) : Span{0, 0};
    auto token = [&](int32_t q) { return div_by(q, group, a.magic); };

    int32_t kb = run.begin, ke = run.end;  // the block's keys
    if constexpr (!GROUPS) {               // a sequence's rows see no less at either end the later they stand
        const int32_t before = seg.key1 - seg.rows;
        kb = max(kb, visible(before + token(local * TILE), seg.key1, pf, a.window).begin);
        ke = min(ke, visible(before + token(min(local * TILE + TILE, qrows) - 1), seg.key1, pf, a.window).end);
    }
    kb = __builtin_amdgcn_readfirstlane(kb & ~(KW * WK - 1));
    ke = __builtin_amdgcn_readfirstlane(ke);
    const int32_t k_first = kb + wk * KW;
    // the pages of 64 table entries from pbase on, lane l that of pbase + l; the first ones on their way before all else
    const int32_t *tab = a.b.table + int64_t(seg.seq0) * a.b.page_ld;
    const int shift = a.c.shift;
    const int32_t last_page = run.end > run.begin ? (run.end - 1) >> shift : 0, first_page = run.begin >> shift;
    int32_t pg = 0, pbase = max(k_first >> shift, first_page);
    bool checked = false, bad_page = false;
    if (k_first < ke) pg = tab[min(pbase + lane, last_page)];

    // this lane's query row
    const int32_t u = local * TILE + wq * NQ + col;
    const bool valid = u < qrows;
    const int32_t tok = valid ? token(u) : 0, row = seg.row0 + tok, head = g * group + (valid ? u - tok * group : 0);
    // the queries, raw: needed only after the first keys are on their way
    constexpr int NK = HDP / KD;
    u32x4 qraw[NK][kSplit ? 2 : 1];
    {
        const T *qr = static_cast<const T *>(a.q) + int64_t(row) * a.ld_q + int64_t(head) * hd;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            const int d = KD * c + 8 * lh;
            const bool in = valid && d < hd;
            qraw[c][0] = in ? *reinterpret_cast<const u32x4 *>(qr + d) : u32x4{0u, 0u, 0u, 0u};
            if constexpr (kSplit) qraw[c][1] = in ? *reinterpret_cast<const u32x4 *>(qr + d + 4) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    const float slope_raw = a.slopes ? a.slopes[head] : 0.f;
    int32_t pos, lo_any, hi_any, lo_all, hi_all;  // of the wave's rows: the keys that any sees, and those that all see
    int32_t lo_blk, hi_blk;                       // of the block's rows: those that all see
    int32_t parts = gruns + runs.count;           // of this lane's row
    Span see;
    if constexpr (GROUPS) {
        // the sequence that holds the row: by the guess of one row each, or halving
        int32_t seq = min(seg.seq0 + tok, seg.seq1 - 1);
        if (!(a.b.row_start[seq] <= row && row < a.b.row_start[seq + 1])) {
            int32_t lo = seg.seq0, hi = seg.seq1;  // the last s with row_start[s] <= row
            while (hi - lo > 1) {
                const int32_t mid = (lo + hi) >> 1;
                if (a.b.row_start[mid] <= row) lo = mid;
                else hi = mid;
            }
            seq = lo;
        }
        const SeqRows sr = seq_rows(a.b, a.c.shift, seq);
        pos = sr.len - sr.n + (row - sr.first);
        see = visible(pos, sr.len, a.prefix ? a.prefix[seq] : 0, a.window);
        gruns = runs.count;
        parts = gruns + runs_of(min(seg.key1, sr.len), sr.len, a.ssplits, a.sleast).count;
        lo_any = run.begin;
        hi_any = run.end;
        const bool all = __all(!valid || (see.begin <= run.begin && see.end >= run.end));
        lo_all = lo_blk = all ? run.begin : INT32_MAX;
        hi_all = hi_blk = run.end;
        if constexpr (WQ > 1) {
            __shared__ int32_t least[4];
            if (lane == 0) least[wave] = lo_all;
            read_barrier();
            lo_blk = max(max(least[0], least[1]), max(least[2], least[3]));
        }
    } else {
        const int32_t len = seg.key1, before = len - seg.rows, w0 = local * TILE + wq * NQ;
        pos = before + tok;
        see = visible(pos, len, pf, a.window);
        auto at = [&](int32_t q) { return visible(before + token(min(q, qrows - 1)), len, pf, a.window); };
        const Span b0 = at(local * TILE), b1 = at(local * TILE + TILE - 1), first = at(w0), last = at(w0 + NQ - 1);
        lo_any = w0 < qrows ? max(first.begin, run.begin) : INT32_MAX;
        hi_any = min(last.end, run.end);
        lo_all = max(last.begin, run.begin);
        hi_all = min(first.end, run.end);
        lo_blk = WQ > 1 ? max(b1.begin, run.begin) : lo_all;
        hi_blk = WQ > 1 ? min(b0.end, run.end) : hi_all;
    }
    see.begin = max(see.begin, run.begin);
    see.end = valid ? min(see.end, run.end) : 0;
    if (see.begin >= see.end) see = Span{0, 0};
    const uint32_t see_n = uint32_t(see.end - see.begin);
    kb = __builtin_amdgcn_readfirstlane(kb & ~(KW * WK - 1));
    ke = __builtin_amdgcn_readfirstlane(ke);

    constexpr float kLog2e = 1.44269504088896341f;
    const bool capped = a.cap > 0.f, biased = a.slopes != nullptr;
    const float sc = fabsf(a.scale) * kLog2e * (capped ? 2.f / a.cap : 1.f), cap2 = a.cap * kLog2e;  // capped: 2 x log2 e of tanh(x)
    const float slope = slope_raw * kLog2e;

    // DMA: this lane's key of R and piece of CPR; where the swizzle needs more of the key than its place in the DMA, by the DMA's
    // number. K: piece ^ key, so that 16 keys' reads of one piece meet nowhere; V: by pairs of pieces, which its blocks of 16
    // dims are.
    constexpr int VK = PITCH == 256 ? 4 : 2;
    static_assert(NI % VK == 0, "the swizzle goes by the DMA's number");
    const int rin = lane / CPR, piece = lane % CPR;
    uint32_t koff[VK], voff[VK];
    uint32_t kin = 0, vin = 0;  // bit n: the piece lies inside head_dim
#pragma unroll
    for (int n = 0; n < VK; ++n) {
        const int kp = piece ^ (PITCH == 256 ? 4 * n + rin : 4 * n + (rin >> 1));
        const int vp = piece ^ (PITCH == 256 ? ((4 * n + rin) & 7) << 1 : ((rin >> 1) & 3) << 1);
        koff[n] = (uint32_t(rin) * uint32_t(a.c.pos_stride) + 8 * kp) * 2;
        voff[n] = (uint32_t(rin) * uint32_t(a.c.pos_stride) + 8 * vp) * 2;
        kin |= uint32_t(8 * kp < hd) << n;
        vin |= uint32_t(8 * vp < hd) << n;
    }
    // K (or V, by its pool's first byte of this kv head) of the keys kt .. kt + KW - 1 to buf. A tile inside the run, of whole
    // pitches and pages of the pool, takes its addresses from scalars alone; otherwise lanes without a key read zeros.
    const uint8_t *const kpool = static_cast<const uint8_t *>(a.c.k) + int64_t(g) * a.c.head_stride * 2;
    const uint8_t *const vpool = static_cast<const uint8_t *>(a.c.v) + int64_t(g) * a.c.head_stride * 2;
    const int64_t page_bytes = a.c.page_stride * 2;
    const uint32_t pos_bytes = uint32_t(a.c.pos_stride) * 2;
    auto issue = [&](int32_t kt, const uint8_t *from, const uint32_t (&off)[VK], uint32_t inside, uint32_t buf) {
        const int32_t i0 = max(kt >> shift, first_page), i1 = min((kt + KW - 1) >> shift, last_page);
        if (i1 >= pbase + 64) {
            pbase = i0;
            pg = tab[min(i0 + lane, last_page)];
            checked = false;
        }
        if (!checked) {
            pg = uint32_t(pg) < uint32_t(a.c.pages) ? pg : -1;
            bad_page |= __any(pg < 0);
            checked = true;
        }
        auto at = [&](int32_t page, int32_t key) { return int64_t(page) * page_bytes + int64_t(uint64_t(key & ((1 << shift) - 1)) * pos_bytes); };
        if (hd == PITCH / 2 && !bad_page && kt >= run.begin && kt + KW <= run.end) {
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const int i = wq * NI + n;
                const int32_t key = kt + R * i;
                dma_off16(from + at(__builtin_amdgcn_readlane(pg, (key >> shift) - pbase), key), off[n % VK], buf + i * 1024);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const int i = wq * NI + n;
                const int32_t key = kt + R * i, mine = key + rin;
                const int32_t page = __builtin_amdgcn_readlane(pg, (min(max(key >> shift, i0), i1) - pbase) & 63);
                const bool in = page >= 0 && (inside >> (n % VK) & 1) && mine >= run.begin && mine < run.end;
                const uint8_t *zero = reinterpret_cast<const uint8_t *>(kZero16);
                dma_lane16(in ? from + at(page, key) + off[n % VK] : zero, buf + i * 1024);
            }
        }
    };
    // WQ = 4: two stages of K and V, the next tile on its way during this one. WQ = 1: one buffer each, refilled as soon as the
    // wave has read it: K's during the softmax and V's product, V's during the next K's.
    const uint32_t stream = uint32_t(wk) * STAGES * STAGE, buf0 = lds0 + stream;
    if (k_first < ke) {
        issue(k_first, kpool, koff, kin, buf0);
        issue(k_first, vpool, voff, vin, buf0 + KB);
    }

    // queries as the second operand of S^T: column col, K elements 8 lh .. of every product. A negative scale turns them
    // around, so that the largest product is the largest score.
    v8 qh[NK], ql[kSplit ? NK : 1];
    {
        bool bad = false;
        const uint32_t flip = a.scale < 0.f ? (kSplit ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            if constexpr (kSplit) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    _Float16 hi, lo;
                    bad |= split_f16(__uint_as_float(qraw[c][e / 4][e & 3] ^ flip), hi, lo);
                    qh[c][e] = hi;
                    ql[c][e] = lo;
                }
            } else {
                qh[c] = __builtin_bit_cast(v8, qraw[c][0] ^ u32x4{flip, flip, flip, flip});
            }
        }
        raise_status(a.status, bad, kStatusF16Range);
    }

    acc o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < AV; ++i) o[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;  // m: the running maximum in log2 units; l: this lane's share of the sum
    // LDS addresses: K operand, key col (+ NQ j), piece (KD / 8) c + lh; V^T operand, key 4 (lane / 16 or lh) + lane / 4 % 4,
    // dims 4 (lane % 4) of 16 (and the upper 16 of 32 for odd lane / 16)
    const int ksw = PITCH == 256 ? col & 15 : (col >> 1) & 7;
    const int vi = lane & 15, vkey = (NQ == 32 ? 4 * lh : 4 * (lane >> 4)) + (vi >> 2), vd = (NQ == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((vi & 3) >> 1);
    const int vsw = PITCH == 256 ? (vkey & 7) << 1 : ((vkey >> 1) & 3) << 1;
    // value i of S^T product j: its key in the tile
    auto key_in = [&](int j, int i) { return SUB * j + (NQ == 32 ? (i & 3) + 8 * (i >> 2) + 4 * lh : i + 4 * lh); };

    int stage = 0;
    for (int32_t kt = k_first; kt < ke; kt += KW * WK, stage ^= STAGES - 1) {
        const int32_t next = kt + KW * WK;
        const bool more = next < ke, seen = lo_any < kt + KW && hi_any > kt;
        const uint8_t *Ks = smem + stream + stage * STAGE, *Vs = Ks + KB;
        if constexpr (WQ > 1) {
            if (more) {
                issue(next, kpool, koff, kin, buf0 + (stage ^ 1) * STAGE);
                issue(next, vpool, voff, vin, buf0 + (stage ^ 1) * STAGE + KB);
                wait_step<2 * NI>();
            } else {
                wait_step<0>();
            }
            block_barrier();
        } else {
            wait_step<NI>();  // K; V may still be on its way
        }
        acc s[NSUB];
        float unit = sc;  // of s, in log2 units
        if (seen) {
#pragma unroll
            for (int j = 0; j < NSUB; ++j) {
#pragma unroll
                for (int i = 0; i < AV; ++i) s[j][i] = 0.f;
#pragma unroll
                for (int c = 0; c < NK; ++c) {
                    const v8 k = *reinterpret_cast<const v8 *>(Ks + (SUB * j + col) * PITCH + (((KD / 8 * c + lh) ^ ksw) << 4));
                    s[j] = Mx<C>::mm(k, qh[c], s[j]);
                    if constexpr (kSplit) s[j] = Mx<C>::mm(k, ql[c], s[j]);
                }
            }
        }
        if constexpr (WQ == 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
            if (more) {
                issue(next, kpool, koff, kin, buf0);
                wait_step<NI>();  // V
            } else {
                wait_step<0>();
            }
        }
        auto v_at = [&](int c, int d) {
            // keys KD c + (4 neighbours, then 4 neighbours 8 or 16 on), dims NQ d ..
            const uint8_t *at = Vs + (KD * c + vkey) * PITCH + (((NQ / 8 * d + vd) ^ vsw) << 4) + (vi & 1) * 8;
            union {
                s16x4 half[2];
                v8 whole;
            } r;
            r.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)at);
            r.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at + (NQ == 32 ? 8 : 16) * PITCH));
            return r.whole;
        };
        // A value that is not finite may stand at a key that only some rows see, and 0 times it would reach the others. Then a
        // row that sees one becomes NaN in its place, and V goes on without them. All waves of a shared tile look at the same
        // values, and so decide alike.
        if (WQ > 1 ? !(lo_blk <= kt && hi_blk >= kt + KW) : seen && !(lo_all <= kt && hi_all >= kt + KW)) {
            u16x8 top = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KB / 1024; ++i)
                top = __builtin_elementwise_max(top, *reinterpret_cast<const u16x8 *>(Vs + i * 1024 + lane * 16) & uint16_t(0x7FFF));
            bool wild = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) wild |= top[e] >= Mx<C>::kExp;
            if (__builtin_expect(__any(wild), 0)) {
                if (seen) {
#pragma unroll 1
                    for (int c = 0; c < NC; ++c) {
                        u16x8 eye;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int key = KD * c + (NQ == 32 ? (e & 3) + 8 * (e >> 2) : (e & 3) + 16 * (e >> 2)) + 4 * lh;
                            eye[e] = uint32_t(kt + key - see.begin) < see_n ? Mx<C>::kOne : 0;
                        }
#pragma unroll
                        for (int d = 0; d < ND; ++d) {
                            u16x8 w = __builtin_bit_cast(u16x8, v_at(c, d));
#pragma unroll
                            for (int e = 0; e < 8; ++e) w[e] = (w[e] & 0x7FFF) >= Mx<C>::kExp ? Mx<C>::kOne : 0;
                            acc hit;
#pragma unroll
                            for (int i = 0; i < AV; ++i) hit[i] = 0.f;
                            hit = Mx<C>::mm(__builtin_bit_cast(v8, w), __builtin_bit_cast(v8, eye), hit);
#pragma unroll
                            for (int i = 0; i < AV; ++i) o[d][i] = hit[i] > 0.f ? __builtin_nanf("") : o[d][i];
                        }
                    }
                }
                if constexpr (WQ > 1) read_barrier();
                for (int i = wq; i < KB / 1024; i += WQ) {
                    u16x8 *at = reinterpret_cast<u16x8 *>(smem + stream + stage * STAGE + KB + i * 1024 + lane * 16);
                    u16x8 x = *at;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = (x[e] & 0x7FFF) >= Mx<C>::kExp ? 0 : x[e];
                    *at = x;
                }
                if constexpr (WQ > 1) read_barrier();
            }
        }
        if (seen) {
            const bool full = lo_all <= kt && hi_all >= kt + KW;
            if (capped || biased || sc == 0.f) {  // (a scale of zero times a masked score is no number)
                const float from = float(pos - kt - 4 * lh);  // this row's distance to the lane's first key
#pragma unroll
                for (int j = 0; j < NSUB; ++j)
#pragma unroll
                    for (int i = 0; i < AV; ++i) {
                        float z = s[j][i] * sc;
                        if (capped) z = tanh_f<kSplit>(z, cap2);
                        s[j][i] = z;
                    }
                if (biased) {
#pragma unroll
                    for (int j = 0; j < NSUB; ++j)
#pragma unroll
                        for (int i = 0; i < AV; ++i)
                            s[j][i] = fmaf(-slope, fabsf(from - float(SUB * j + (NQ == 32 ? (i & 3) + 8 * (i >> 2) : i))), s[j][i]);
                }
                unit = 1.f;
            }
            if (!full) {
#pragma unroll
                for (int j = 0; j < NSUB; ++j)
#pragma unroll
                    for (int i = 0; i < AV; ++i)
                        s[j][i] = uint32_t(kt + key_in(j, i) - see.begin) < see_n ? s[j][i] : -INFINITY;
            }
            float mx = s[0][0];
#pragma unroll
            for (int j = 0; j < NSUB; ++j)
#pragma unroll
                for (int i = 0; i < AV; ++i) mx = fmaxf(mx, s[j][i]);
            mx = rows_max<NQ>(mx);
            mx *= unit;
            if (__any(mx > m + kLag || (m == -INFINITY && mx != m))) {
                const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : exp2_fast(m - mn);
                m = mn;
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < AV; ++i) o[d][i] *= f;
            }
            const float add = m == -INFINITY ? 0.f : kUp - m;
            // P^T operand c, and its share of the sum
            auto weights = [&](int c, v8 &ph, v8 &pl) {
                float p[8], sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // 32 x 32: 8 neighbouring registers; 16 x 16: the 4 of two products
                    const float x = NQ == 32 ? s[c / 2][(8 * c + e) & 15] : s[2 * c + e / 4][e & 3];
                    p[e] = exp2_fast(fmaf(x, unit, add));
                    if constexpr (kSplit) sum += p[e];
                }
                if constexpr (kSplit) {
                    // (no asm here: what it writes, the compiler would not keep apart from a product that still reads)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        ph[e] = _Float16(p[e]);
                        pl[e] = _Float16(p[e] - float(ph[e]));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) ph[e] = C(p[e]);
                    sum = Mx<C>::sum(ph, sum);  // of the rounded weights, which V meets
                }
                return sum;
            };
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                v8 ph, pl;
                l += weights(c, ph, pl);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const v8 v = v_at(c, d);
                    o[d] = Mx<C>::mm(v, ph, o[d]);
                    if constexpr (kSplit) o[d] = Mx<C>::mm(v, pl, o[d]);
                }
            }
        }
        if constexpr (WQ > 1) {
            read_barrier();
        } else if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V has been read
            issue(next, vpool, voff, vin, buf0 + KB);
        }
    }
    raise_status(a.status, bad_page, kStatusBadPage);
    l = rows_sum<NQ>(l);

    T *out = static_cast<T *>(a.out) + int64_t(row) * a.ld_out + int64_t(head) * hd;
    const int64_t rh = int64_t(row) * a.heads + head, part = rh * a.slots + (GROUPS ? 0 : a.gsplits) + split;
    auto put = [&](int e, f32x4 x, float inv) {
        if (whole) {
            store4(out + e, x * inv);
        } else if (a.count) {
            put_far(a.po + part * hd + e, x[0], x[1]);
            put_far(a.po + part * hd + e + 2, x[2], x[3]);
        } else {
            *reinterpret_cast<f32x4 *>(a.po + part * hd + e) = x;
        }
    };
    if constexpr (WK == 1) {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        if (valid) {
            if (!whole && lh == 0) put_far(a.ml + 2 * part, m, l);
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < AV; i += 4) {
                    const int e = NQ * d + (NQ == 32 ? 2 * i + 4 * lh : 4 * lh);
                    if (e < hd) put(e, f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]}, inv);
                }
        }
    } else {
        // the waves' parts side by side in LDS, then every lane adds its 4 dims of a row, in wave order
        constexpr int LDO = HDP + 4;
        float *sm = reinterpret_cast<float *>(smem), *so = sm + 2 * WK * NQ;
        wait_step<0>();
        block_barrier();  // every stream has been read
        if (lh == 0) {
            sm[wk * NQ + col] = m;
            sm[(WK + wk) * NQ + col] = l;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < AV; i += 4) {
                const int e = NQ * d + (NQ == 32 ? 2 * i + 4 * lh : 4 * lh);
                *reinterpret_cast<f32x4 *>(so + (wk * NQ + col) * LDO + e) = f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
            }
        read_barrier();
        float M = -INFINITY, L = 0.f, f[WK];
#pragma unroll
        for (int w = 0; w < WK; ++w) M = fmaxf(M, f[w] = sm[w * NQ + col]);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            f[w] = f[w] == -INFINITY ? 0.f : exp2_fast(f[w] - M);
            L += f[w] * sm[(WK + w) * NQ + col];
        }
        const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
        if (valid) {
            if (!whole && wave == 0 && lh == 0) put_far(a.ml + 2 * part, M, L);
            // lane (col, lh) of wave w takes 4 dims at 4 (w (64 / NQ) + lh), and every 4 x 256 / NQ on
            for (int e = 4 * (wave * (64 / NQ) + lh); e < hd; e += 4 * 256 / NQ) {
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WK; ++w) x += *reinterpret_cast<const f32x4 *>(so + (w * NQ + col) * LDO + e) * f[w];
                put(e, x, inv);
            }
        }
    }
    if (whole || !a.count) return;
    // The last of a row's blocks to come here joins its parts, in slot order whoever it is: they were written past the caches
    // that other XCDs do not see, before the count (the wait). It leaves the count at zero for the next launch.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    read_barrier();
    int32_t *mine = reinterpret_cast<int32_t *>(smem);  // of each query row: parts of the group | own << 16 where it is to join, else 0
    int64_t *which = reinterpret_cast<int64_t *>(smem + 512);
    if (wk == 0 && lh == 0) {
        bool last = false;
        if (valid) {
            last = __hip_atomic_fetch_add(a.count + rh, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
            if (last) __hip_atomic_store(a.count + rh, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        mine[wq * NQ + col] = last ? gruns | (parts - gruns) << 16 : 0;
        which[wq * NQ + col] = rh;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    read_barrier();
    for (int i = int(threadIdx.x) / 32; i < TILE; i += 8)
        if (mine[i]) join_row<T, true>(a, which[i], mine[i] & 0xFFFF, mine[i] >> 16);
}

// The tiles of the groups' shared keys (GN query rows a wave, GW waves beside each other; 0: no groups), then those of the
// sequences' own: one launch, so that neither waits for the other.
template <class T, class C, int HDP, int GN, int GW, int SN, int SW>
__global__ __launch_bounds__(256, 2) void k_paged_attn(PagedAttnArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    int id = blockIdx.x;
    if constexpr (GN > 0) {
        const int n = a.gtiles * a.gsplits * a.c.kv_heads;
        if (id < n) {
            attn_tile<T, C, HDP, GN, GW, true>(a, id, smem);
            return;
        }
        id -= n;
    }
    attn_tile<T, C, HDP, SN, SW, false>(a, id, smem);
}

// The join as a launch of its own, where a block has so many rows that joining them in turn would take longer (a prompt of 512 rows:
// 18 us so, 43 with the last block joining). desc[row] (0:
// written already): parts of the group, own parts 16 bits up. grid x = rows x ceil(heads / 8), block 256.
template <class T>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttnArgs a) {
    const int hb = (a.heads + 7) / 8, row = int(blockIdx.x) / hb, head = int(blockIdx.x) % hb * 8 + int(threadIdx.x) / 32;
    const int32_t r0 = a.b.row_start[0], r1 = a.b.row_start[a.b.seqs], desc = a.desc[row];
    if (row < r0 || row >= r1 || desc == 0 || head >= a.heads) return;
    join_row<T, false>(a, int64_t(row) * a.heads + head, min(desc & 0xFFFF, a.gsplits), min(desc >> 16, a.ssplits));
}

}  // namespace vh
