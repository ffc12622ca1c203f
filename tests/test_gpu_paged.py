"""The paged cache on the device: the append of rows and the attention over pages, against their definitions in 64 bits
(tests/paged.py, which also derives the tolerances). Pages and slots that hold no key are NaN, so a key that is read without
being visible shows."""
import math

import numpy as np
import pytest
import torch

from paged import BF16, CACHE, F16, F32, ROW, Batch, Dev, off

pytestmark = pytest.mark.gpu
TYPES = [F32, F16, BF16]
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}


class Run:
    """A batch's pools and structs on the device; free() gives everything back."""

    def __init__(self, hip, b):
        self.hip, self.b, self.bufs = hip, b, []
        self.k, self.v = self.dev(b.k), self.dev(b.v)
        self.kv, self.batch = b.kv_struct(hip, self.k, self.v), b.batch_struct(hip, self.bufs)

    def dev(self, t):
        self.bufs.append(Dev(self.hip, t))
        return self.bufs[-1]

    def attend(self, q, scale=None, cap=0.0, slopes=None, prefix=None, window=0, shared=None, ld=0, out=None, sync=True):
        b, hip = self.b, self.hip
        qd = b.heads * b.hd
        ld = ld or qd
        wide = torch.full((b.n_rows, ld), 7.0, dtype=ROW[b.wtype])
        wide[:, :qd] = q
        d_q, d_out = self.dev(wide), out or self.dev(torch.full((b.n_rows, ld), 5.0, dtype=ROW[b.wtype]))
        rows = hip.attn_rows(b.wtype, b.heads, d_q, ld, d_out, ld, 1.0 / math.sqrt(b.hd) if scale is None else scale, cap,
                             None if slopes is None else self.dev(slopes), None if prefix is None else self.dev(torch.tensor(prefix, dtype=torch.int32)),
                             window)
        groups = b.groups if shared is None else shared
        if groups:
            starts = [a for a, _, _ in groups] + [groups[-1][1]]
            sh = hip.shared_prefix(len(groups), max(n for _, _, n in groups), self.dev(torch.tensor(starts, dtype=torch.int32)),
                                   self.dev(torch.tensor([n for _, _, n in groups], dtype=torch.int32)))
            hip.attn_shared_dev(self.kv, self.batch, sh, rows)
        else:
            hip.attn_paged_dev(self.kv, self.batch, rows)
        if sync:
            hip.sync()
        got = d_out.get()
        assert bool((got[:, qd:] == 5.0).all()), "columns behind a row"
        used = int(b.first[-1])
        assert bool((got[used:] == 5.0).all()), "rows behind the last sequence"
        return got[:, :qd].reshape(b.n_rows, b.heads, b.hd)

    def free(self):
        for d in self.bufs + [self.k, self.v]:
            d.free()


def check(hip, b, std=2.0, ld=0, **kw):
    r = Run(hip, b)
    try:
        q = b.normal(b.n_rows, b.heads * b.hd).mul(std).to(ROW[b.wtype])
        got = r.attend(q, ld=ld, **kw)
        scale = kw.pop("scale", None) or 1.0 / math.sqrt(b.hd)
        want, tol = b.attend(q, scale, kw.get("cap", 0.0), kw.get("slopes"), kw.get("prefix"), kw.get("window", 0))
        used = int(b.first[-1])
        print(IDS[b.wtype], b.rows[:8], b.lens[:8], "off", off(got[:used], want[:used], tol[:used], b.wtype), flush=True)
        assert off(got[:used], want[:used], tol[:used], b.wtype) <= 1.0
        return got
    finally:
        r.free()


# ---------------------------------------------------------------- append
def turned(x, w, eps, rope, rot, inter):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if rope is None:
        return x
    c, s = rope[..., 0].double()[:, None], rope[..., 1].double()[:, None]
    y = x.clone()
    ia = torch.arange(rot // 2) * (2 if inter else 1)
    ib = ia + (1 if inter else rot // 2)
    y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ib] * c + x[..., ia] * s
    return y


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("hd,heads,kv_heads,rot,inter,norm,nhd,page,gap", [
    (64, 14, 2, 64, False, False, False, 16, 0), (128, 16, 8, 128, False, True, False, 64, 0), (128, 4, 4, 64, True, True, True, 8, 24),
    (80, 5, 1, 40, False, True, False, 32, 8), (96, 6, 3, 96, True, False, True, 128, 0), (40, 3, 1, 8, False, True, False, 16, 0),
    (8, 2, 1, 8, True, True, False, 8, 0), (64, 4, 2, 0, False, True, True, 16, 0), (48, 2, 1, 24, False, True, False, 16, 0), (72, 3, 1, 72, True, True, False, 16, 0)])
def test_append(hip, wtype, hd, heads, kv_heads, rot, inter, norm, nhd, page, gap):
    rows, lens = [5, 0, 1, 17, 3, 2], [5, 9, 40, 17, 200, 1]  # the last has a row at position -1
    b = Batch(rows, lens, wtype, heads, kv_heads, hd, page, seed=hd + rot, pad_rows=3, nhd=nhd, gap=gap)
    qd, kd, ld = heads * hd, kv_heads * hd, heads * hd + 2 * kv_heads * hd + 8
    x = b.normal(b.n_rows, ld).to(ROW[wtype])
    w = [1.0 + 0.1 * b.normal(hd) for _ in range(2)] if norm else [None, None]
    angle = torch.arange(200, dtype=torch.float64)[:, None] * (1.0 / 1e4 ** (torch.arange(max(rot // 2, 1)) / max(rot // 2, 1)))[None]
    rope = torch.stack([angle.cos(), angle.sin()], -1).float() if rot else None
    r = Run(hip, b)
    try:
        dq = r.dev(torch.full((b.n_rows, qd + 16), 5.0, dtype=ROW[wtype]))
        ap = hip.append_rows(wtype, heads, r.dev(x), ld, dq, qd + 16, None if w[0] is None else r.dev(w[0]), None if w[1] is None else r.dev(w[1]),
                             1e-6, None if rope is None else r.dev(rope), 200, rot, inter)
        hip.kv_append_dev(r.kv, r.batch, ap)
        hip.sync()
        got_q, got_k, got_v = dq.get(), r.k.get(), r.v.get()
        want_k, want_v = b.k.clone().double(), b.v.clone().double()
        want_q = torch.full((b.n_rows, qd + 16), 5.0, dtype=torch.float64)
        new = torch.zeros(want_k.shape, dtype=torch.bool)
        for s, (n, total) in enumerate(zip(rows, lens)):
            for i in range(n):
                p, row = total - n + i, int(b.first[s]) + i
                if p < 0:
                    continue
                h = x[row, :qd + 2 * kd].view(1, heads + 2 * kv_heads, hd)
                at = rope[p:p + 1] if rope is not None else None
                want_q[row, :qd] = turned(h[:, :heads], w[0], 1e-6, at, rot, inter).reshape(-1)
                kk, vv = turned(h[:, heads:heads + kv_heads], w[1], 1e-6, at, rot, inter)[0], h[0, heads + kv_heads:].double()
                for g in range(kv_heads):
                    o = b.at(s, p, g)
                    want_k[o:o + hd], want_v[o:o + hd], new[o:o + hd] = kk[g], vv[g], True
        # f32: the norm's sum hd u relative, a few roundings and two products: (hd + 16) u of the largest value
        size = float(want_q[:, :qd].abs().max())
        tol = torch.full((), (hd + 16) * 2.0 ** -24 * size, dtype=torch.float64)
        assert off(got_q, want_q, tol, wtype) <= 1.0
        cache = BF16 if wtype == BF16 else F16
        assert off(got_k[new], want_k[new], tol, cache) <= 1.0
        assert torch.equal(got_v[new], want_v[new].to(CACHE[wtype]))  # copied, rounded once
        same = ~new  # everything else, NaN and gaps among it, bit for bit
        for got, was in ((got_k, b.k), (got_v, b.v)):
            assert torch.equal(got.view(torch.int16)[same], was.view(torch.int16)[same])
    finally:
        r.free()


def test_append_without_q_and_many_sequences(hip):
    # more sequences than one sample of row_start (64) and than 64 x 64 covers; no q wanted
    for S in (1, 63, 64, 65, 700, 5000):
        rows = [1] * S
        b = Batch(rows, [1 + (i * 7) % 30 for i in range(S)], F16, 2, 1, 8, 8, seed=S)
        x = b.normal(S, 4 * 8).to(torch.float16)
        r = Run(hip, b)
        try:
            hip.kv_append_dev(r.kv, r.batch, hip.append_rows(F16, 2, r.dev(x), 32))
            hip.sync()
            k, v = r.k.get(), r.v.get()
            for s in range(0, S, max(1, S // 50)):
                o = b.at(s, b.lens[s] - 1, 0)
                assert torch.equal(k[o:o + 8], x[s, 16:24]) and torch.equal(v[o:o + 8], x[s, 24:32]), s
        finally:
            r.free()


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("hd,heads,kv_heads,rot", [(64, 3, 1, 64), (128, 2, 2, 8), (24, 1, 1, 24)])
def test_append_of_many_rows(hip, wtype, hd, heads, kv_heads, rot):
    """As many rows as fill the chip, a wave each: 2048 and a few more, the last ones behind the last sequence."""
    rows = [1000, 0, 1, 1047, 3]
    b = Batch(rows, [1000, 5, 1, 1050, 3], wtype, heads, kv_heads, hd, 64, seed=7, pad_rows=2)
    qd, kd = heads * hd, kv_heads * hd
    x = b.normal(b.n_rows, qd + 2 * kd).to(ROW[wtype])
    angle = torch.arange(1100, dtype=torch.float64)[:, None] * (1.0 / 1e4 ** (torch.arange(rot // 2) / (rot // 2)))[None]
    rope = torch.stack([angle.cos(), angle.sin()], -1).float()
    w = 1.0 + 0.1 * b.normal(hd)
    r = Run(hip, b)
    try:
        dq = r.dev(torch.full((b.n_rows, qd), 5.0, dtype=ROW[wtype]))
        hip.kv_append_dev(r.kv, r.batch, hip.append_rows(wtype, heads, r.dev(x), qd + 2 * kd, dq, qd, k_norm=r.dev(w), rope=r.dev(rope), rope_len=1100, rot_dim=rot))
        hip.sync()
        got_q, got_k, got_v = dq.get(), r.k.get(), r.v.get()
        pos = torch.cat([torch.arange(l - n, l) for n, l in zip(rows, b.lens)])
        n = pos.numel()
        h = x[:n].view(n, heads + 2 * kv_heads, hd)
        at = rope[pos]
        tol = torch.full((), (hd + 16) * 2.0 ** -24 * 8, dtype=torch.float64)  # values below 8
        assert off(got_q[:n].view(n, heads, hd), turned(h[:, :heads], None, 0, at, rot, False), tol, wtype) <= 1.0
        assert bool((got_q[n:] == 5.0).all())
        want_k = turned(h[:, heads:heads + kv_heads], w, 1e-6, at, rot, False)
        row = 0
        for s, (m, total) in enumerate(zip(rows, b.lens)):
            for i in range(m):
                for g in range(kv_heads):
                    o = b.at(s, total - m + i, g)
                    if i % 97 == 0 or i == m - 1:
                        assert off(got_k[o:o + hd], want_k[row, g], tol, BF16 if wtype == BF16 else F16) <= 1.0, (s, i)
                        assert torch.equal(got_v[o:o + hd], h[row, heads + kv_heads + g].to(CACHE[wtype])), (s, i)
                row += 1
    finally:
        r.free()


# ---------------------------------------------------------------- attention
SHAPES = [(16, 8, 128), (14, 2, 64), (8, 8, 64), (5, 1, 80), (12, 4, 96), (32, 4, 128), (3, 3, 8), (40, 1, 32)]


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
def test_steps(hip, wtype, heads, kv_heads, hd):
    """One row per session: lengths of one key, around pages and tiles, none at all."""
    b = Batch([1, 1, 1, 0, 1, 1, 1, 1, 1], [1, 16, 17, 9, 64, 129, 333, 0, 65], wtype, heads, kv_heads, hd, 16, seed=hd, pad_rows=2)
    got = check(hip, b)
    assert bool((got[int(b.first[7])] == 0).all())  # no key: zeros


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
def test_prompts(hip, wtype, heads, kv_heads, hd):
    """Ragged prompts from empty, with cached keys and with padding in front (rows at negative positions)."""
    b = Batch([7, 130, 0, 1, 65, 6], [7, 130, 4, 70, 100, 4], wtype, heads, kv_heads, hd, 32, seed=hd + 1, pad_rows=1)
    got = check(hip, b, ld=heads * hd + 24)
    assert bool((got[int(b.first[5]):int(b.first[5]) + 2] == 0).all())


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("page,nhd,gap", [(8, False, 0), (8, True, 8), (16, True, 0), (128, False, 40), (1024, True, 0)])
def test_layouts(hip, wtype, page, nhd, gap):
    check(hip, Batch([1, 20, 1], [90, 75, 300], wtype, 4, 2, 64, page, seed=page, nhd=nhd, gap=gap))
    check(hip, Batch([1, 20, 1], [90, 75, 300], wtype, 4, 2, 128, page, seed=page, nhd=nhd, gap=gap))


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("kw", [
    dict(cap=30.0), dict(cap=0.5), dict(slopes=True), dict(prefix=[40, 0, 3, 200]), dict(window=1), dict(window=33), dict(window=5000),
    dict(cap=20.0, slopes=True, prefix=[9, 100, 0, 64], window=70), dict(scale=0.0), dict(scale=-0.3), dict(scale=2.0)], ids=str)
def test_scores(hip, wtype, kw):
    """Cap, distance bias, prefix (longer and shorter than the sequence) and window, steps and prompts in one batch."""
    b = Batch([50, 1, 90, 33], [50, 180, 140, 33], wtype, 6, 2, 64, 16, seed=5)
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = 2.0 ** -torch.arange(1, 7, dtype=torch.float32)
    scale = kw.get("scale")
    r = Run(hip, b)
    try:
        q = b.normal(b.n_rows, 6 * 64).mul(2.0).to(ROW[wtype])
        got = r.attend(q, **kw)
        want, tol = b.attend(q, 0.125 if scale is None else scale, kw.get("cap", 0.0), kw.get("slopes"), kw.get("prefix"), kw.get("window", 0))
        assert off(got, want, tol, wtype) <= 1.0
    finally:
        r.free()


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
def test_hidden_values_do_not_count(hip, wtype):
    """Infinities and NaN in keys and values that a row does not see leave it alone: later keys of its own prompt, keys before
    its window. Rows that do see them are not finite."""
    n = 150
    b = Batch([n], [n], wtype, 4, 2, 64, 16, seed=9)
    bad = {60: math.nan, 61: math.inf, 100: -math.inf, 149: math.nan}
    for j, x in bad.items():
        for h in range(2):
            o = b.at(0, j, h)
            (b.v if j != 100 else b.k)[o + 3] = x
    r = Run(hip, b)
    try:
        q = b.normal(n, 256).to(ROW[wtype])
        for window in (0, 30):
            got = r.attend(q, window=window)
            want, tol = b.attend(q, 0.125, window=window)
            clean = [i for i in range(n) if not any((j <= i and (not window or j > i - window)) for j in bad)]
            assert len(clean) > 40
            assert off(got[clean], want[clean], tol[clean], wtype) <= 1.0
            assert bool((~torch.isfinite(got[60])).any()) and bool((~torch.isfinite(got[149])).any())
    finally:
        r.free()


def test_one_key_far_above_the_rest(hip):
    """Weights that underflow, and a row whose largest score comes last: the running maximum has to move everything before it."""
    for wtype in TYPES:
        b = Batch([1, 3], [700, 300], wtype, 2, 1, 64, 16, seed=3)
        q = torch.zeros(b.n_rows, 128)
        q[:, 0] = 1.0
        q[:, 64] = 1.0
        for s, n in enumerate(b.lens):
            for j in range(n):
                b.k[b.at(s, j, 0):b.at(s, j, 0) + 64] = 0
                b.k[b.at(s, j, 0)] = float(j) if s == 0 else float(300 - j) * 0.25
        r = Run(hip, b)
        try:
            q = q.to(ROW[wtype])
            got = r.attend(q, scale=1.0)
            want, tol = b.attend(q, 1.0)
            assert off(got, want, tol, wtype) <= 1.0
        finally:
            r.free()


@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
def test_flat_scores_of_many_keys(hip, wtype):
    """All scores but one alike and far below it, so many that together they weigh: small weights keep their share."""
    n = 5000
    b = Batch([1], [n], wtype, 1, 1, 8, 64, seed=4)
    b.v[~torch.isnan(b.v)] = 0.0
    for j in range(n):
        o = b.at(0, j, 0)
        b.k[o:o + 8] = 0
        b.k[o] = 0.0 if j == 77 else -8.75
        b.v[o] = 0.0 if j == 77 else 1.0
    r = Run(hip, b)
    try:
        q = torch.zeros(1, 8)
        q[0, 0] = 1.0
        q = q.to(ROW[wtype])
        got = r.attend(q, scale=1.0)
        want, tol = b.attend(q, 1.0)
        assert off(got, want, tol, wtype) <= 1.0
    finally:
        r.free()


def test_f32_rows_keep_their_bits(hip):
    """What f16 halves without their low parts would lose: scores that differ by the 13th bit of a query, and weights of few
    keys with small scores, where the bound is a few 2^-22."""
    b = Batch([1], [2], F32, 1, 1, 8, 16, seed=1)
    for j in range(2):
        b.k[b.at(0, j, 0):b.at(0, j, 0) + 8] = 0
        b.k[b.at(0, j, 0) + j] = 2048.0
        b.v[b.at(0, j, 0):b.at(0, j, 0) + 8] = float(j)
    r = Run(hip, b)
    try:
        q = torch.zeros(1, 8)
        q[0, 0], q[0, 1] = 1.0 + 2.0 ** -13, 1.0
        got = float(r.attend(q, scale=1.0)[0, 0, 0])
        assert abs(got - 1.0 / (1.0 + math.exp(0.25))) < 1e-3  # 0.5 without the low half
    finally:
        r.free()
    check(hip, Batch([1, 9], [20, 9], F32, 2, 1, 8, 16, seed=2), std=0.02)
    check(hip, Batch([1, 40], [50, 40], F32, 2, 1, 64, 16, [(0, 1, 32)], seed=3), std=0.002)


# ---------------------------------------------------------------- shared prefixes
@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("heads,kv_heads,hd", [(16, 8, 128), (14, 2, 64), (5, 1, 80)])
@pytest.mark.parametrize("rows,lens,groups", [
    ([1] * 8, [130, 140, 129, 200, 131, 150, 133, 190], [(0, 8, 128)]),
    ([1] * 5, [64, 70, 65, 90, 20], [(1, 4, 64)]),                                # outside every group: the first and the last
    ([3, 1, 20, 1, 2, 1, 0], [40, 90, 70, 300, 301, 20, 320], [(0, 3, 32), (3, 7, 272)]),  # the second is shorter than what its group shares
    ([1] * 3, [40, 50, 60], [(0, 3, 0)]), ([1, 4], [100, 104], [(0, 1, 48), (1, 2, 96)]),
    ([1] * 70, [40 + i for i in range(70)], [(0, 30, 40), (30, 31, 16), (31, 70, 64)])])
def test_shared(hip, wtype, heads, kv_heads, hd, rows, lens, groups):
    check(hip, Batch(rows, lens, wtype, heads, kv_heads, hd, 16, groups, seed=len(rows), pad_rows=1))


def test_shared_with_masks(hip):
    for wtype in TYPES:
        for kw in (dict(window=50), dict(prefix=[100, 20, 0, 7]), dict(cap=10.0, slopes=2.0 ** -torch.arange(4.0), window=100)):
            check(hip, Batch([2, 1, 30, 1], [150, 140, 170, 100], wtype, 4, 2, 64, 16, [(0, 4, 96)], seed=8), **kw)


def test_shared_part_of_a_page(hip):
    # 20 shared keys of pages of 16: the second page of the others holds its own keys from slot 4 on
    for wtype in TYPES:
        check(hip, Batch([1, 1, 2], [60, 25, 21], wtype, 4, 2, 64, 16, [(0, 3, 20)], seed=8))


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("wtype", TYPES, ids=IDS.get)
def test_a_server_s_steps(hip, wtype):
    """Prompts, then steps, appended and attended in place, two voices: every step's outputs against the definition over the
    cache as it then is."""
    heads, kv_heads, hd, page = 6, 2, 64, 16
    qd, kd = heads * hd, kv_heads * hd
    final = [80, 71, 95, 60]
    groups = [(0, 2, 32), (2, 4, 48)]
    b = Batch([1] * 4, final, wtype, heads, kv_heads, hd, page, groups, seed=12)
    # the whole shared prefixes are there; each session's own keys begin as NaN
    for pool in (b.k, b.v):
        for s in range(4):
            for j in range(b.shared[s], final[s]):
                for h in range(kv_heads):
                    pool[b.at(s, j, h):b.at(s, j, h) + hd] = math.nan
    r = Run(hip, b)
    angle = torch.arange(128, dtype=torch.float64)[:, None] * (1.0 / 1e4 ** (torch.arange(32) / 32.0))[None]
    rope = torch.stack([angle.cos(), angle.sin()], -1).float()
    d_rope = r.dev(rope)
    lens = [s + 1 for s in b.shared]
    try:
        for step in range(12):
            rows = [min(17 if step == 0 else 1 + (step + s) % 3, final[s] - (lens[s] - 1)) for s in range(4)]
            rows = [max(0, n) for n in rows]
            lens = [l - 1 + n for l, n in zip(lens, rows)]
            b.rows, b.lens, b.n_rows = rows, lens, sum(rows)
            b.first = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
            if not b.n_rows:
                break
            r.batch = b.batch_struct(hip, r.bufs)
            x = b.normal(b.n_rows, qd + 2 * kd).to(ROW[wtype])
            dq = r.dev(torch.zeros(b.n_rows, qd, dtype=ROW[wtype]))
            hip.kv_append_dev(r.kv, r.batch, hip.append_rows(wtype, heads, r.dev(x), qd + 2 * kd, dq, qd, rope=d_rope, rope_len=128, rot_dim=hd))
            sh = hip.shared_prefix(2, 48, r.dev(torch.tensor([0, 2, 4], dtype=torch.int32)), r.dev(torch.tensor([32, 48], dtype=torch.int32)))
            hip.attn_shared_dev(r.kv, r.batch, sh, hip.attn_rows(wtype, heads, dq, qd, dq, qd, 0.125))  # in place
            hip.sync()
            b.k, b.v = r.k.get(), r.v.get()
            q = torch.zeros(b.n_rows, heads, hd, dtype=torch.float64)
            for s in range(4):
                for i in range(rows[s]):
                    p, row = lens[s] - rows[s] + i, int(b.first[s]) + i
                    q[row] = turned(x[row, :qd].view(1, heads, hd), None, 0, rope[p:p + 1], hd, False)[0]
            want, tol = b.attend(q.float().to(ROW[wtype]).view(b.n_rows, -1), 0.125)
            # the queries' own rounding (f32: their products' 4 u, 16 bits: half a step, of a row in few cases) moves a score by
            # that share of sum |q k|, at most 8 * |q| |k| / 8 here
            slack = {F32: 2.0 ** -20, F16: 0.0, BF16: 0.0}[wtype] * 64
            got = dq.get().view(b.n_rows, heads, hd)
            if wtype == F32:
                assert off(got, want, tol + slack, wtype) <= 1.0, step
            else:  # a query on a rounding border may go the other way: one step of one of 64 products
                assert off(got, want, tol + 4 * {F16: 2.0 ** -10, BF16: 2.0 ** -7}[wtype], wtype) <= 1.0, step
            lens = [l + 1 for l in lens]
    finally:
        r.free()


def test_same_bits_again(hip):
    """A call's bits do not depend on the calls before it, other shapes among them."""
    for wtype in TYPES:
        a = Batch([1] * 6, [900, 30, 444, 71, 800, 2], wtype, 8, 2, 64, 16, [(0, 6, 0)], seed=1)
        c = Batch([70, 1], [300, 999], wtype, 8, 2, 64, 16, seed=2)
        ra, rc = Run(hip, a), Run(hip, c)
        try:
            qa, qc = a.normal(6, 512).to(ROW[wtype]), c.normal(71, 512).to(ROW[wtype])
            first = (ra.attend(qa), rc.attend(qc))
            for _ in range(3):
                assert torch.equal(rc.attend(qc), first[1])
                assert torch.equal(ra.attend(qa), first[0])
        finally:
            ra.free()
            rc.free()


# ---------------------------------------------------------------- far offsets, bad contents
def test_offsets_past_32_bits(hip):
    """Pages whose values lie more than 4 GiB (2^31 elements) into the pool."""
    stride, page, hd = (1 << 30) + 64, 16, 64
    b = Batch([1, 20], [40, 30], F16, 2, 1, hd, page, seed=6)
    perm = [0, 2, 1]  # the pages in use, in a pool of three pages a GiB of elements apart
    b.table[:] = -1
    b.table[0, :1], b.table[1, :2] = 2, [0, 1]
    b.lens, b.rows, b.n_rows = [16, 30], [1, 20], 21
    pools = []
    try:
        for _ in range(2):
            pools.append(hip.DevBuf((2 * stride + page * hd) * 2))
        b.page_stride, b.pages = stride, 3
        data = [[b.normal(page, hd).half() for _ in range(3)] for _ in range(2)]
        for pool, pages in zip(pools, data):
            for i, t in enumerate(pages):
                hip._check(hip.lib().voxhip_memcpy_h2d(pool.ptr + i * stride * 2, hip._p(t.numpy()), t.numel() * 2), "memcpy_h2d")
        bufs = []
        batch = b.batch_struct(hip, bufs)
        kv = hip.paged_kv(pools[0], pools[1], F16, 3, page, 1, hd, stride, page * hd, hd)
        x = b.normal(21, 4 * hd).half()
        dq, dx, out = Dev(hip, torch.zeros(21, 2 * hd).half()), Dev(hip, x), Dev(hip, torch.zeros(21, 2 * hd).half())
        bufs += [dq, dx, out]
        hip.kv_append_dev(kv, batch, hip.append_rows(F16, 2, dx, 4 * hd, dq, 2 * hd))
        hip.attn_paged_dev(kv, batch, hip.attn_rows(F16, 2, dq, 2 * hd, out, 2 * hd, 0.125))
        hip.sync()
        where = [(2, 15)] + [(0 if p < 16 else 1, p % 16) for p in range(10, 30)]
        for row, (pg, slot) in enumerate(where):
            data[0][pg][slot], data[1][pg][slot] = x[row, 2 * hd:3 * hd], x[row, 3 * hd:]
        k = [torch.cat([data[j][2]]) for j in range(2)], [torch.cat(data[j][:2])[:30] for j in range(2)]
        got = out.get().double().view(21, 2, hd)
        for row in range(21):
            kk, vv = k[0 if row == 0 else 1]
            n = 16 if row == 0 else 10 + row
            z = x[row, :2 * hd].view(2, hd).double() @ kk[:n].double().T * 0.125
            want = torch.softmax(z, -1) @ vv[:n].double()
            assert float((got[row] - want).abs().max()) < 2.0 ** -10 * 4, row
        for f in bufs:
            f.free()
    finally:
        for p in pools:
            p.free()


def test_bad_tables_are_reported(hip):
    """A table entry outside the pool, lengths and rows outside the batch: nothing outside is touched, sync fails, and the next
    call is as if nothing had been."""
    b = Batch([1, 4], [60, 90], F32, 4, 2, 64, 16, seed=2)
    good = b.table.copy()
    q = b.normal(5, 256)
    r = Run(hip, b)
    try:
        before = r.attend(q)
        for bad in (-1, b.pages, 1 << 30, -(1 << 31)):
            b.table[0, 1] = bad
            r.batch = b.batch_struct(hip, r.bufs)
            with pytest.raises(hip.VoxHipError, match="page table entry"):
                r.attend(q)
            b.table[0, 3] = bad  # the page a row is written to
            b.table[0, 1] = good[0, 1]
            r.batch = b.batch_struct(hip, r.bufs)
            hip.kv_append_dev(r.kv, r.batch, hip.append_rows(F32, 4, r.dev(b.normal(5, 512)), 512))
            with pytest.raises(hip.VoxHipError, match="page table entry"):
                hip.sync()
            b.table[:] = good
        for lens, first in (([1 << 20, 90], None), ([60, -5], None), (None, [0, 9, 5]), (None, [-3, 1, 5]), (None, [0, 1, 9])):
            b.lens, keep, was = lens or b.lens, b.lens, b.first
            b.first = np.array(first or b.first, np.int32)
            batch = b.batch_struct(hip, r.bufs)
            batch.max_rows, batch.max_len = 4, 90
            b.lens, b.first = keep, was
            rows = hip.attn_rows(F32, 4, r.dev(q), 256, r.dev(torch.zeros(5, 256)), 256, 0.125)
            hip.attn_paged_dev(r.kv, batch, rows)
            with pytest.raises(hip.VoxHipError, match="row_start, len"):
                hip.sync()
            hip.kv_append_dev(r.kv, batch, hip.append_rows(F32, 4, r.dev(b.normal(5, 512)), 512))
            with pytest.raises(hip.VoxHipError, match="row_start, len|page table"):
                hip.sync()
        # a position behind the rope table
        batch = b.batch_struct(hip, r.bufs)
        hip.kv_append_dev(r.kv, batch, hip.append_rows(F32, 4, r.dev(b.normal(5, 512)), 512, rope=r.dev(torch.zeros(50, 64)), rope_len=50, rot_dim=64))
        with pytest.raises(hip.VoxHipError, match="rope table"):
            hip.sync()
        r.k.buf.upload(b.k.numpy())
        r.v.buf.upload(b.v.numpy())
        r.batch = b.batch_struct(hip, r.bufs)
        assert torch.equal(r.attend(q), before)
    finally:
        r.free()


def test_no_room_for_the_parts(hip):
    """The attention's workspace refused by the memory limit: the call fails, the next one with room runs."""
    n = 20000  # rows of 2 heads in 2 slots: 21 MB of parts, more than any other test here needs
    b = Batch([1, 1], [40, 44], F16, 2, 1, 64, 16, [(0, 2, 32)], seed=3)
    r = Run(hip, b)
    big = r.dev(torch.zeros(n, 128, dtype=torch.float16))
    batch = b.batch_struct(hip, r.bufs)
    batch.rows = n
    sh = hip.shared_prefix(1, 32, r.dev(torch.tensor([0, 2], dtype=torch.int32)), r.dev(torch.tensor([32], dtype=torch.int32)))
    rows = hip.attn_rows(F16, 2, big, 128, big, 128, 0.125)
    q = b.normal(2, 128).half()
    before = r.attend(q)
    try:
        hip.lib().voxhip_set_vram_limit(1)  # less than any weight copies of other tests' models, which would give way, can make room for
        with pytest.raises(hip.VoxHipError, match="VRAM limit"):
            hip.attn_shared_dev(r.kv, batch, sh, rows)
        hip.lib().voxhip_set_vram_limit(0)
        assert torch.equal(r.attend(q), before)  # the old workspace is gone; its like is made again
        hip.attn_shared_dev(r.kv, batch, sh, rows)
        hip.sync()
    finally:
        hip.lib().voxhip_set_vram_limit(0)
        r.free()


def test_range_of_f32_queries(hip):
    """A query beyond the f16 range, which the split of f32 rows cannot hold, is reported as elsewhere in the library."""
    b = Batch([1], [20], F32, 2, 1, 64, 16, seed=2)
    q = b.normal(1, 128)
    q[0, 5] = 7e4
    r = Run(hip, b)
    try:
        with pytest.raises(hip.VoxHipError, match="f16 range"):
            r.attend(q)
        r.attend(b.normal(1, 128))
    finally:
        r.free()
