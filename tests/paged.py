"""Ragged batches on a paged cache for the tests: their inputs, the definition in 64 bits, and how far 32-bit arithmetic on
matrix cores may be from it. Pages that no key was written to, and the slots behind a sequence's last key, hold NaN."""
import math

import numpy as np
import torch

F32, F16, BF16 = 0, 1, 2
ROW = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
CACHE = {F32: torch.float16, F16: torch.float16, BF16: torch.bfloat16}


def raw(t):
    """A CPU tensor's bytes as numpy has them (bf16 as uint16)."""
    t = t.contiguous()
    return t.view(torch.int16).numpy() if t.dtype == torch.bfloat16 else t.numpy()


class Dev:
    """A CPU tensor in a device buffer of the library."""

    def __init__(self, hip, t):
        self.hip, self.dtype, self.shape = hip, t.dtype, tuple(t.shape)
        self.buf = hip.DevBuf(max(16, t.numel() * t.element_size()))
        self.ptr = self.buf.ptr
        if t.numel():
            self.buf.upload(raw(t))

    def get(self):
        d = torch.int16 if self.dtype == torch.bfloat16 else self.dtype
        a = self.buf.download(self.shape, torch.empty(0, dtype=d).numpy().dtype)
        t = torch.from_numpy(a)
        return t.view(torch.bfloat16) if self.dtype == torch.bfloat16 else t

    def free(self):
        self.buf.free()


class Batch:
    """rows / lens of every sequence, pages of a shuffled pool. groups: (first, behind last, shared keys): those sequences
    begin with the pages of the first; their own table entries for whole shared pages name no page."""

    def __init__(self, rows, lens, wtype=F32, heads=4, kv_heads=2, hd=64, page=16, groups=(), seed=0, pad_rows=0, nhd=False, gap=0):
        self.rows, self.lens, self.groups = list(rows), list(lens), list(groups)
        self.wtype, self.heads, self.kv_heads, self.hd, self.page = wtype, heads, kv_heads, hd, page
        self.g = torch.Generator().manual_seed(seed)
        S = len(self.rows)
        self.n_rows = sum(self.rows) + pad_rows
        self.first = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.ld = max(1, max(-(-n // page) for n in self.lens)) + 1
        need = sum(-(-n // page) for n in self.lens) + 3
        order = torch.randperm(need, generator=self.g).tolist()
        self.table = np.full((S, self.ld), -1, np.int32)
        self.lead = list(range(S))
        self.shared = [0] * S
        for a, b, n in self.groups:
            for s in range(a, b):
                self.lead[s], self.shared[s] = a, n
        at = 0
        for s in range(S):
            for i in range(-(-self.lens[s] // page)):
                if self.lead[s] != s and (i + 1) * page <= self.shared[s]:
                    continue
                self.table[s, i] = order[at]
                at += 1
        self.pages = need
        self.shape = (need, page, kv_heads, hd) if nhd else (need, kv_heads, page, hd)
        self.nhd = nhd
        # strides in elements; gap: between pages
        inner = kv_heads * page * hd
        self.page_stride = inner + gap
        self.gap = gap
        self.head_stride, self.pos_stride = (hd, kv_heads * hd) if nhd else (page * hd, hd)
        self.k, self.v = self._pool(), self._pool()

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, dtype=torch.float32)

    def _pool(self):
        """A pool whose written slots are N(0, 1), the rest NaN."""
        p = torch.full((self.pages * self.page_stride,), math.nan, dtype=CACHE[self.wtype])
        for s, n in enumerate(self.lens):
            for j in range(n):
                if self.lead[s] != s and j < self.shared[s]:
                    continue
                for h in range(self.kv_heads):
                    o = self.at(s, j, h)
                    p[o:o + self.hd] = self.normal(self.hd).to(p.dtype)
        return p

    def at(self, s, j, h):
        src = self.lead[s] if j < self.shared[s] else s
        return int(self.table[src, j // self.page]) * self.page_stride + h * self.head_stride + (j % self.page) * self.pos_stride

    def keys(self, pool, s, h):
        n = self.lens[s]
        idx = torch.tensor([self.at(s, j, h) for j in range(n)], dtype=torch.int64).view(-1, 1) + torch.arange(self.hd)
        return pool[idx.view(-1)].view(n, self.hd)

    def kv_struct(self, hip, k, v):
        return hip.paged_kv(k, v, BF16 if self.wtype == BF16 else F16, self.pages, self.page, self.kv_heads, self.hd, self.page_stride,
                            self.head_stride, self.pos_stride)

    def batch_struct(self, hip, bufs):
        bufs += [Dev(hip, torch.from_numpy(self.first)), Dev(hip, torch.tensor(self.lens, dtype=torch.int32)),
                 Dev(hip, torch.from_numpy(self.table))]
        return hip.paged_batch(len(self.rows), self.n_rows, max(1, max(self.rows)), max(1, max(self.lens)), *bufs[-3:], self.ld)

    def spans(self, s, prefix=None, window=0):
        """(begin, end) of the visible keys of every row of sequence s."""
        n, total, out = self.rows[s], self.lens[s], []
        for i in range(n):
            p = total - n + i
            if p < 0:
                out.append((0, 0))
                continue
            b = max(0, p - window + 1) if window else 0
            out.append((b, max(b, min(total, max(p + 1, prefix[s] if prefix is not None else 0)))))
        return out

    def attend(self, q, scale, cap=0.0, slopes=None, prefix=None, window=0):
        """The definition in 64 bits, and per row and head a bound on what the kernels' arithmetic may be off by."""
        H, G, hd = self.heads, self.kv_heads, self.hd
        out = torch.zeros((self.n_rows, H, hd), dtype=torch.float64)
        tol = torch.zeros((self.n_rows, H, 1), dtype=torch.float64)
        q = q.double().view(self.n_rows, H, hd)
        for s in range(len(self.rows)):
            if not self.rows[s]:
                continue
            for g in range(G):
                k, v = self.keys(self.k, s, g).double(), self.keys(self.v, s, g).double()
                for i, (b, e) in enumerate(self.spans(s, prefix, window)):
                    if b >= e:
                        continue
                    r, p = int(self.first[s]) + i, self.lens[s] - self.rows[s] + i
                    hs = slice(g * (H // G), (g + 1) * (H // G))
                    z = q[r, hs] @ k[b:e].T * scale
                    size = (q[r, hs].abs() @ k[b:e].abs().T * abs(scale)).amax(-1, keepdim=True)
                    if cap:
                        z = cap * torch.tanh(z / cap)
                    bias = 0.0
                    if slopes is not None:
                        d = (torch.arange(b, e, dtype=torch.float64) - p).abs()
                        z = z - slopes[hs].double()[:, None] * d
                        bias = (slopes[hs].double()[:, None] * d).amax(-1, keepdim=True)
                    w = torch.softmax(z, -1)
                    out[r, hs] = w @ v[b:e]
                    tol[r, hs] = self.bound(e - b, size, bias, cap) * v[b:e].abs().max()
        return out, tol

    def bound(self, n, size, bias, cap):
        """Of the weighted mean, in units of max |v|. u = 2^-24. A score of products summing to `size` in absolute value is
        off by (hd + 4) u size for f32 sums in any order, 2^-22 size more where f32 queries go as two f16 halves; cap's tanh
        by 4 u cap, scaling and bias by 4 u (size + bias). A score off by d makes weights off by 2 d after division; weights
        rounded to the rows' 16 bits add half a step (f32 rows: two halves, 2^-22), sums of n terms n u each, twice."""
        u = 2.0 ** -24
        d = (self.hd + 4) * u * size + 4 * u * (size + bias) + 4 * u * cap + (2.0 ** -22 * size if self.wtype == F32 else 0.0)
        return 2 * d + 2 * n * u + {F32: 2.0 ** -22, F16: 2.0 ** -11, BF16: 2.0 ** -8}[self.wtype] + 8 * u


def off(got, want, tol, wtype):
    """The largest error in units of what is allowed: tol, and half a step of the rows' type."""
    half = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[wtype]
    tiny = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}[wtype]
    err = (got.double() - want).abs()
    allowed = tol + half * want.abs() * (1 + 2.0 ** -10) + half * tol + tiny
    bad = ~(err <= allowed)  # NaN counts
    return float("inf") if bool(torch.isnan(err).any()) else float((err / allowed.clamp_min(1e-300)).max()) if err.numel() else (1.0 if bool(bad.any()) else 0.0)
