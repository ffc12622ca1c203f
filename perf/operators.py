"""What a speech server asks of the paged key/value cache, as cases that can be timed and compared.

A server speaks many texts in a few voices at once. Its sessions keep their keys and values in pages of one pool: `append`
rotates a step's new rows and writes them there, `attend` is the attention of those rows (one per session while it
speaks, a whole prompt at its begin), and `shared` the same where groups of sessions begin with the same voice prompt.

A ragged batch is described by row_start [seqs + 1] (the rows of sequence s), len [seqs] (its keys, those of this step
among them) and pages [seqs][page_ld] (its page table): row i of a sequence of n rows stands at position len - n + i. A
page holds [kv_heads][page][head_dim] keys, or values.

`own` picks the library's operators; else `run` computes them in elementary torch operations in 32 bits. `exact` restates
them in 64 bits, sequence by sequence.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def _case(name, kind, seqs, rows, past, act="f32", heads=(16, 8), hd=128, page=16, **more):
    c = {"kind": kind, "seqs": seqs, "rows": rows, "past": past, "act": act, "heads": heads[0], "kv_heads": heads[1], "hd": hd,
         "page": page, "cap": 0.0, "slopes": False, "prefix": 0, "window": 0, "groups": 0, "shared": 0, "rot": hd,
         "interleaved": False, "norm": True}
    c.update(more)
    if name:
        c["name"] = name
    return c


LM = {"heads": (14, 2), "hd": 64}  # the CosyVoice2 LM's heads; the Qwen3-TTS talker's are the default


def listed():
    return [
        # one step of eight talker sessions: as little as there is, a launch's own time
        _case("append_step_8", "append", 8, 1, 1024),
        # the prompts of 24 LM sessions that begin together, 1 to 512 rows each, no norm of q and k
        _case("append_prompts_lm", "append", 24, 512, 0, page=64, norm=False, **LM),
        # 16-bit rows of long prompts, half of each head rotated, neighbours paired, behind cached keys
        _case("append_prompts_bf16", "append", 16, 1024, 2000, act="bf16", page=128, rot=64, interleaved=True),
        # one token of one session 512 tokens into an utterance: the smallest call, latency
        _case("step_1", "attend", 1, 1, 512),
        # eight sessions of a talker under load
        _case("step_8", "attend", 8, 1, 1024),
        # 64 LM sessions of very different lengths in 16 bits: the cache's bytes
        _case("step_64_lm_f16", "attend", 64, 1, 8192, act="f16", page=64, **LM),
        # the LM's prompt before it generates
        _case("prompt_lm_512", "attend", 1, 512, 0, page=64, **LM),
        # prompts of 24 sessions, capped scores, a distance bias, the first 100 positions seen by every row
        _case("prompts_capped_bf16", "attend", 24, 700, 0, act="bf16", page=32, cap=30.0, slopes=True, prefix=100),
        # a chunk of a long text behind 30000 cached keys: the most arithmetic
        _case("chunk_long_f16", "attend", 1, 2048, 30000, act="f16", page=128),
        # eight sentences read in one voice, each with a few tokens of its own behind the voice prompt
        _case("voice_8", "shared", 8, 1, 150, groups=1, shared=368),
        # 64 sentences behind a long prompt
        _case("voice_64_bf16", "shared", 64, 1, 600, act="bf16", page=64, groups=1, shared=8192),
        # three voices of different prompts, a few rows a session, capped scores
        _case("voices_3_lm_f16", "shared", 24, 12, 300, act="f16", cap=50.0, groups=3, shared=2048, **LM),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(("append", "attend", "attend", "attend", "shared", "shared"))
    more = {"act": rng.choice(("f32", "f16", "bf16")), "page": rng.choice((16, 32, 64, 128))}
    more.update(rng.choice((LM, {"heads": (16, 8), "hd": 128}, {"heads": (8, 8), "hd": 64}, {"heads": (32, 4), "hd": 128},
                            {"heads": (5, 1), "hd": 80}, {"heads": (12, 4), "hd": 96})))
    if kind == "append":
        hd = more["hd"]
        more.update(rot=rng.choice((hd, hd, hd // 2)), interleaved=rng.random() < 0.3, norm=rng.random() < 0.6)
        return _case("", kind, size(1, 64), size(1, 500), rng.choice((0, size(1, 4000))), **more)
    if rng.random() < 0.4:
        more.update(rng.choice(({"cap": 30.0}, {"cap": 50.0}, {"slopes": True}, {"cap": 20.0, "slopes": True})))
    if kind == "shared":
        return _case("", kind, size(2, 64), rng.choice((1, 1, size(2, 24))), size(1, 1500), groups=rng.choice((1, 1, 2, 3)),
                     shared=size(32, 8000), **more)
    if rng.random() < 0.5:  # a step
        more["window"] = rng.choice((0, 0, 0, size(16, 2000)))
        return _case("", kind, size(1, 64), 1, size(3, 8000), **more)
    more.update(prefix=rng.choice((0, 0, size(2, 200))), window=rng.choice((0, 0, 0, size(16, 1000))))
    seqs = size(1, 24)
    return _case("", kind, seqs, size(2, 6000 // seqs), rng.choice((0, 0, size(1, 24000 // seqs))), **more)


# ---------------------------------------------------------------- shapes: what a case's sizes stand for
def _lengths(c):
    """Rows and keys of every sequence, and the groups' (first sequence, shared keys): from the case's sizes alone. One
    sequence has the full sizes; of several the first has, the others are spread below."""
    r = random.Random("%d %d %d %d" % (c["seqs"], c["rows"], c["past"], c["shared"]))
    rows = [c["rows"]] + [r.randint(1, c["rows"]) for _ in range(c["seqs"] - 1)]
    past = [c["past"]] + [r.randint(c["past"] // 8, c["past"]) for _ in range(c["seqs"] - 1)]
    groups = []
    if c["groups"]:
        n = min(c["groups"], c["seqs"])
        cuts = [0] + sorted(r.sample(range(1, c["seqs"]), n - 1)) + [c["seqs"]]
        pages = max(1, c["shared"] // c["page"])
        groups = [(cuts[i], cuts[i + 1], c["page"] * (pages if i == 0 else r.randint(1, pages))) for i in range(n)]
        for a, b, shared in groups:
            past[a:b] = [p + shared for p in past[a:b]]
    return rows, [p + n for p, n in zip(past, rows)], groups


def work(case):
    c = case
    rows, keys, groups = _lengths(c)
    n, size, cache = sum(rows), (4 if c["act"] == "f32" else 2), 2
    qd, kd = c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
    if c["kind"] == "append":
        return {"bytes": n * ((qd + 2 * kd + qd) * size + 2 * kd * cache + c["rot"] * 4), "flops": n * (qd + kd) * (3 + 4 * c["norm"])}
    pairs = seen = 0  # (row, key) pairs that are visible, and keys that any row sees
    for new, total in zip(rows, keys):
        low = total
        for p in range(total - new, total):
            lo = max(0, p - c["window"] + 1) if c["window"] else 0
            pairs += max(0, min(total, max(p + 1, c["prefix"])) - lo)
            low = min(low, lo)
        seen += total - low
    seen -= sum((b - a - 1) * shared for a, b, shared in groups)
    return {"bytes": 2 * n * qd * size + 2 * seen * kd * cache, "flops": 4 * pairs * qd}


# ---------------------------------------------------------------- inputs
class _State:
    """A step's batch and buffers, as a server keeps them."""

    def __init__(self, **kw):
        self.__dict__.update(kw)
        self.call = None  # the library's description of them, made by the first call


class _Buf:
    """A torch tensor as a device buffer of the binding."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(c, keys, groups, g):
    """Page tables over a shuffled pool; the sequences of a group begin with the pages of its first. A few pages stay free."""
    counts = torch.tensor([-(-k // c["page"]) for k in keys])
    ld = int(counts.max())
    common = torch.zeros(len(keys), dtype=torch.int64)
    lead = torch.arange(len(keys))
    for a, b, shared in groups:
        common[a + 1:b] = shared // c["page"]
        lead[a:b] = a
    fresh = counts - common
    starts = torch.cumsum(fresh, 0) - fresh
    n = int(fresh.sum()) + 5
    order = torch.randperm(n, generator=g)
    at = torch.arange(ld)[None, :]
    index = starts[:, None] + at - common[:, None]
    table = torch.where(at < counts[:, None], order[index.clamp(0, n - 1)], torch.zeros((), dtype=torch.int64))
    table = torch.where(at < common[:, None], table[lead], table)
    return n, ld, table.to(torch.int32).to(DEV)


def prepare(case, seed):
    c = case
    rows, keys, groups = _lengths(c)
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gd, device=DEV) * std
    act = TYPES[c["act"]]
    cache = torch.bfloat16 if c["act"] == "bf16" else torch.float16
    qd, kd = c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
    n = sum(rows)
    n_pages, page_ld, table = _tables(c, keys, groups, g)
    shape = (n_pages, c["kv_heads"], c["page"], c["hd"])
    st = _State(c=c, rows=n, max_rows=max(rows), max_len=max(keys), n_pages=n_pages, page_ld=page_ld, pages=table,
                row_start=_ints([sum(rows[:i]) for i in range(len(rows) + 1)]), len=_ints(keys),
                k=normal(*shape).to(cache), v=normal(*shape).to(cache))
    if c["kind"] == "append":
        half = c["rot"] // 2
        inv = 1.0 / 1e6 ** (torch.arange(half, dtype=torch.float64, device=DEV) / half)
        angle = torch.arange(st.max_len, dtype=torch.float64, device=DEV)[:, None] * inv
        st.rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        st.qkv = normal(n, qd + 2 * kd).to(act)
        st.q = torch.zeros((n, qd), dtype=act, device=DEV)
        st.qn, st.kn = (1.0 + normal(c["hd"], std=0.02), 1.0 + normal(c["hd"], std=0.02)) if c["norm"] else (None, None)
    else:
        st.q = normal(n, qd, std=2.0).to(act)
        st.out = torch.zeros((n, qd), dtype=act, device=DEV)
        st.slopes = 2.0 ** (-8.0 * (torch.arange(c["heads"], device=DEV) + 1) / c["heads"]) if c["slopes"] else None
        st.prefix = _ints([min(c["prefix"], k) for k in keys]) if c["prefix"] else None
        st.group_start = _ints([a for a, _, _ in groups] + [c["seqs"]]) if groups else None
        st.group_len = _ints([shared for _, _, shared in groups]) if groups else None
        st.groups, st.max_shared = len(groups), max([shared for _, _, shared in groups], default=0)
    return st


# ---------------------------------------------------------------- the operators: the library's, and their plain form
def run(state):
    if own:
        return _own(state)
    return _append(state) if state.c["kind"] == "append" else _attend(state)


def _own(st):
    from vox_amd import voxhip as vh
    c = st.c
    if st.call is None:
        vh.init("hip:0")
        wt = {"f32": vh.F32, "f16": vh.F16, "bf16": vh.BF16}[c["act"]]
        kv = vh.paged_kv(_Buf(st.k), _Buf(st.v), vh.BF16 if c["act"] == "bf16" else vh.F16, st.n_pages, c["page"], c["kv_heads"], c["hd"])
        batch = vh.paged_batch(c["seqs"], st.rows, st.max_rows, st.max_len, _Buf(st.row_start), _Buf(st.len), _Buf(st.pages), st.page_ld)
        qd, kd = c["heads"] * c["hd"], c["kv_heads"] * c["hd"]

        def buf(t):
            return None if t is None else _Buf(t)
        if c["kind"] == "append":
            st.call = (vh.kv_append_dev, kv, batch,
                       vh.append_rows(wt, c["heads"], _Buf(st.qkv), qd + 2 * kd, _Buf(st.q), qd, q_norm=buf(st.qn), k_norm=buf(st.kn), eps=EPS,
                                      rope=_Buf(st.rope), rope_len=st.max_len, rot_dim=c["rot"], interleaved=c["interleaved"]))
        else:
            rows = vh.attn_rows(wt, c["heads"], _Buf(st.q), qd, _Buf(st.out), qd, 1.0 / math.sqrt(c["hd"]), cap=c["cap"], slopes=buf(st.slopes),
                                prefix=buf(st.prefix), window=c["window"])
            st.call = (vh.attn_paged_dev, kv, batch, rows) if c["kind"] == "attend" else \
                (vh.attn_shared_dev, kv, batch, vh.shared_prefix(st.groups, st.max_shared, _Buf(st.group_start), _Buf(st.group_len)), rows)
    st.call[0](*st.call[1:])
    return {"q": st.q, "k": st.k, "v": st.v} if c["kind"] == "append" else st.out


def _rows_of(st):
    """Sequence, index in it and position of every row of the batch."""
    i = torch.arange(st.rows, device=DEV)
    seq = torch.searchsorted(st.row_start, i, right=True) - 1
    at = i - st.row_start[seq]
    n = st.row_start[1:] - st.row_start[:-1]
    return seq, at, st.len[seq] - n[seq] + at


def _append(st):
    c = st.c
    H, G, hd, rot = c["heads"], c["kv_heads"], c["hd"], c["rot"]
    seq, _, pos = _rows_of(st)
    q, k, v = st.qkv.float().view(st.rows, H + 2 * G, hd).split((H, G, G), 1)

    def turn(x, w):
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        cos, sin = st.rope[pos].unbind(-1)
        cos, sin = cos[:, None], sin[:, None]
        if c["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., rot:]], -1)
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)
    st.q.copy_(turn(q, st.qn).reshape(st.rows, -1))
    page, slot = st.pages[seq, pos // c["page"]].long(), pos % c["page"]
    st.k[page, :, slot] = turn(k, st.kn).to(st.k.dtype)
    st.v[page, :, slot] = v.to(st.v.dtype)
    return {"q": st.q, "k": st.k, "v": st.v}


def _attend(st):
    c = st.c
    H, G, hd, L = c["heads"], c["kv_heads"], c["hd"], st.page_ld * c["page"]
    seq, at, pos = _rows_of(st)
    k, v = (t[st.pages].transpose(1, 2).reshape(c["seqs"], G, L, hd).float() for t in (st.k, st.v))
    q = torch.zeros((c["seqs"], st.max_rows, H, hd), device=DEV)
    q[seq, at] = st.q.float().view(st.rows, H, hd)
    p = torch.full((c["seqs"], st.max_rows), -1, dtype=torch.int64, device=DEV)
    p[seq, at] = pos
    q = q.view(c["seqs"], st.max_rows, G, H // G, hd).permute(0, 2, 3, 1, 4).reshape(c["seqs"], G, -1, hd)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(hd)).view(c["seqs"], H, st.max_rows, L)
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    j = torch.arange(L, device=DEV)
    if st.slopes is not None:
        s -= st.slopes[:, None, None] * (p[:, None, :, None] - j).abs()
    end = p + 1 if st.prefix is None else torch.maximum(p + 1, st.prefix[:, None])
    seen = j < torch.minimum(end, st.len[:, None])[..., None]
    if c["window"]:
        seen &= j > p[..., None] - c["window"]
    s.masked_fill_(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(c["seqs"], G, -1, L), v).view(c["seqs"], H, st.max_rows, hd)
    o = torch.where(total > 0, o / total, torch.zeros((), device=DEV))
    st.out.copy_(o.transpose(1, 2)[seq, at].reshape(st.rows, -1))
    return st.out


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st, c = prepare(case, seed), case
    rows, keys, _ = _lengths(c)
    H, G, hd, first = c["heads"], c["kv_heads"], c["hd"], 0
    table = st.pages.cpu().tolist()
    if c["kind"] == "append":
        k_all, v_all = st.k.double(), st.v.double()
        q_out = torch.zeros((st.rows, H * hd), dtype=torch.float64, device=DEV)
        half = c["rot"] // 2
        left = torch.arange(half, device=DEV) * (2 if c["interleaved"] else 1)
        right = left + (1 if c["interleaved"] else half)
        for s, (n, total) in enumerate(zip(rows, keys)):
            x = st.qkv[first:first + n].double().view(n, H + 2 * G, hd)
            qk = x[:, :H + G].clone()
            if c["norm"]:
                qk *= (qk.square().sum(-1, keepdim=True) / hd + EPS).rsqrt()
                qk[:, :H] *= st.qn.double()
                qk[:, H:] *= st.kn.double()
            turn = torch.view_as_complex(st.rope[total - n:total].double().contiguous())[:, None]
            z = torch.complex(qk[..., left], qk[..., right]) * turn
            qk[..., left], qk[..., right] = z.real, z.imag
            q_out[first:first + n] = qk[:, :H].reshape(n, -1)
            where = torch.arange(total - n, total)
            page = torch.tensor(table[s])[where // c["page"]].to(DEV)
            slot = (where % c["page"]).to(DEV)
            k_all[page, :, slot] = qk[:, H:]
            v_all[page, :, slot] = x[:, H + G:]
            first += n
        return {"q": q_out, "k": k_all, "v": v_all}
    out = torch.zeros((st.rows, H, hd), dtype=torch.float64, device=DEV)
    for s, (n, total) in enumerate(zip(rows, keys)):
        own_pages = st.pages[s, :-(-total // c["page"])].long()
        pos = torch.arange(total - n, total, device=DEV, dtype=torch.float64)[:, None]
        j = torch.arange(total, device=DEV, dtype=torch.float64)[None, :]
        hidden = j > pos
        if c["prefix"]:
            hidden &= j >= c["prefix"]
        if c["window"]:
            hidden |= pos - j >= c["window"]
        for h in range(H):
            kh, vh_ = (t[own_pages, h // (H // G)].reshape(-1, hd)[:total].double() for t in (st.k, st.v))
            z = st.q[first:first + n].view(n, H, hd)[:, h].double() @ kh.t() / math.sqrt(hd)
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            if c["slopes"]:
                z = z - st.slopes[h].double() * (pos - j).abs()
            out[first:first + n, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ vh_
        first += n
    return out.view(st.rows, -1)
