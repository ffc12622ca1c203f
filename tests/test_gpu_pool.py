"""A transformer over a pool of pages (voxhip_xfmr_forward_paged): prompts and steps of many sessions in one call, shared prompts
read from one session's pages, against the oracle run on each session alone over its own f16 cache. Bar: the library's for
whole transformers (1e-3 of max(1, max |ref|)), which an append into a wrong page or a wrong key in the attention misses by far."""
import numpy as np
import pytest

from conftest import rel_err
from models import BF16, F16, F32, Q4, Q8, Model

pytestmark = pytest.mark.gpu
TOL = 1e-3


class Server:
    """Sessions over one pool: their page tables, and each one's oracle cache."""

    def __init__(self, hip, mdl, sessions, pages=64, size=16, cap=200, seed=0):
        self.hip, self.mdl, self.size = hip, mdl, size
        self.xf = hip.xfmr_create(mdl.hx, "pool")
        self.head = hip.upload(mdl.head[1]) if mdl.head else -1
        self.pool = hip.pool_create(self.xf, pages, size)
        rng = np.random.default_rng(seed)
        self.rng, self.free = rng, list(rng.permutation(pages))
        self.ld = -(-cap // size)
        self.table = np.full((sessions, self.ld), -1, np.int32)
        self.len = np.zeros(sessions, np.int32)
        self.kv = [mdl.oracle_kv(cap, kv_f16=1) for _ in range(sessions)]

    def step(self, rows, groups=(), check=None):
        """New random rows for every session; the device's outputs against the oracle's."""
        rows = np.array(rows, np.int32)
        shared, lead = np.zeros(len(rows), int), list(range(len(rows)))
        for a, b, n in groups:
            shared[a:b], lead[a:b] = n, [a] * (b - a)
        for s, n in enumerate(rows):
            self.len[s] += n
            for p in range(-(-int(self.len[s]) // self.size)):
                if self.table[s, p] < 0 and not (lead[s] != s and (p + 1) * self.size <= shared[s]):
                    self.table[s, p] = self.free.pop()
        x = self.rng.standard_normal((int(rows.sum()), self.mdl.hidden)).astype(np.float32)
        out, logits = self.hip.forward_paged(self.xf, self.pool, rows, self.len, self.table, x, self.mdl.hidden, head=self.head, groups=groups)
        import pyoracle as po
        at = 0
        for s, n in enumerate(rows):
            if not n:
                assert not out[s].any()
                continue
            ref = po.transformer_forward(self.mdl.ox, self.kv[s], x[at:at + n])
            at += n
            assert rel_err(out[s], ref) < TOL, (s, rel_err(out[s], ref))
            if self.head >= 0:  # on the device's own state, as elsewhere
                want = po.matmul(self.mdl.head[0], out[s][None])[0]
                assert rel_err(logits[s], want) < TOL, (s, rel_err(logits[s], want))
        return out, logits


@pytest.mark.parametrize("wt", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 128), (7, 1, 64), (3, 3, 40)])
def test_prompts_and_steps(hip, oracle, wt, heads, kv_heads, hd):
    mdl = Model(300 + wt + hd, 2, 256, heads, kv_heads, hd, 512, wtype=wt, head_rows=130, qk_norm=hd != 64, bias=hd == 64)
    sv = Server(hip, mdl, 5)
    sv.step([20, 1, 0, 33, 7])
    sv.step([1, 1, 1, 1, 1])
    sv.step([1, 30, 2, 0, 1])   # a prompt chunk among steps
    sv.step([0, 0, 1, 0, 0])
    hip.pool_free(sv.pool)


def test_long_batch_in_passes(hip, oracle):
    # 700 rows: two passes of the layers, the border inside a session; the last pass ends several sessions
    mdl = Model(31, 2, 256, 4, 2, 64, 512, wtype=F16, head_rows=64)
    sv = Server(hip, mdl, 4, pages=80, cap=500)
    sv.step([300, 330, 20, 50])
    sv.step([1, 1, 1, 1])
    hip.pool_free(sv.pool)


@pytest.mark.parametrize("wt", [Q8, Q4])
def test_quantized_steps(hip, oracle, wt):
    # up to 8 rows in a call take the int8 activations that one row alone takes in the oracle
    mdl = Model(41 + wt, 2, 256, 4, 2, 128, 512, wtype=wt, head_rows=64)
    sv = Server(hip, mdl, 8)
    for _ in range(4):
        sv.step([1] * 8)
    sv.step([1, 0, 0, 1, 0, 0, 0, 1])
    hip.pool_free(sv.pool)


def test_quantized_prompts(hip, oracle):
    # more than 8 rows in every session: f32 activations on both sides
    mdl = Model(51, 2, 256, 4, 2, 128, 512, wtype=Q8, head_rows=0)
    sv = Server(hip, mdl, 3)
    sv.step([12, 40, 9])
    hip.pool_free(sv.pool)


def test_more_sessions_than_the_head_takes_at_once(hip, oracle):
    # a q4 head takes 8 rows a product; f16 layers take all 21 sessions' rows in one pass
    mdl = Model(57, 1, 256, 4, 2, 64, 256, wtype=F16, head_rows=96, head_type=Q4)
    sv = Server(hip, mdl, 21, pages=128, cap=60)
    sv.step([2] * 20 + [30])
    sv.step([1] * 21)
    hip.pool_free(sv.pool)


@pytest.mark.parametrize("wt", [F32, F16])
def test_shared_prompt(hip, oracle, wt):
    """One session of each voice reads the prompt, the others begin behind its whole pages (32 of 37 keys of the second voice's);
    the oracle's sessions each hold the prompt themselves."""
    mdl = Model(61 + wt, 2, 256, 4, 2, 64, 512, wtype=wt, head_rows=64)
    sv = Server(hip, mdl, 6, seed=3)
    sv.step([48, 0, 0, 37, 0, 0])
    for s, lead, n in ((1, 0, 48), (2, 0, 48), (4, 3, 32), (5, 3, 32)):
        sv.len[s] = n
        for src, dst in ((sv.kv[lead].k, sv.kv[s].k), (sv.kv[lead].v, sv.kv[s].v)):
            dst[:, :n] = src[:, :n]
        sv.kv[s].c.len = n
    groups = [(0, 3, 48), (3, 6, 32)]
    sv.step([1, 1, 1, 1, 1, 1], groups)
    sv.step([1, 20, 3, 0, 1, 9], groups)
    for _ in range(3):
        sv.step([1, 1, 1, 1, 1, 1], groups)
    hip.pool_free(sv.pool)


def test_refusals(hip, oracle):
    mdl = Model(71, 1, 256, 4, 2, 64, 256, wtype=F16)
    other = Model(72, 1, 256, 4, 4, 64, 256, wtype=F16)
    xf, xo = hip.xfmr_create(mdl.hx, "a"), hip.xfmr_create(other.hx, "b")
    pool = hip.pool_create(xf, 8, 16)
    x = np.zeros((4, 256), np.float32)

    def call(rows, lens, pages, groups=(), xfmr=xf, p=pool, head=-1):
        return hip.forward_paged(xfmr, p, rows, lens, pages, x, 256, head=head, groups=groups)
    call([1, 1], [1, 1], [[0], [1]])
    for args, why in (
            (([1, 1], [1, 1], [[0], [0]]), "write one page"), (([1], [1], [[8]]), "outside the pool"), (([1], [1], [[-1]]), "outside the pool"),
            (([1], [17], [[0]]), "exceeds the page table"), (([2], [1], [[0]]), "more than len"), (([-1], [1], [[0]]), "negative"),
            (([1, 1], [20, 3], [[0, 1], [2, 3]], [(0, 2, 16)]), "among its group's"), (([0, 1], [4, 18], [[0, 1], [2, 3]], [(0, 2, 16)]), "first sequence has"),
            (([1, 1], [18, 18], [[0, 1], [-1, -1]], [(0, 2, 16)]), "outside the pool"), (([1, 1], [18, 18], [[9, 1], [-1, 2]], [(0, 2, 16)]), "outside the pool")):
        with pytest.raises(hip.VoxHipError, match=why):
            call(*args)
    with pytest.raises(hip.VoxHipError, match="another transformer shape"):
        call([1], [1], [[0]], xfmr=xo)
    with pytest.raises(hip.VoxHipError, match="bad pool handle"):
        call([1], [1], [[0]], p=99)
    with pytest.raises(hip.VoxHipError, match="bad matrix handle"):
        hip._check(hip.lib().voxhip_xfmr_forward_paged(xf, pool, _one(hip), hip._p(x), None, 9999, None), "x")
    call([1, 1], [2, 2], [[0], [1]])  # and after them all a right one runs
    used = hip.mem_info().used
    big = hip.pool_create(xf, 64, 128)
    assert hip.mem_info().used - used == 2 * 64 * 128 * 2 * 64 * 2
    hip.pool_free(big)
    assert hip.mem_info().used == used
    with pytest.raises(hip.VoxHipError, match="bad pool handle"):
        hip.pool_free(big)
    hip.pool_free(pool)


def test_no_room(hip, oracle):
    """A pool that the memory limit refuses."""
    mdl = Model(81, 1, 256, 4, 2, 64, 256, wtype=F16)
    sv = Server(hip, mdl, 2)
    try:
        used = hip.mem_info().used
        hip.lib().voxhip_set_vram_limit(1)  # weight copies of other tests' models, which would give way, cannot make room for it
        with pytest.raises(hip.VoxHipError, match="VRAM limit"):
            hip.pool_create(sv.xf, 4096, 128)
        assert hip.mem_info().used == used
    finally:
        hip.lib().voxhip_set_vram_limit(0)
    sv.step([3, 2])
    hip.pool_free(sv.pool)


def _one(hip):
    import ctypes as C
    keep = [np.array(v, np.int32) for v in ([1], [1], [0])]
    _one.keep = keep
    return C.byref(hip.PoolBatch(1, keep[0].ctypes.data, keep[1].ctypes.data, keep[2].ctypes.data, 1, 0, None, None))
