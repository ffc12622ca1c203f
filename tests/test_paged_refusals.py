"""What the paged-cache entry points refuse, before anything touches a device: every call here has one thing wrong, and the
call that has nothing wrong gets as far as the missing device (or, where there is one, is not made)."""
import ctypes as C

import pytest

from vox_amd import voxhip as vh

A = 1 << 20  # an aligned address, never followed


class At:
    def __init__(self, ptr):
        self.ptr = ptr


def parts(**kw):
    kv = vh.paged_kv(At(A), At(2 * A), vh.F16, 10, 16, 2, 64)
    b = vh.paged_batch(3, 7, 4, 100, At(A), At(A), At(A), 7)
    ap = vh.append_rows(vh.F32, 4, At(A), 512, At(8 * A), 256, rope=At(A), rope_len=200, rot_dim=64)
    at = vh.attn_rows(vh.F32, 4, At(A), 256, At(A), 256, 0.125)
    sh = vh.shared_prefix(1, 50, At(A), At(A))
    named = {"kv": kv, "b": b, "ap": ap, "at": at, "sh": sh}
    for k, v in kw.items():
        who, field = k.split("_", 1)
        setattr(named[who], field, v)
    return kv, b, ap, at, sh


def error(fn, *args):
    L = vh.lib()
    assert getattr(L, fn)(*[None if a is None else C.byref(a) for a in args]) == 0
    return L.voxhip_last_error().decode()


BOTH = [
    (dict(kv_type=vh.F32), "f16 or bf16"), (dict(kv_type=vh.BF16), "bf16 rows need a bf16 cache"),
    (dict(kv_head_dim=136), "head_dim"), (dict(kv_head_dim=60), "head_dim"), (dict(kv_head_dim=0), "head_dim"),
    (dict(kv_page_size=24), "page_size"), (dict(kv_page_size=4), "page_size"), (dict(kv_page_size=2048), "page_size"),
    (dict(kv_pages=0), "no pages"), (dict(kv_kv_heads=0), "kv_heads"), (dict(kv_kv_heads=3), "overlap"),
    (dict(kv_pos_stride=56), "strides"), (dict(kv_pos_stride=68), "strides"), (dict(kv_page_stride=-2048), "strides"), (dict(kv_pos_stride=(1 << 26) + 8), "too large"),
    (dict(kv_head_stride=64), "overlap"), (dict(kv_page_stride=1024), "pages overlap"), (dict(kv_page_stride=1 << 60), "too large"),
    (dict(kv_k=None), "k is missing"), (dict(kv_v=None), "v is missing"), (dict(kv_k=A + 8), "k is not aligned"),
    (dict(b_seqs=-1), "out of range"), (dict(b_rows=-1), "out of range"), (dict(b_rows=(1 << 24) + 1), "out of range"),
    (dict(b_max_rows=0), "max_rows"), (dict(b_max_rows=8), "max_rows"), (dict(b_max_len=0), "max_len"), (dict(b_max_len=113), "max_len"),
    (dict(b_page_ld=0), "page_ld"), (dict(b_page_ld=1 << 40), "page_ld"), (dict(b_row_start=None), "row_start is missing"),
    (dict(b_len=None), "len is missing"), (dict(b_pages=None), "pages is missing"), (dict(b_pages=A + 2), "pages is not aligned"),
]


@pytest.mark.parametrize("change,why", BOTH, ids=lambda v: "-".join(v) if isinstance(v, dict) else None)
def test_cache_and_batch(change, why):
    kv, b, ap, at, sh = parts(**change)
    for args in (("voxhip_kv_append_dev", kv, b, ap), ("voxhip_attn_paged_dev", kv, b, at), ("voxhip_attn_shared_dev", kv, b, sh, at)):
        assert why in error(*args), args[0]


@pytest.mark.parametrize("change,why", [
    (dict(ap_type=vh.Q8), "rows are"), (dict(ap_type=vh.BF16), "bf16"), (dict(ap_heads=3), "multiple"), (dict(ap_heads=0), "heads"),
    (dict(ap_qkv=None), "qkv is missing"), (dict(ap_qkv=A + 4), "qkv is not aligned"), (dict(ap_ld_qkv=511), "shorter"),
    (dict(ap_ld_qkv=516), "multiple of 8"), (dict(ap_ld_q=248), "shorter"), (dict(ap_q=A), "overlaps"), (dict(ap_q=A + 1024), "overlaps"),
    (dict(ap_q=A + 512 * 4 * 6 + 512 * 4 - 16), "overlaps"), (dict(ap_qkv=8 * A + 255 * 4 * 4), "overlaps"),
    (dict(ap_rope_len=0), "rope_len"), (dict(ap_rot_dim=72), "rot_dim"), (dict(ap_rot_dim=0), "rot_dim"), (dict(ap_rot_dim=12), "rot_dim"),
    (dict(ap_rope=A + 8), "rope is not aligned"), (dict(ap_q_norm=A + 4), "q_norm"), (dict(ap_k_norm=A, ap_eps=-1.0), "eps"),
    (dict(ap_k_norm=A, ap_eps=float("nan")), "eps")], ids=lambda v: "-".join(v) if isinstance(v, dict) else None)
def test_append(change, why):
    kv, b, ap, _, _ = parts(**change)
    assert why in error("voxhip_kv_append_dev", kv, b, ap)


@pytest.mark.parametrize("change,why", [
    (dict(at_type=vh.Q4), "rows are"), (dict(at_heads=5), "multiple"), (dict(at_heads=2048), "heads"), (dict(at_q=None), "q is missing"),
    (dict(at_out=None), "out is missing"), (dict(at_ld_q=248), "shorter"), (dict(at_ld_out=260), "multiple of 8"),
    (dict(at_scale=float("inf")), "scale"), (dict(at_cap=-1.0), "cap"), (dict(at_cap=float("nan")), "cap"), (dict(at_window=-1), "window"),
    (dict(at_slopes=A + 2), "slopes"), (dict(at_prefix=A + 1), "prefix"), (dict(at_out=A + 16), "partly"),
    (dict(at_heads=1024, b_rows=(1 << 20) + 1), "rows x heads")],
    ids=lambda v: "-".join(v) if isinstance(v, dict) else None)
def test_attention(change, why):
    kv, b, _, at, sh = parts(**change)
    assert why in error("voxhip_attn_paged_dev", kv, b, at)
    assert why in error("voxhip_attn_shared_dev", kv, b, sh, at)


@pytest.mark.parametrize("change,why", [
    (dict(sh_groups=-1), "more groups"), (dict(sh_groups=4), "more groups"), (dict(sh_max_len=-1), "shared max_len"),
    (dict(sh_max_len=101), "shared max_len"), (dict(sh_seq_start=None), "seq_start is missing"), (dict(sh_len=None), "len is missing")],
    ids=lambda v: "-".join(v) if isinstance(v, dict) else None)
def test_shared(change, why):
    kv, b, _, at, sh = parts(**change)
    assert why in error("voxhip_attn_shared_dev", kv, b, sh, at)


def pool_step(rows, lens, pages, groups=(), change=()):
    import numpy as np
    r, n, p = (np.array(v, np.int32) for v in (rows, lens, pages))
    starts = np.array([a for a, _, _ in groups] + [groups[-1][1]] if groups else [0], np.int32)
    shared = np.array([k for _, _, k in groups] or [0], np.int32)
    b = vh.PoolBatch(len(rows), r.ctypes.data, n.ctypes.data, p.ctypes.data, p.shape[1], len(groups), starts.ctypes.data, shared.ctypes.data)
    for k, v in change:
        setattr(b, k, v)
    x = np.zeros((8, 8), np.float32)
    assert vh.lib().voxhip_xfmr_forward_paged(0, 0, C.byref(b), x.ctypes.data, None, -1, None) == 0
    return vh.lib().voxhip_last_error().decode()


def test_pool():
    L = vh.lib()
    for pages, size in ((0, 16), (-1, 16), (1 << 28, 16)):
        assert L.voxhip_pool_create(0, pages, size) == -1 and b"pages out of range" in L.voxhip_last_error()
    for size in (0, 4, 24, 2048):
        assert L.voxhip_pool_create(0, 4, size) == -1 and b"page_size" in L.voxhip_last_error()
    assert L.voxhip_pool_free(0) == 0
    assert "missing" in pool_step([1], [1], [[0]], change=[("rows", None)])
    assert "missing" in pool_step([1], [1], [[0]], change=[("pages", None)])
    assert "missing" in pool_step([1], [1], [[0]], change=[("page_ld", 0)])
    assert L.voxhip_xfmr_forward_paged(0, 0, None, None, None, -1, None) == 0
    assert L.voxhip_xfmr_forward_paged(0, 0, C.byref(vh.PoolBatch(0)), None, None, -1, None) == 1  # nothing to do


def test_missing_structs():
    kv, b, ap, at, sh = parts()
    assert "no cache" in error("voxhip_kv_append_dev", None, b, ap)
    assert "no batch" in error("voxhip_kv_append_dev", kv, None, ap)
    assert "no rows" in error("voxhip_kv_append_dev", kv, b, None)
    assert "no cache" in error("voxhip_attn_paged_dev", None, b, at)
    assert "no batch" in error("voxhip_attn_paged_dev", kv, None, at)
    assert "no rows" in error("voxhip_attn_paged_dev", kv, b, None)
    assert "no shared prefixes" in error("voxhip_attn_shared_dev", kv, b, None, at)


def test_nothing_to_do():
    # no sequence or no row: done, whatever the buffers are
    for change in (dict(b_seqs=0), dict(b_rows=0)):
        kv, b, ap, at, sh = parts(**change)
        b.row_start = b.len = b.pages = None
        assert vh.lib().voxhip_kv_append_dev(C.byref(kv), C.byref(b), C.byref(ap)) == 1
        assert vh.lib().voxhip_attn_paged_dev(C.byref(kv), C.byref(b), C.byref(at)) == 1
        assert vh.lib().voxhip_attn_shared_dev(C.byref(kv), C.byref(b), C.byref(sh), C.byref(at)) == 1


def test_right_arguments_reach_the_device():
    if vh.device_count() > 0:
        pytest.skip("a HIP device is present: the addresses here are not to be followed")
    kv, b, ap, at, sh = parts()
    for args in (("voxhip_kv_append_dev", kv, b, ap), ("voxhip_attn_paged_dev", kv, b, at), ("voxhip_attn_shared_dev", kv, b, sh, at)):
        assert "not initialised" in error(*args) or "init failed" in error(*args), args[0]
