"""Refusals of the paged-cache operators at the C entry: wrong descriptors and
arguments are named on the host, before any CUDA call."""
import ctypes as C

import pytest

from rapidocrvl_b200 import _lib


def cache(**kw):
    d = _lib.KVCache(type=0, head_dim=128, num_kv_heads=2, num_layers=1, page_size=16, num_pages=4, batch=1, max_pages=4,
                     page_stride=2 * 2 * 16 * 128, layer_stride=2 * 2 * 16 * 128, head_stride=2 * 16 * 128, token_stride=128,
                     table_stride=4, k=1 << 20, v=(1 << 20) + 8192, table=1 << 21)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def compact(d, e=None, keep=4, idx=1 << 22):
    L = _lib.load()
    rc = L.ocrvl_op_kv_compact(C.byref(d), C.byref(e or d), idx, keep, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(type=1000), "type"), (dict(head_dim=96), "head_dim"), (dict(num_kv_heads=0), "positive"), (dict(num_layers=0), "positive"),
    (dict(batch=0), "positive"), (dict(max_pages=0), "positive"), (dict(num_pages=0), "positive"), (dict(page_size=8), "page_size"),
    (dict(page_size=24), "page_size"), (dict(k=None), "null"), (dict(table=None), "null"), (dict(v=(1 << 20) + 4), "aligned"),
    (dict(page_stride=-16), "strides"), (dict(token_stride=130), "strides"), (dict(token_stride=64), "token_stride"),
    (dict(batch=2, table_stride=3), "table_stride"), (dict(max_pages=1 << 28), "positions"), (dict(batch=70000), "sequences")])
def test_bad_caches_are_refused(kw, msg):
    rc, said = compact(cache(**kw))
    assert rc == _lib.E_INVALID and msg in said, said


def test_bad_moves_are_refused():
    for rc, said in (compact(cache(), keep=0), compact(cache(), idx=None), compact(cache(), cache(type=1)), compact(cache(), cache(num_layers=2)),
                     compact(cache(), cache(token_stride=256)), compact(cache(), keep=1 << 30)):
        assert rc == _lib.E_INVALID and said
    L = _lib.load()
    assert L.ocrvl_op_kv_compact(None, None, None, 1, None) == _lib.E_INVALID
    assert L.ocrvl_op_kv_select(1, 1, 1, None, 8, 8, None, 4, 0, 0, None, None, None, None) == _lib.E_INVALID
    p = 1 << 20
    for args in ((0, 1, 1, p, 8, 8, p, 4, 0, 0), (1, 1, 1, p, 8, 7, p, 4, 0, 0), (1, 1, 1, p, 8, 8, p, 0, 0, 0), (1, 1, 1, p, 8, 8, p, 4, 3, 2),
                 (1, 1, 1, p, 8, 8, p, 4, -1, 2)):
        assert L.ocrvl_op_kv_select(*args, p, None, None, None) == _lib.E_INVALID, args
    assert L.ocrvl_op_kv_select(1, 1, 1, p, 8, 8, p, 4, 0, 0, p, None, p, None) == _lib.E_INVALID  # new_lens is lens


def test_bad_tokens_are_refused():
    L, c, p = _lib.load(), cache(), 1 << 20

    def tree(c=c, layer=0, heads=16, n=1, draft=1, lens=p, indptr=p, mask=p, q=p, qs=2048, k=p, ks=256, scale=0.1, out=p, os=2048, work=p, wb=1 << 30):
        return L.ocrvl_op_tree_attn(C.byref(c), layer, heads, n, draft, lens, indptr, mask, q, qs, k, k, ks, scale, out, os, None, work, wb, None)

    for kw in (dict(layer=1), dict(layer=-1), dict(heads=0), dict(heads=3), dict(heads=34), dict(n=-1), dict(draft=0), dict(draft=65), dict(lens=None),
               dict(indptr=None), dict(mask=None), dict(q=None), dict(q=p + 4), dict(qs=2050), dict(qs=1024), dict(k=None), dict(ks=128), dict(scale=float("nan")),
               dict(out=None), dict(os=100), dict(work=None)):
        assert tree(**kw) == _lib.E_INVALID, kw
        assert _lib.last_error()
    assert tree(n=0) == _lib.OK  # nothing to do
    assert L.ocrvl_op_tree_attn_workspace(C.byref(c), 16, 1, None) == _lib.E_INVALID

    def mass(n=1, lse=p, decay=1.0, acc=None, aw=0, a_s=0, out=p, ow=64, os=64):
        return L.ocrvl_op_attn_mass(C.byref(c), 0, 16, n, 1, p, p, None, p, 2048, lse, 0.1, decay, acc, aw, a_s, out, ow, os, None)

    for kw in (dict(lse=None), dict(decay=float("inf")), dict(out=None), dict(ow=0), dict(os=63), dict(acc=p + 4096, aw=8, a_s=4), dict(acc=p, aw=64, a_s=32),
               dict(acc=p, aw=64, a_s=128)):
        assert mass(**kw) == _lib.E_INVALID, kw

    def append(n=1, lens=p, path=None, n_path=None, most=0, k=p, ks=256, new=p + 64):
        return L.ocrvl_op_kv_append(C.byref(c), n, lens, p, path, n_path, most, k, k, ks, 0, new, None)

    for kw in (dict(n=-1), dict(lens=None), dict(path=p), dict(path=p, n_path=p, most=0), dict(k=None), dict(k=p + 8), dict(ks=255), dict(ks=128), dict(new=None),
               dict(new=p)):
        assert append(**kw) == _lib.E_INVALID, kw


def test_sequence_entries_reject_null():
    L, d = _lib.load(), _lib.KVCache()
    assert L.ocrvl_seq_kv_view(None, C.byref(d)) == _lib.E_INVALID
    assert L.ocrvl_seq_truncate(None, 0) == _lib.E_INVALID


def test_set_position_rejects_null():
    assert _lib.load().ocrvl_seq_set_position(None, 0) == _lib.E_INVALID
    assert "null" in _lib.last_error()


def test_moves_into_too_little_room_are_refused():
    small = cache(max_pages=2, table=3 << 20, k=4 << 20, v=(4 << 20) + 8192)
    rc, said = compact(cache(), small, keep=33)
    assert rc == _lib.E_INVALID and "room" in said
