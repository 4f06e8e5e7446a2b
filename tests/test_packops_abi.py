"""Refusals of the packed cache's operators and of the rotation at the C entry:
wrong descriptors and arguments are named on the host, before any CUDA call."""
import ctypes as C
import math

import pytest

from rapidocrvl_b200 import _lib

K = 1 << 20


def cache(**kw):
    d = _lib.PackedCache(head_dim=128, num_kv_heads=2, num_layers=1, page_size=16, num_pages=4, batch=1, max_pages=4, reserved=0,
                         page_stride=2 * 1024, layer_stride=2 * 1024, head_stride=1024, scale_page_stride=128, scale_layer_stride=128,
                         scale_head_stride=64, table_stride=4, k=K, v=K + 8192, k_scale=2 * K, v_scale=2 * K + 1024, table=3 * K)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def read(c, type=30, n=1, lens=K, indptr=K, k=K, v=K, stride=256, layer=256):
    return _lib.load().ocrvl_op_packed_read(c and C.byref(c), type, n, lens, indptr, k, v, stride, layer, None), _lib.last_error()


def append(c, type=30, n=1, lens=K, indptr=K, path=None, n_path=None, most=0, k=K, v=K, stride=256, layer=256, new=K + 64):
    return _lib.load().ocrvl_op_packed_append(c and C.byref(c), type, n, lens, indptr, path, n_path, most, k, v, stride, layer, new, None), _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(head_dim=96), "head_dim"), (dict(num_kv_heads=0), "positive"), (dict(num_layers=0), "positive"), (dict(batch=0), "positive"),
    (dict(max_pages=0), "positive"), (dict(num_pages=-1), "positive"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(reserved=1), "reserved"), (dict(k=None), "null"), (dict(v_scale=None), "null"), (dict(table=None), "null"), (dict(v=K + 8), "aligned"),
    (dict(k_scale=2 * K + 8), "aligned"), (dict(page_stride=-16), "strides of the codes"), (dict(head_stride=1000), "strides of the codes"),
    (dict(scale_layer_stride=4), "strides of the scales"), (dict(scale_head_stride=-8), "strides of the scales"),
    (dict(batch=2, table_stride=3), "table_stride"), (dict(max_pages=1 << 28), "positions"), (dict(batch=70000), "sequences")])
def test_bad_caches_are_refused(kw, msg):
    for call in (read, append):
        rc, said = call(cache(**kw))
        assert rc == _lib.E_INVALID and msg in said, said


def test_bad_moves_are_refused():
    for call in (read, append):
        assert call(None)[0] == _lib.E_INVALID
        for kw in (dict(type=1000), dict(type=2), dict(n=-1), dict(lens=None), dict(indptr=None), dict(k=None), dict(v=None), dict(k=K + 8), dict(stride=255),
                   dict(stride=128), dict(stride=-256), dict(layer=4), dict(layer=-256)):
            rc, said = call(cache(), **kw)
            assert rc == _lib.E_INVALID and said, kw
    for kw in (dict(path=K), dict(path=K, n_path=K), dict(new=None), dict(new=K)):
        assert append(cache(), **kw)[0] == _lib.E_INVALID, kw
    assert read(cache(), n=0, k=None, v=None)[0] == _lib.OK  # nothing to do


def test_bad_attention_calls_are_refused():
    L, c, p = _lib.load(), cache(), K

    def attend(c=c, type=30, layer=0, heads=16, n=1, draft=1, lens=p, indptr=p, mask=p, q=p, qs=2048, k=p, ks=256, scale=0.1, out=p, os=2048, work=p, wb=1 << 30):
        return L.ocrvl_op_packed_attn(c and C.byref(c), type, layer, heads, n, draft, lens, indptr, mask, q, qs, k, k, ks, scale, out, os, None, work, wb, None)

    for kw in (dict(c=None), dict(type=2), dict(layer=1), dict(layer=-1), dict(heads=0), dict(heads=3), dict(heads=34), dict(n=-1), dict(draft=0), dict(draft=65), dict(lens=None),
               dict(indptr=None), dict(mask=None), dict(q=None), dict(q=p + 4), dict(qs=2050), dict(qs=1024), dict(k=None), dict(k=p + 8), dict(ks=128), dict(ks=1 << 30),
               dict(scale=math.nan), dict(out=None), dict(os=100), dict(work=None)):
        assert attend(**kw) == _lib.E_INVALID, kw
        assert _lib.last_error()
    assert attend(n=0) == _lib.OK
    n = C.c_int64()
    assert L.ocrvl_op_packed_attn_workspace(C.byref(c), 30, 16, 1, None) == _lib.E_INVALID
    assert L.ocrvl_op_packed_attn_workspace(C.byref(c), 2, 16, 1, C.byref(n)) == _lib.E_INVALID
    assert L.ocrvl_op_packed_attn_workspace(C.byref(c), 30, 3, 1, C.byref(n)) == _lib.E_INVALID


def rotary(**kw):
    r = _lib.Rotary(head_dim=128, pairs=64, num_axes=3, neighbours=0)
    for p in range(64):
        r.freq[p], r.axis[p] = 0.5, p % 3
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def rotate(r, type=30, n=1, pos=K, pos_stride=3, heads=16, q=K, qs=2048, qo=2 * K, qos=2048, kv=2, k=3 * K, ks=256, ko=4 * K, kos=256, wt=0, qw=None, kw=None, eps=1e-6):
    rc = _lib.load().ocrvl_op_rotate(r and C.byref(r), type, n, pos, pos_stride, heads, q, qs, qo, qos, kv, k, ks, ko, kos, wt, qw, kw, eps, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(head_dim=100), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(pairs=62), "pairs"), (dict(pairs=68), "pairs"),
    (dict(pairs=0), "pairs"), (dict(num_axes=0), "num_axes"), (dict(num_axes=9), "num_axes"), (dict(num_axes=2), "axis"), (dict(neighbours=2), "neighbours")])
def test_bad_rotaries_are_refused(kw, msg):
    rc, said = rotate(rotary(**kw))
    assert rc == _lib.E_INVALID and msg in said, said


def test_bad_rotations_are_refused():
    assert rotate(None)[0] == _lib.E_INVALID
    r = rotary()
    r.freq[63] = math.nan
    assert rotate(r)[0] == _lib.E_INVALID
    for kw in (dict(type=1000), dict(n=-1), dict(pos=None), dict(pos_stride=2), dict(heads=0), dict(heads=1 << 20), dict(q=None), dict(q=K + 8), dict(qs=2047), dict(qs=1024), dict(qo=None),
               dict(qos=1024), dict(qo=K, qos=4096), dict(kv=0), dict(kv=-1), dict(ks=128), dict(ko=None), dict(ko=4 * K + 2), dict(kos=255), dict(ko=3 * K, kos=512), dict(qw=K), dict(kw=K),
               dict(qw=K, kw=K, wt=1), dict(qw=K + 4, kw=K), dict(qw=K, kw=K, eps=-1.0), dict(qw=K, kw=K, eps=math.inf), dict(qw=K, kw=K, eps=math.nan)):
        rc, said = rotate(rotary(), **kw)
        assert rc == _lib.E_INVALID and said, kw
    assert rotate(rotary(), n=0)[0] == _lib.OK


def test_reads_into_shared_memory_are_refused():
    for kw in (dict(v=K), dict(layer=0), dict(n=4, layer=128), dict(n=4, layer=256), dict(n=4, stride=256, layer=768)):
        rc, said = read(cache(num_layers=2), **{"v": K + 4096, **kw})
        assert rc == _lib.E_INVALID and "share" in said, kw
