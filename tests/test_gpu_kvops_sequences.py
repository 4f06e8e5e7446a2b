"""The paged-cache operators on engine sequences that grow, shrink and share
the engine's pool with others."""
import numpy as np
import pytest

from test_gpu_kvops_engine import _prefill, _runtime

pytestmark = pytest.mark.gpu


def _cache(seq, cfg):
    kv = [seq.read_kv(layer) for layer in range(cfg.num_hidden_layers)]
    return np.stack([x[0] for x in kv]), np.stack([x[1] for x in kv])


def _append(seq, cfg, at, tokens):
    import torch

    from rapidocrvl_b200 import kvops

    x = torch.full((cfg.num_hidden_layers, tokens, cfg.num_key_value_heads, cfg.head_dim), 77.0, device="cuda")
    kvops.append(kvops.PagedCache.of_sequence(seq), x, x, torch.tensor([at], dtype=torch.int32, device="cuda"),
                 torch.tensor([0, tokens], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


def _same(a, b):
    return all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))


def test_append_behind_a_view_reaches_no_other_sequence():
    """Pages that a sequence never had, gave back by truncate, or by reset are unmapped for it."""
    rt, cfg = _runtime()
    first, seq = _prefill(rt, cfg, 20, 1), _prefill(rt, cfg, 48, 2)  # `first` has the pool's first page
    kept = _cache(first, cfg)
    _append(seq, cfg, 48, 30)
    assert _same(_cache(first, cfg), kept)
    seq.truncate(17)
    mine = _cache(seq, cfg)
    other = _prefill(rt, cfg, 20, 3)  # takes the page that came back
    theirs = _cache(other, cfg)
    _append(seq, cfg, 32, 16)
    assert _same(_cache(first, cfg), kept) and _same(_cache(other, cfg), theirs) and _same(_cache(seq, cfg), mine)
    seq.reset()
    third = _prefill(rt, cfg, 40, 4)
    theirs = _cache(other, cfg), _cache(third, cfg)
    _append(seq, cfg, 0, 64)
    assert _same(_cache(first, cfg), kept) and _same(_cache(other, cfg), theirs[0]) and _same(_cache(third, cfg), theirs[1])
    rt.close()


def test_lengths_past_a_sequences_pages_attend_nothing():
    import torch

    from rapidocrvl_b200 import kvops

    rt, cfg = _runtime()
    _prefill(rt, cfg, 40, 1)
    seq = _prefill(rt, cfg, 60, 2)
    view = kvops.PagedCache.of_sequence(seq)  # taken once: the table follows the sequence
    H, KVH, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    q, kv = torch.randn(1, H, D, device="cuda"), torch.randn(1, KVH, D, device="cuda")

    def attend(n):
        one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        return kvops.tree_attention(q, kv, kv, view, torch.tensor([n], dtype=torch.int32, device="cuda"), one, torch.ones(1, dtype=torch.int64, device="cuda"))

    for n in (64, 32):  # whole pages: 60 positions have four of them
        a, b = attend(n), attend(140)
        assert torch.allclose(a[0], b[0], rtol=0, atol=1e-5) and torch.allclose(a[1], b[1], rtol=0, atol=1e-5)
        seq.truncate(32)
        _prefill(rt, cfg, 40, 5)  # takes the pages that came back
    for t in range(20):  # and grows again
        rt.step([seq], ids=[3 + t], need_logits=False)
    assert abs(float(attend(52)[1].sum() - attend(32)[1].sum())) > 1e-3
    rt.close()


@pytest.mark.parametrize("q,n,keep", [("q8", 50, 20), ("q4", 37, 32), ("q6", 90, 33)])
def test_evicted_sequence_counts_on_without_positions_given(q, n, keep):
    """Steps without positions and the device-fed loop after evict, truncate
    and set_position give what steps with explicit positions give."""
    import torch

    from rapidocrvl_b200 import kvops
    from rapidocrvl_b200._lib import OcrvlError

    rt, cfg = _runtime(q)
    seq = _prefill(rt, cfg, n, 3)
    acc = torch.rand(cfg.num_hidden_layers, 1, cfg.num_key_value_heads, n, generator=torch.Generator().manual_seed(n)).cuda()
    kvops.evict(kvops.PagedCache.of_sequence(seq), acc, torch.tensor([n], dtype=torch.int32, device="cuda"), keep=keep, sinks=2, recent=5)
    torch.cuda.synchronize()
    seq.truncate(keep)
    seq.set_position(n)
    ref = rt.new_sequence(n + 80)
    ref.import_kv(*_cache(seq, cfg))
    tok, at = 7, n
    for _ in range(4):  # steps
        a, la = rt.step([seq], ids=[tok], return_logits=True)
        b, lb = rt.step([ref], ids=[tok], positions=[(at,) * 3], return_logits=True)
        assert int(a[0]) == int(b[0]) and np.array_equal(la.view(np.uint32), lb.view(np.uint32))
        tok, at = int(b[0]), at + 1
    got, want = rt.decode_device([seq], [tok], 20).ravel().tolist(), []  # the loop
    first = tok
    for _ in range(20):
        tok = int(rt.step([ref], ids=[tok], positions=[(at,) * 3])[0][0])
        want.append(tok)
        at += 1
    assert got == want and _same(_cache(seq, cfg), _cache(ref, cfg))
    seq.truncate(len(seq) - 6)  # taken back: the positions go back too
    ref.truncate(len(ref) - 6)
    (a, la), (b, lb) = rt.step([seq], ids=[first], return_logits=True), rt.step([ref], ids=[first], positions=[(at - 6,) * 3], return_logits=True)
    assert np.array_equal(la.view(np.uint32), lb.view(np.uint32))
    for bad in (len(seq) - 1, 2048, -1):
        with pytest.raises(OcrvlError):
            seq.set_position(bad)
    seq.set_position(2048 - 3)
    with pytest.raises(OcrvlError):
        rt.decode_device([seq], [first], 4)
    rt.decode_device([seq], [first], 3)
    with pytest.raises(OcrvlError):
        rt.step([seq], ids=[first])
    seq.reset()
    ref.reset()
    (_, la), (_, lb) = rt.step([seq], ids=[5], return_logits=True), rt.step([ref], ids=[5], return_logits=True)
    assert np.array_equal(la.view(np.uint32), lb.view(np.uint32))
    rt.close()
