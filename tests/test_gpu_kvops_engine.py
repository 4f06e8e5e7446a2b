"""The paged-cache operators on the engine's own cache (ocrvl_seq_kv_view,
ocrvl_seq_truncate), and the example that runs them together."""
import math
import os
import runpy

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _runtime(q="q8"):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from rapidocrvl_b200 import LoadOptions, Runtime, config, synth

    d = synth.ensure("tiny", q)
    return Runtime.load(d, LoadOptions(quantization=q, max_position=2048, kv_pool_bytes=64 << 20)), config.load(d)


def _prefill(rt, cfg, n, seed):
    from rapidocrvl_b200 import synth

    seq = rt.new_sequence(n + 80)
    for t in synth.random_prompt(n, cfg.vocab_size, seed):
        rt.step([seq], ids=[t], need_logits=False)
    return seq


@pytest.mark.parametrize("n,keep", [(50, 20), (37, 32), (16, 16), (90, 33)])
def test_evicted_engine_sequence_goes_on_like_one_with_the_kept_positions(n, keep):
    """After evict in place and truncate, the cache holds the chosen positions
    of each layer and head, and further steps give the same logits, bit for
    bit, as a sequence that these keys and values were imported into."""
    import torch

    from rapidocrvl_b200 import kvops

    rt, cfg = _runtime()
    seq = _prefill(rt, cfg, n, 3)
    L, KVH, D = cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.head_dim
    before = [seq.read_kv(layer) for layer in range(L)]
    cache = kvops.PagedCache.of_sequence(seq)
    assert (cache.layers, cache.kv_heads, cache.head_dim, cache.batch) == (L, KVH, D, 1)
    acc = torch.rand(L, 1, KVH, n, generator=torch.Generator().manual_seed(n)).cuda()
    idx, _, new = kvops.evict(cache, acc, torch.tensor([n], dtype=torch.int32, device="cuda"), keep=keep, sinks=2, recent=5)
    torch.cuda.synchronize()
    held = int(new[0])
    assert held == min(n, keep)
    seq.truncate(held)
    assert len(seq) == held
    k = np.zeros((L, held, KVH * D), np.float32)
    v = np.zeros_like(k)
    for layer in range(L):
        gk, gv = seq.read_kv(layer)
        for h in range(KVH):
            pick, cols = idx[layer, 0, h, :held].cpu().numpy(), slice(h * D, (h + 1) * D)
            k[layer, :, cols], v[layer, :, cols] = before[layer][0][pick, cols], before[layer][1][pick, cols]
        assert np.array_equal(gk, k[layer]) and np.array_equal(gv, v[layer])
    other = rt.new_sequence(n + 80)
    other.import_kv(k, v)
    for i in range(20):  # over a page's end
        pos = [(n + i,) * 3]
        a, la = rt.step([seq], ids=[7 + i], positions=pos, return_logits=True)
        b, lb = rt.step([other], ids=[7 + i], positions=pos, return_logits=True)
        assert int(a[0]) == int(b[0]) and np.array_equal(la.view(np.uint32), lb.view(np.uint32)), i
    rt.close()


def test_truncate_takes_positions_back():
    from rapidocrvl_b200._lib import OcrvlError

    rt, cfg = _runtime()
    seq, ref = _prefill(rt, cfg, 40, 5), _prefill(rt, cfg, 33, 5)
    seq.truncate(33)
    assert len(seq) == 33
    for i in range(3):
        a, la = rt.step([seq], ids=[9 + i], return_logits=True)
        b, lb = rt.step([ref], ids=[9 + i], return_logits=True)
        assert np.array_equal(la.view(np.uint32), lb.view(np.uint32))
    for bad in (-1, len(seq) + 1):
        with pytest.raises(OcrvlError):
            seq.truncate(bad)
    seq.truncate(0)
    assert len(seq) == 0
    # every page went back: the pool can be filled again
    pages = 0
    rest = []
    while True:
        s = rt.new_sequence(1024)
        try:
            s.fill_synthetic(1024, 1)
        except OcrvlError:
            break
        rest.append(s)
        pages += 64
    ref.truncate(0)
    rest.pop().close()
    seq.fill_synthetic(120, 2)
    assert len(seq) == 120
    rt.close()


def test_attention_over_the_engines_cache():
    """tree_attention of the last layer's query over a sequence's own cache
    agrees with the engine's attention output for the same token (work buffers
    2 and 3 of ocrvl_debug_read), whose softmax the reference's order of sums
    fixes: every 16 positions exactly, so 48 of them here."""
    import ctypes as C

    import torch

    from rapidocrvl_b200 import _lib, kvops

    rt, cfg = _runtime()
    seq = _prefill(rt, cfg, 47, 11)
    rt.step([seq], ids=[5], need_logits=True)
    H, KVH, D, L = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, cfg.num_hidden_layers
    qkv, head = np.zeros((H + 2 * KVH) * D, np.float32), np.zeros(H * D, np.float32)
    for which, a in ((2, qkv), (3, head)):
        _lib.check(_lib.load().ocrvl_debug_read(rt._h, which, a.ctypes.data_as(C.c_void_p), a.size))
    half = D // 2
    ang = 47 * cfg.rope_theta ** (-np.arange(half) * 2.0 / D)
    c, s = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    q = qkv[:H * D].reshape(H, D)
    q = np.concatenate((q[:, :half] * c - q[:, half:] * s, q[:, half:] * c + q[:, :half] * s), 1)
    zeros = torch.zeros(1, KVH, D, device="cuda")
    out, _ = kvops.tree_attention(torch.from_numpy(q[None]).cuda(), zeros, zeros, kvops.PagedCache.of_sequence(seq),
                                  torch.tensor([48], dtype=torch.int32, device="cuda"),
                                  torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"),
                                  layer=L - 1, scale=1 / math.sqrt(D))
    # two rotations of f32 values (2^-23 each) and the exponential of the engine's own
    # polynomial (a few 2^-23): 1e-5 of the largest value is far above them all
    want = head.reshape(H, D)
    assert np.abs(out[0].cpu().numpy() - want).max() <= 1e-5 * np.abs(want).max() + 1e-6
    rt.close()


def test_example_runs(capsys, monkeypatch):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    monkeypatch.setattr("sys.argv", ["tree_decode.py", "--tokens", "24", "--budget", "40"])
    runpy.run_path(os.path.join(ROOT, "examples", "tree_decode.py"), run_name="__main__")
    said = capsys.readouterr().out
    assert "the same tokens" in said and "cut to at most 40" in said
