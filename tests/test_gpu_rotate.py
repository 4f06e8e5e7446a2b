"""kvops.rotate against the formula in 64 bits.

Tolerance, relative to the pair's length r = sqrt(u^2 + v^2) after the norm: the angle in half turns is rounded
once to 32 bits (2^-25 of a half turn at most, 2^-23.3 rad), sine and cosine are off by 2 ulp (2^-23), and the two products and the
sum by 3 halves of 2^-24: below 2^-21.  The norm adds its sum of up to 256 squares (in at most 21 roundings a value, half of them
behind the root: 2^-20.6), the root (2 ulp) and three products: below 2^-20 more.  2^-19 r is allowed for all, and half a step
of the type (eps / 2 of the value, or of its smallest normal number)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kvops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from rapidocrvl_b200 import kvops

    return kvops


def want(x, pos, freq, axis, neighbours, weight=None, eps=0.0):
    """The rotated heads and each value's r, in 64 bits."""
    y, P = x.cpu().double(), len(freq)
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.cpu().double()
    a = (pos.cpu().double()[:, axis] * torch.tensor(freq, dtype=torch.float64))[:, None]
    i = torch.arange(P)
    u, v = (2 * i, 2 * i + 1) if neighbours else (i, i + P)
    out, r = y.clone(), y.abs()
    out[..., u], out[..., v] = y[..., u] * a.cos() - y[..., v] * a.sin(), y[..., v] * a.cos() + y[..., u] * a.sin()
    r[..., u] = r[..., v] = torch.hypot(y[..., u], y[..., v])
    return out, r


def check(got, x, *a, **kw):
    w, r = want(x, *a, **kw)
    f = torch.finfo(x.dtype)
    off = (got.cpu().double() - w).abs()
    bound = 2.0 ** -19 * r + f.eps / 2 * w.abs().clamp(min=f.smallest_normal)
    assert bool((off <= bound).all()), float((off / bound).max())


def inputs(dtype, n, heads, kv_heads, dim, axes, far, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = (1.5 * torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g)).to(TYPES[dtype]).cuda()
    q, k = qkv[:, :heads * dim].view(n, heads, dim), qkv[:, heads * dim:(heads + kv_heads) * dim].view(n, kv_heads, dim)
    pos = torch.randint(0, far, (n, axes), generator=g, dtype=torch.int32).cuda()
    w = [(1 + 0.2 * torch.randn(dim, generator=g)).to(TYPES[dtype]).cuda() for _ in range(2)]
    return qkv, q, k, pos, w


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,heads,kv_heads,dim,pairs,sections,neighbours,norm", [
    (1, 16, 2, 128, 64, (16, 24, 24), False, False), (1, 16, 2, 128, 64, (16, 24, 24), False, True), (5, 4, 2, 64, 32, None, True, True),
    (7, 16, 16, 72, 36, (18, 18), False, False), (33, 3, 1, 72, 36, (18, 18), False, True), (300, 12, 4, 96, 24, (8, 8, 8), True, False),
    (3000, 2, 2, 128, 32, (8, 0, 12, 12), False, True), (2, 1, 1, 256, 64, None, False, True), (9, 5, 5, 256, 128, (128,), True, True), (4, 8, 8, 8, 4, None, False, True),
    (3, 7, 3, 24, 4, (1, 1, 2), True, False), (40, 32, 8, 80, 40, (20, 20), False, True)])
def test_rotate(kvops, dtype, n, heads, kv_heads, dim, pairs, sections, neighbours, norm):
    axes = len(sections) if sections else 1
    _, q, k, pos, w = inputs(dtype, n, heads, kv_heads, dim, axes, 5000)
    rot = kvops.Rotary(dim, theta=5e5, pairs=pairs, sections=sections, neighbours=neighbours)
    assert rot.axes == axes
    kw = dict(q_weight=w[0], k_weight=w[1], eps=1e-5) if norm else {}
    rq, rk = kvops.rotate(q, k, pos, rot, **kw)
    freq, axis = [5e5 ** (-p / pairs) for p in range(pairs)], [a for a, m in enumerate(sections or (pairs,)) for _ in range(m)]
    for got, x, i in ((rq, q, 0), (rk, k, 1)):
        assert got.dtype is x.dtype and got.shape == x.shape and got.is_contiguous()
        check(got, x, pos, freq, axis, neighbours, w[i] if norm else None, 1e-5)


@pytest.mark.parametrize("far", [1 << 17, 1 << 30, 2 ** 31 - 1])
def test_far_and_negative_positions(kvops, far):
    """The 64-bit angle is off by 2^-52 of itself: 2^-21 at 2^31, counted on top."""
    _, q, k, pos, _ = inputs("f32", 64, 2, 1, 128, 2, far)
    pos[::2] *= -1
    rot = kvops.Rotary(128, sections=(32, 32))
    rq, _ = kvops.rotate(q, k, pos, rot)
    w, r = want(q, pos, [1e4 ** (-p / 64) for p in range(64)], [p // 32 for p in range(64)], False)
    assert bool(((rq.cpu().double() - w).abs() <= (2.0 ** -19 + far * 2.0 ** -52) * r + 2.0 ** -24 * w.abs()).all())


def test_own_frequencies_axis_orders_and_one_axis_vectors(kvops):
    _, q, k, pos, _ = inputs("bf16", 19, 4, 2, 64, 3, 900)
    freq, axis = [0.5 / (1 + p) ** 2 for p in range(32)], [p % 3 for p in range(32)]
    rq, rk = kvops.rotate(q, k, pos, kvops.Rotary(64, freq=freq, axis=axis))
    check(rq, q, pos, freq, axis, False), check(rk, k, pos, freq, axis, False)
    one = kvops.Rotary(64, freq=freq)
    flat = pos[:, 1]  # a strided vector
    rq, none = kvops.rotate(q, None, flat, one)
    assert none is None
    check(rq, q, flat[:, None], freq, [0] * 32, False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_strides_weights_and_what_lies_between(kvops, dtype):
    qkv, q, k, pos, w = inputs(dtype, 21, 6, 2, 64, 1, 3000)
    before = qkv.clone()
    rot = kvops.Rotary(64, pairs=16)
    w32 = [x.float() for x in w]
    a = kvops.rotate(q, k, pos, rot, q_weight=w32[0], k_weight=w32[1], eps=1e-6)
    assert torch.equal(qkv, before)
    version = qkv._version
    b = kvops.rotate(q, k, pos, rot, q_weight=w[0], k_weight=w[1], eps=1e-6, q_out=q, k_out=k)
    assert b[0].data_ptr() == q.data_ptr() and qkv._version > version
    assert torch.equal(a[0], q) and torch.equal(a[1], k) and torch.equal(qkv[:, 8 * 64:], before[:, 8 * 64:])
    check(a[0], before[:, :6 * 64].view(21, 6, 64), pos, [1e4 ** (-p / 16) for p in range(16)], [0] * 16, False, w[0], 1e-6)


def test_values_that_are_not_finite_stay_in_their_pairs(kvops):
    _, q, k, pos, _ = inputs("f32", 2, 2, 1, 128, 1, 50)
    q[0, 0, 3], q[0, 1, 100], q[1, 0, 127] = math.nan, math.inf, -math.inf
    rq, _ = kvops.rotate(q, k, pos, kvops.Rotary(128, pairs=40))
    bad = ~rq.isfinite()
    where = torch.zeros_like(bad)
    where[0, 0, 3] = where[0, 0, 43] = where[0, 1, 100] = where[1, 0, 127] = True  # the last two do not turn
    assert torch.equal(bad, where) and rq[0, 1, 100] == math.inf and rq[1, 0, 127] == -math.inf


def test_no_tokens_a_graph_and_a_side_stream(kvops):
    rot = kvops.Rotary(128, sections=(16, 24, 24))
    _, q, k, pos, _ = inputs("bf16", 12, 16, 2, 128, 3, 999)
    assert kvops.rotate(q[:0], k[:0], pos[:0], rot)[0].shape == (0, 16, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = kvops.rotate(q, k, pos, rot)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = kvops.rotate(q, k, pos, rot)
    graph.replay()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    pos += 5
    graph.replay()
    assert torch.equal(kvops.rotate(q, k, pos, rot)[0], b[0]) and not torch.equal(a[0], b[0])


def test_rotations_of_a_step_and_of_the_operator_agree(kvops):
    """The engine's step rotates its keys by the same three axes: a key it cached at some position is the operator's."""
    from rapidocrvl_b200 import LoadOptions, Runtime, config, synth

    d = synth.ensure("tiny", "q8")
    cfg = config.load(d)
    rt = Runtime.load(d, LoadOptions(quantization="q8", max_position=1024, kv_pool_bytes=32 << 20))
    try:
        rows = []
        for thw in ((0, 0, 0), (700, 30, 401)):  # the first is not turned at all
            seq = rt.new_sequence(4)
            rt.step([seq], ids=[17], positions=[thw])
            rows.append(torch.from_numpy(seq.read_kv(0)[0]).view(1, cfg.num_key_value_heads, cfg.head_dim).cuda())
            seq.close()
        rot = kvops.Rotary(cfg.head_dim, theta=cfg.rope_theta, sections=cfg.mrope_section)
        got, _ = kvops.rotate(rows[0], None, torch.tensor([[700, 30, 401]], dtype=torch.int32, device="cuda"), rot)
        r = rows[0].abs().max()
        assert bool(((got - rows[1]).abs() <= 2.0 ** -18 * r).all())  # both sides are off by 2^-19
    finally:
        rt.close()


def test_refusals(kvops):
    qkv, q, k, pos, w = inputs("bf16", 4, 2, 1, 64, 1, 50)
    rot = kvops.Rotary(64)
    for bad in (lambda: kvops.Rotary(100), lambda: kvops.Rotary(264), lambda: kvops.Rotary(64, pairs=36), lambda: kvops.Rotary(64, pairs=6), lambda: kvops.Rotary(64, sections=(16, 24)),
                lambda: kvops.Rotary(64, sections=(16, 24, -8)), lambda: kvops.Rotary(64, axis=[0] * 31), lambda: kvops.Rotary(64, axis=[-1] * 32), lambda: kvops.Rotary(64, axis=[8] * 32),
                lambda: kvops.Rotary(64, freq=[1.0]), lambda: kvops.Rotary(64, freq=[math.inf] * 32), lambda: kvops.Rotary(64, sections=(32,), axis=[0] * 32),
                lambda: kvops.Rotary(64, theta=0), lambda: kvops.Rotary(64, theta=-2.0), lambda: kvops.Rotary(64, theta=math.nan),
                lambda: kvops.rotate(q, k, pos, None), lambda: kvops.rotate(q.cpu(), k, pos, rot), lambda: kvops.rotate(q, k.cpu(), pos, rot), lambda: kvops.rotate(q, k.float(), pos, rot),
                lambda: kvops.rotate(q.int(), k, pos, rot), lambda: kvops.rotate(qkv, k, pos, rot), lambda: kvops.rotate(q, k[:3], pos, rot), lambda: kvops.rotate(q, k, pos.long(), rot),
                lambda: kvops.rotate(q, k, pos[:3], rot), lambda: kvops.rotate(q, k, pos.expand(4, 2), rot), lambda: kvops.rotate(q, k, pos.cpu(), rot),
                lambda: kvops.rotate(q[..., :32], k, pos, rot), lambda: kvops.rotate(q.transpose(0, 1), k, pos, rot), lambda: kvops.rotate(q, k, pos, rot, q_weight=w[0]),
                lambda: kvops.rotate(q, None, pos, rot, k_weight=w[0]), lambda: kvops.rotate(q, k, pos, rot, q_weight=w[0], k_weight=w[1].float()),
                lambda: kvops.rotate(q, k, pos, rot, q_weight=w[0].half(), k_weight=w[1].half()), lambda: kvops.rotate(q, k, pos, rot, q_weight=w[0][:32], k_weight=w[1]),
                lambda: kvops.rotate(q, k, pos, rot, q_out=k), lambda: kvops.rotate(q, None, pos, rot, k_out=k), lambda: kvops.rotate(q, k, pos, rot, eps="x"),
                lambda: kvops.rotate(q.float().requires_grad_(), k.float(), pos, rot)):
        with pytest.raises(ValueError):
            bad()
    from rapidocrvl_b200._lib import OcrvlError

    odd = torch.zeros(4 * 2 * 64 + 8, dtype=torch.bfloat16, device="cuda")[4:-4].view(4, 2, 64)
    for bad in (lambda: kvops.rotate(odd, k, pos, rot), lambda: kvops.rotate(q, k, pos, rot, q_out=odd), lambda: kvops.rotate(q, k, pos, rot, q_weight=w[0], k_weight=w[1], eps=-1.0),
                lambda: kvops.rotate(q, k, pos, rot, q_weight=w[0], k_weight=w[1], eps=math.nan)):
        with pytest.raises(OcrvlError):
            bad()
