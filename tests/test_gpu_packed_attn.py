"""kvops.tree_attention over a packed cache against a plain implementation in 64 bits.

Drafts, masks, types and the tolerances' base are test_gpu_kvops.py's: the numbers of a packed
cache are exact, so only the products' roundings count.  f32: codes meet all 24 bits of q
and of the weights.  16 bits: a score's group of 32 dims is summed from -24 sum q on, magnitudes of at
most 31 sum |q| <= 31 * 32 * 1.5 (2^10.6) here, in about four cut steps of 2^-23: 2^-10.4, times the group's scale
(at most 0.5) and the softmax's (2^-3.5), over four groups: 2^-12.9 at the very most, 1.3e-4 of a weight and in the lse."""
import math

import pytest
import torch

from test_gpu_kvops import TYPES, Setup, kvops, masks  # noqa: F401 (kvops: the fixture)
from test_gpu_kvops_edges import MANY_ROWS, MANY_TILES, check, want, want_nonfinite
from test_gpu_packed import ints, quantised

pytestmark = pytest.mark.gpu

EXTRA = {"f32": 0.0, "f16": 1.3e-4, "bf16": 1.3e-4}


def numbers(codes, scales):
    """What rows of bytes and scales stand for, in 64 bits, on the rows' device."""
    G = codes.shape[-1] // 16
    b = codes.long().unflatten(-1, (-1, 2))
    half = (b[..., 0] + 256 * b[..., 1]).unflatten(-1, (8, G)).transpose(-1, -2)  # [..., group, halfword]
    c = torch.stack([(half >> 4 * i) % 16 - 8 for i in range(4)], -1).flatten(-2).double()
    return (c * scales.double()[..., None]).flatten(-2)


class Packed(Setup):
    """A packed cache of random codes and five-bit scales; NaN scales where no position is."""

    def __init__(self, kvops, dtype, lens, counts, heads=16, kv_heads=2, dim=128, page=16, layers=1, seed=0, room=0, scale=0.35, one_pool=False):
        super().__init__(kvops, dtype, lens, counts, heads, kv_heads, dim, page, layers, seed, room)
        there = ~self.pool.isnan().any(-1).cpu()  # [pages, layers, kv heads, k or v, page]
        g = torch.Generator().manual_seed(seed + 1)
        u = torch.randint(1, 16, (2,) + self.pool[:, :, :, 0].shape, generator=g)
        m = torch.randint(16, 32, u.shape[:-1] + (dim // 32,), generator=g) / 32 * scale
        scales = torch.frexp(m)  # scale itself need not have five bits
        m = torch.ldexp(torch.round(scales.mantissa * 32) / 32, scales.exponent)
        m = torch.where(there.permute(3, 0, 1, 2, 4)[..., None], m, math.nan).to(torch.bfloat16)
        nib = u.unflatten(-1, (dim // 32, 8, 4)).transpose(-2, -3).flatten(-3)  # [halfword][group][dim] in order
        codes = (nib[..., 0::2] + 16 * nib[..., 1::2]).to(torch.uint8)
        if one_pool:  # keys and values as views of one tensor, heads outermost
            codes, m = (x.permute(1, 3, 2, 0, 4, 5).contiguous().permute(3, 0, 2, 1, 4, 5) for x in (codes.cuda(), m.cuda()))
        self.codes, self.scales = codes.cuda(), m.cuda()
        self.table = self.table_h.cuda()
        self.remake(kvops)

    def remake(self, kvops):
        self.cache = kvops.PackedCache(self.codes[0], self.codes[1], self.scales[0], self.scales[1], self.table)

    def rows(self, b, layer=0, n=None):
        t = torch.arange(self.lens_h[b] if n is None else n, device="cuda")
        pages = self.table_h[b].cuda()[t // self.page].long()
        return tuple(numbers(self.codes[i][pages, layer, :, t % self.page], self.scales[i][pages, layer, :, t % self.page]).cpu() for i in range(2))

    def ok(self, got, wanted=None, extra=0.0):
        check(self, got, wanted or want(self), EXTRA[self.name] + extra)


def test_the_formats_of_the_tests_agree():
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(0))
    codes, scales, n = quantised(x.double())
    assert torch.equal(numbers(codes, scales), n)


ANY = [([1], [1]), ([0], [1]), ([0], [64]), ([648], [1]), ([15, 16, 17, 0, 129], [1, 2, 3, 4, 5]), ([300, 0, 77], [16, 0, 33]), ([2000, 31], [1, 7]),
       ([5], [0]), ([700], [2])]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,counts", ANY)
def test_attention(kvops, dtype, lens, counts):
    s = Packed(kvops, dtype, lens, counts, seed=1)
    s.ok(s.run(kvops))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (32, 8, 64, 32), (8, 8, 64, 64), (12, 4, 128, 128), (16, 1, 128, 16),
                                                    (3, 3, 64, 16), (7, 1, 128, 1024), (16, 2, 64, 16)])
def test_head_layouts(kvops, dtype, heads, kv_heads, dim, page):
    s = Packed(kvops, dtype, [211, 40], [5, 21], heads, kv_heads, dim, page, seed=heads)
    s.ok(s.run(kvops))


@pytest.mark.parametrize("dtype,dim", [("f32", 128), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("counts", [[1], [2], [4]])
def test_long_cache_is_split(kvops, dtype, dim, counts):
    s = Packed(kvops, dtype, [9001], counts, dim=dim, seed=3)
    s.ok(s.run(kvops))


def test_many_sequences(kvops):
    lens = [(37 * b) % 90 for b in range(150)]
    s = Packed(kvops, "bf16", lens, [b % 4 for b in range(150)], heads=4, dim=64, seed=5)
    s.ok(s.run(kvops))
    lens = [(97 * b) % 2900 for b in range(60)]  # runs over several segments
    s = Packed(kvops, "f32", lens, [b % 2 for b in range(60)], seed=6)
    s.ok(s.run(kvops, max_draft=1))


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 128)])
@pytest.mark.parametrize("shape", MANY_ROWS)
def test_many_rows(kvops, shape, dtype, dim):
    lens, counts, most = MANY_ROWS[shape]
    s = Packed(kvops, dtype, lens, counts, dim=dim, seed=61)
    s.ok(s.run(kvops, max_draft=most))


# Rows a kv head 6 to 96, a few short caches to many and long ones: blocks of 8, 16 and 32 rows, one and several a segment, clusters of
# one to eight, runs, and the fifth generation's products, each with drafts in one block and in several.
SHAPES = [([300], [3]), ([300] * 5, [2] * 5), ([1500] * 9, [1] * 9), ([700] * 40, [1 + b % 4 for b in range(40)]), ([9000, 20], [4, 4]), ([20000], [2]), ([20000], [3]),
          ([30, 2900] * 10, [12, 1] * 10), ([2500] * 20, [4] * 20), ([(251 * b) % 1200 for b in range(90)], [b % 3 for b in range(90)]), ([6000] * 3, [12, 7, 0])]


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f16", 128), ("f32", 128), ("f32", 64)])
@pytest.mark.parametrize("lens,counts", SHAPES)
def test_shapes(kvops, lens, counts, dtype, dim):
    s = Packed(kvops, dtype, lens, counts, dim=dim, seed=33)
    s.ok(s.run(kvops, max_draft=max(counts)))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_calls_behind_one_another_without_a_wait(kvops, dtype):
    """A launch may begin before the one before it ends: it has to wait for what that one writes, and for what it reads."""
    t, g = TYPES[dtype], torch.Generator().manual_seed(9)
    rot = kvops.Rotary(128, sections=(32, 32))
    x = torch.randn(40, 8 + 2 * 2, 128, generator=g).to(t).cuda()
    pos = torch.randint(0, 500, (40, 2), generator=g, dtype=torch.int32).cuda()
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    mask, indptr = masks([1 << i | 1 for b in range(4) for i in range(10)]), ints([0, 10, 20, 30, 40])

    def steps(wait):
        cache = kvops.PackedCache.empty(4 * 30, 1, 2, 128, torch.arange(120, dtype=torch.int32, device="cuda").view(4, 30))
        lens, out, y = ints([0, 3, 17, 40]), [], x.clone()
        q, k, v = y[:, :8], y[:, 8:10], y[:, 10:]
        for i in range(30):
            kvops.rotate(q, k, pos, rot, q_out=q, k_out=k)
            if wait:
                torch.cuda.synchronize()
            o, lse = kvops.tree_attention(q, k, v, cache, lens, indptr, mask, max_draft=10)
            if wait:
                torch.cuda.synchronize()
            new = kvops.append(cache, k[None], v[None], lens, indptr)
            if wait:
                torch.cuda.synchronize()
            kk, vv = kvops.read(cache, lens, indptr, 40, dtype=t)
            if wait:
                torch.cuda.synchronize()
            k.copy_(kk[0]), v.copy_(o[:, ::4])
            lens = new
            out += [o, lse, kk, vv, new]
        torch.cuda.synchronize()
        return out

    a = steps(True)
    for _ in range(3):
        assert all(torch.equal(m, n) for m, n in zip(a, steps(False)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_second_layer_strides_and_one_pool(kvops, dtype):
    s = Packed(kvops, dtype, [50, 33], [3, 9], layers=3, seed=8, one_pool=True)
    assert s.cache.k.stride(3) == 64 and not s.cache.k.is_contiguous()
    N = s.q.shape[0]
    fused = torch.full((N, 16 + 4 + 1, 128), math.nan, device="cuda", dtype=s.dtype)  # q | k | v side by side, and a gap
    fused[:, :16], fused[:, 16:18], fused[:, 18:20] = s.q, s.k, s.v
    s.q, s.k, s.v = fused[:, :16], fused[:, 16:18], fused[:, 18:20]
    out = torch.full((N, 17, 128), 7.0, device="cuda", dtype=s.dtype)
    rows = s.rows
    s.rows = lambda b: rows(b, layer=2)
    s.ok(s.run(kvops, layer=2, out=out[:, :16]))
    assert bool((out[:, 16] == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masks_that_leave_a_row_empty(kvops, dtype):
    s = Packed(kvops, dtype, [0, 40, 0], [3, 2, 40], seed=9)
    m = s.mask.clone()
    m[0] = m[2] = m[3] = m[10] = 0
    s.mask = m
    s.ok(s.run(kvops))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,dim", [("f32", 128), ("f16", 64), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("shape", [*MANY_ROWS, "few rows", "one row"])
def test_rows_get_the_values_they_see(kvops, shape, dtype, dim, bad):
    """As for a plain cache: a draft's value that is not finite reaches the rows that see it, in its dims alone."""
    lens, counts, most = {**MANY_ROWS, "few rows": ([40, 7], [2, 1], 2), "one row": ([300, 0], [1, 1], 1)}[shape]
    s = Packed(kvops, dtype, lens, counts, dim=dim, seed=62)
    starts = s.indptr.tolist()
    for b, t in enumerate(counts):
        if t:
            s.v[starts[b] + t // 2, b % 2, [1, dim // 2 - 1, dim // 2, dim - 2][b % 4]] = bad
    for d in (0, dim // 2 + 1):
        s.v[starts[0], 1, d] = bad
    s.ok(s.run(kvops, max_draft=most), want_nonfinite(s))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts,heads", [([4, 1], 4), ([6, 20], 16)])
def test_masked_keys_may_hold_anything(kvops, dtype, counts, heads, bad):
    s = Packed(kvops, dtype, [40, 7], counts, heads=heads, seed=11)
    s.mask = masks([1 << i | (i > 0) for t in counts for i in range(t)])
    s.k[3], s.v[3] = bad, bad  # only token 3 sees it
    got = s.run(kvops)
    s.k[3], s.v[3] = 0.5, 0.5
    rest = [i for i in range(sum(counts)) if i != 3]
    s.ok([x[rest] for x in got], [x[rest] for x in want(s)])


@pytest.mark.parametrize("big", [torch.finfo(torch.float32).min, torch.finfo(torch.float32).max, 3.402e38])
@pytest.mark.parametrize("counts,heads", [([6, 1], 4), ([20, 3], 16), ([64, 3], 16)])
def test_f32_drafts_as_large_as_the_type_goes(kvops, counts, heads, big):
    s = Packed(kvops, "f32", [40, 300], counts, heads=heads, seed=63)
    s.mask = masks([1 << i | (i > 0) for t in counts for i in range(t)])
    s.k[3], s.v[3] = big, big
    got = s.run(kvops)
    s.k[3], s.v[3] = 0.5, 0.5
    rest = [i for i in range(sum(counts)) if i != 3]
    s.ok([x[rest] for x in got], [x[rest] for x in want(s)])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinite_drafted_keys_that_are_seen(kvops, dtype):
    """A key with one infinite dim: its score is that infinity's with the query's sign, so it takes nothing or leaves NaN."""
    s = Packed(kvops, dtype, [40], [2], heads=4, seed=64)
    s.mask = masks([3, 3])
    s.k[1, :, 5] = math.inf
    s.q[:, :, 5] = -s.q[:, :, 5].abs() - 0.25
    s.ok(s.run(kvops))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts,most", [([1, 1], 1), ([9, 64], 64)])
def test_scales_that_are_not_numbers(kvops, dtype, counts, most):
    """A group that was written from values that are not finite: a key's makes the row NaN, a value's its 32 dims."""
    s = Packed(kvops, dtype, [70, 200], counts, seed=65)
    p0, p1 = int(s.table_h[0, 2]), int(s.table_h[1, 5])
    s.scales[0][p0, 0, 1, 3, 2] = math.nan
    s.scales[1][p1, 0, 0, 15, 1] = math.nan
    out, lse = s.run(kvops, max_draft=most)
    n = counts[0]
    assert bool(out[:n, 8:].isnan().all()) and bool(lse[:n, 8:].isnan().all())
    bad = out[n:, :8].isnan()
    assert bool(bad[..., 32:64].all()) and not bool(bad[..., :32].any() or bad[..., 64:].any())
    s.scales[0][p0, 0, 1, 3, 2] = s.scales[1][p1, 0, 0, 15, 1] = 0.25
    w = want(s)
    s.ok((out[:n, :8], lse[:n, :8]), [x[:n, :8] for x in w])
    s.ok((out[n:, 8:], lse[n:, 8:]), [x[n:, 8:] for x in w])


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 128)])
@pytest.mark.parametrize("shape", MANY_TILES)
def test_unmapped_pages_and_nothing_to_see(kvops, shape, dtype, dim):
    lens, counts, most = MANY_TILES[shape]
    s = Packed(kvops, dtype, lens, counts, dim=dim, seed=72)
    starts = s.indptr.tolist()
    mapped = [torch.ones(n, dtype=torch.bool) for n in lens]
    for page in list(range(17)) + [20, 23, 40, 55]:
        if page * 16 < lens[0]:
            s.table[0, page] = -1 if page % 2 else 1 << 30
            mapped[0][page * 16:(page + 1) * 16] = False
    for page in range(-(-lens[1] // 16)):  # the second sequence has nothing cached
        s.table[1, page] = s.codes.shape[1] if page % 3 else -5
        mapped[1][page * 16:(page + 1) * 16] = False
    bits = s.mask.tolist()
    for i in [*range(starts[1], starts[2], 2), *range(starts[0], starts[1], 3)]:
        bits[i] = 0
    s.mask = masks(bits)
    s.ok(s.run(kvops, max_draft=most), want(s, see_cached=mapped))


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 128)])
@pytest.mark.parametrize("shape", MANY_TILES)
def test_scores_that_rise_along_the_context(kvops, shape, dtype, dim):
    """As for a plain cache: some rows' scores rise by 16 powers of two every 32 positions of some tiles and by 100
    at once further on, others fall alike.  Group 0's scale carries that, 2^-20 of a score's size is allowed for its
    sum's roundings; 16 bits: 24 sum q cancels, 4 |c| at most, in two more bits."""
    lens, counts, most = MANY_TILES[shape]
    s = Packed(kvops, dtype, lens, counts, dim=dim, seed=71)
    s.q[:, :, :32] = 0
    s.q[:, ::2, 0], s.q[:, 1::2, 0] = 4, -4
    s.codes[0][..., 0] |= 0x0f  # dim 0 is the lowest nibble of the first byte: 7
    per = 4 * 7 * s.scale / math.log(2)  # powers of two a unit of the scale
    for b, n in enumerate(lens):
        t = torch.arange(n)
        steps = torch.cumsum((t % 32 == 0) & (t // 128 % 7 % 3 == 1) & (t < 2300), 0).clamp(max=12) * 16 + (t >= 700) * 100
        pages = s.table_h[b, t // s.page].long().cuda()
        m = torch.frexp(steps / per)
        five = torch.ldexp(torch.round(m.mantissa * 32) / 32, m.exponent).to(torch.bfloat16)
        for g in range(2):
            s.scales[0][pages, 0, g, (t % s.page).cuda(), 0] = five.cuda()
    w = want(s)
    size = float(w[1][torch.isfinite(w[1])].abs().max())
    s.ok(s.run(kvops, max_draft=most), w, extra=2.0 ** (-20 if dtype == "f32" else -18) * size)


def test_lengths_past_the_table_and_large_scores(kvops):
    s = Packed(kvops, "f32", [48], [1], seed=14)
    s.lens = ints([1 << 30])  # counts as the table's 64, whose 4th page is unmapped
    s.ok(s.run(kvops))
    s.lens = ints([-7])
    s.lens_h = [0]
    s.ok(s.run(kvops))
    for dtype in ("bf16", "f32"):
        s = Packed(kvops, dtype, [200], [4], seed=15)
        s.scale = 12.0  # scores of several hundred: one position takes all
        _, lse = s.run(kvops)
        w_lse = want(s)[1]
        assert float(((lse.cpu().double() - w_lse) / w_lse.abs()).abs().max()) <= 4e-6
        s.scale = 0.0
        s.ok(s.run(kvops))
        s.scale = -0.1
        s.ok(s.run(kvops))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [2.0 ** -9, 2.0 ** 12])
@pytest.mark.parametrize("drafts", [False, True])
def test_small_and_large_numbers(kvops, dtype, scale, drafts):
    """Values of a thousandth, or thousands: the output's error stays that of its own size (f16 holds them exactly
    from 2^-14 on).  Where the drafts' keys are not scaled along, their scores reach 2,300 with the first scale: a score x
    is rounded to 2^-24 of itself a few times (its sum, the factor, the difference to the maximum), 2^-20 x of a weight."""
    s = Packed(kvops, dtype, [900, 40], [2, 30], seed=66, scale=scale)
    s.v *= scale
    if drafts:
        s.k *= scale
    s.scale = 0.1 / scale
    w = want(s)
    s.ok(s.run(kvops), w, extra=3 * EXTRA[dtype] + 2.0 ** -20 * float(w[1].abs().max()))  # the cache's scores are up to four times those above


@pytest.mark.parametrize("n,most", [(1 << 17, 8), (1 << 20, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_long_tails_are_in_the_sum(kvops, n, most, dtype):
    """One position far above all others, each of which has 2^-24 to 2^-27 of its weight: together a 400th or a 50th of the sum."""
    t, B, heads, dim, page = TYPES[dtype], 74, 16, 64, 1024
    pages = n // page
    codes = torch.full((2, 128, 1, 2, page, dim // 2), 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, 128, 1, 2, page, 2), 0.125, dtype=torch.bfloat16, device="cuda")
    codes[1] = torch.randint(0xc, 0x10, codes[1].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(65)).to(torch.uint8) * 0x11
    codes[0, 0, :, :, 0, 0] = 0x8f  # the strong position: dim 0 is 7 / 8, its values 0
    codes[1, 0, :, :, 0] = 0x88
    row = torch.arange(pages, dtype=torch.int32)
    row[128:] = row[128:] % 127 + 1
    cache = kvops.PackedCache(codes[0], codes[1], scales[0], scales[1], row.cuda().repeat(B, 1))
    counts = [most] + [1] * (B - 1)
    N = sum(counts)
    q = torch.zeros(N, heads, dim, dtype=t, device="cuda")
    q[:, :, 0] = torch.linspace(16.0, 18.0, heads, device="cuda").to(t)
    kv = torch.zeros(N, 2, dim, dtype=t, device="cuda")
    scale = 25.6 * math.log(2) / 17.0 / 0.875
    out, lse = kvops.tree_attention(q, kv, kv, cache, torch.full((B,), n, dtype=torch.int32, device="cuda"), ints([0] + [sum(counts[:b + 1]) for b in range(B)]),
                                    torch.zeros(N, dtype=torch.int64, device="cuda"), max_draft=most, scale=scale)
    v = numbers(codes[1], scales[1])[row.cuda().long(), 0].sum((0, 2)).repeat_interleave(heads // 2, 0)
    x = q[0, :, 0].double() * scale * 0.875
    w = torch.exp(-x)[:, None]
    w_out, w_lse = v * w / (1 + (n - 1) * w), x + torch.log1p((n - 1) * w[:, 0])
    # 16 bits: the strong score is off by the cancelling sum's roundings, 24 * 18 in at most four steps of 2^-23
    extra = 0.0 if dtype == "f32" else 4 * 24 * 18 * 2.0 ** -23 * 0.125 * scale
    assert bool(((lse - w_lse).abs() <= 1e-5 + extra).all()), float((lse - w_lse).abs().max())
    if dtype != "bf16":  # bf16's sums of values are the instruction's own, cut ones
        a, r = {"f32": (1e-5, 0.0), "f16": (2.0 ** -11, 2.0 ** -12)}[dtype]
        assert bool(((out - w_out).abs() <= a + (r + extra) * w_out).all()), float((out - w_out).abs().max())


def test_same_bits_every_time_on_a_side_stream_and_with_a_workspace(kvops):
    for dtype, counts in (("bf16", [5, 9]), ("f32", [1, 2]), ("f16", [1, 1])):
        s = Packed(kvops, dtype, [3000, 200], counts, seed=16)
        a, la = s.run(kvops)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b, lb = s.run(kvops)
        side.synchronize()
        most = max(counts)
        work = torch.full((s.cache.work_bytes(16, most, s.dtype),), 0xff, dtype=torch.uint8, device="cuda")
        c, lc = s.run(kvops, max_draft=most, work=work)
        d, ld = s.run(kvops, max_draft=most, work=work)
        assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(c, d) and torch.equal(lc, ld)
        s.ok((c, lc))


def test_two_graphs_that_share_a_workspace(kvops):
    s, r = Packed(kvops, "f32", [3000, 30], [1, 1], seed=17), Packed(kvops, "bf16", [2500, 700], [2, 1], seed=18)
    work = torch.empty(max(s.cache.work_bytes(16, 2), r.cache.work_bytes(16, 2, torch.bfloat16)), dtype=torch.uint8, device="cuda")
    s.run(kvops, max_draft=2, work=work), r.run(kvops, max_draft=2, work=work)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (s, r):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(x.run(kvops, max_draft=2, work=work))
    s.lens.copy_(torch.tensor([333, 12]))
    s.lens_h = [333, 12]
    for g in (*graphs, *graphs):  # one behind the other, on one stream
        g.replay()
    torch.cuda.synchronize()
    s.ok(outs[0])
    r.ok(outs[1])


def test_fewer_drafts_than_the_call_may_have_and_rows_behind_the_last(kvops):
    for dtype in ("f32", "bf16"):
        s = Packed(kvops, dtype, [5000, 40, 0], [1, 20, 3], seed=19)
        N = s.q.shape[0]
        pad = torch.zeros(4, 16, 128, dtype=s.dtype, device="cuda")  # tokens of no sequence
        q, k, v = torch.cat((s.q, pad)), torch.cat((s.k, pad[:, :2])), torch.cat((s.v, pad[:, :2]))
        mask = torch.cat((s.mask, s.mask[:4]))
        out, lse = torch.full_like(q, 7.0), torch.full((N + 4, 16), 7.0, device="cuda")
        kvops.tree_attention(q, k, v, s.cache, s.lens, s.indptr, mask, scale=s.scale, max_draft=64, out=out, lse=lse)
        s.ok((out[:N], lse[:N]))
        assert bool((out[N:] == 7).all()) and bool((lse[N:] == 7).all())
        out.fill_(7)
        kvops.tree_attention(q, k, v, s.cache, s.lens, s.indptr, mask, scale=s.scale, max_draft=16, out=out, lse=lse)
        assert bool((out[17:21] == 7).all())  # the second sequence's tokens past max_draft are not computed
        a = torch.cat((out[:17], out[21:N])), torch.cat((lse[:17], lse[21:N]))
        w = want(s)
        rest = [i for i in range(N) if not 17 <= i < 21]
        s.ok(a, [x[rest] for x in w])


def test_pages_past_32_bits(kvops):
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 13 GB")
    for dtype, counts in (("f32", [16, 1]), ("bf16", [1, 2]), ("bf16", [3, 40])):
        s = Packed(kvops, dtype, [700, 3000], counts, heads=8, seed=95)
        near = s.run(kvops)
        pages, far = s.codes.shape[1], -(-(5 << 30) // s.codes[0, 0].nbytes)
        codes = torch.empty((2, far + pages) + s.codes.shape[2:], dtype=torch.uint8, device="cuda")
        scales = torch.empty((2, far + pages) + s.scales.shape[2:], dtype=torch.bfloat16, device="cuda")
        codes[:, far:], scales[:, far:] = s.codes, s.scales
        s.codes, s.scales, s.table = codes, scales, torch.where(s.table >= 0, s.table + far, s.table)
        s.remake(kvops)
        assert all(torch.equal(a, b) for a, b in zip(near, s.run(kvops)))
        del s, codes, scales


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_step_after_another(kvops, dtype):
    """Prompts, then drafted steps as a decoder takes them: rotate, attend, append the accepted path, read back."""
    t, layers, heads, kv_heads, dim = TYPES[dtype], 2, 8, 2, 128
    g = torch.Generator().manual_seed(5)
    B, room = 3, 6
    table = torch.randperm(B * room, generator=g).to(torch.int32).view(B, room).cuda()
    cache = kvops.PackedCache.empty(B * room, layers, kv_heads, dim, table)
    rot = kvops.Rotary(dim, sections=(16, 24, 24))
    w = (1 + 0.1 * torch.randn(dim, generator=g)).cuda()
    lens, held = ints([0] * B), [torch.zeros(2, layers, 0, kv_heads, dim, dtype=torch.float64) for _ in range(B)]
    for counts, paths in (([30, 1, 47], None), ([4, 1, 7], [[0, 2], [0], [0, 1, 5]]), ([1, 3, 0], [[0], [0, 1, 2], []])):
        N = sum(counts)
        starts = [0] + [sum(counts[:b + 1]) for b in range(B)]
        indptr = ints(starts)
        keys, values = [], []
        for layer in range(layers):
            qkv = torch.randn(N, (heads + 2 * kv_heads) * dim, generator=g).to(t).cuda()
            q, k, v = (x.view(N, -1, dim) for x in qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), 1))
            pos = torch.randint(0, 2000, (N, 3), generator=g, dtype=torch.int32).cuda()
            kvops.rotate(q, k, pos, rot, q_weight=w, k_weight=w, q_out=q, k_out=k)
            keys.append(k), values.append(v)
            if paths is not None:  # drafts (each sees itself and the first) over what the cache holds
                s = Setup.__new__(Setup)
                s.name, s.q, s.k, s.v, s.indptr, s.counts, s.kv_heads, s.heads, s.scale = dtype, q, k, v, indptr, counts, kv_heads, heads, dim ** -0.5
                s.mask = masks([1 << i | 1 for n in counts for i in range(n)])
                s.rows = lambda b: (held[b][0, layer], held[b][1, layer])
                got = kvops.tree_attention(q, k, v, cache, lens, indptr, s.mask, layer=layer)
                check(s, got, want(s), EXTRA[dtype])
        k, v = torch.stack(keys), torch.stack(values)
        took = [list(range(n)) for n in counts] if paths is None else paths
        most = max(map(len, took))
        how = {} if paths is None else dict(path=ints([p + [0] * (most - len(p)) for p in took]), n_path=ints([len(p) for p in took]))
        before = lens
        lens = kvops.append(cache, k, v, lens, indptr, **how)
        assert lens.tolist() == [n + len(p) for n, p in zip(before.tolist(), took)]
        both = torch.stack((k, v)).cpu().double()
        for b, p in enumerate(took):
            held[b] = torch.cat((held[b], quantised(both[:, :, [starts[b] + i for i in p]])[2]), 2)
    k, v = kvops.read(cache, ints([0] * B), ints([0] + torch.cumsum(lens, 0).tolist()), int(lens.sum()), dtype=torch.float32)
    assert torch.equal(torch.stack((k, v)).cpu().double(), torch.cat(held, 2))


def test_refusals(kvops):
    from rapidocrvl_b200._lib import OcrvlError

    s = Packed(kvops, "bf16", [40], [3], seed=1)
    for bad in (dict(q=s.q.float()), dict(q=s.q.double(), k=s.k.double(), v=s.v.double()), dict(k=s.k[:2]), dict(v=s.v.float()), dict(k=s.k[:, :1], v=s.v[:, :1]),
                dict(mask=s.mask[:2]), dict(mask=s.mask.int()), dict(lens=s.lens.long()), dict(lens=s.lens[:0]), dict(indptr=s.indptr[:1]), dict(q=s.q.cpu()),
                dict(q=s.q[..., ::2]), dict(out=torch.empty(2, 16, 128, dtype=s.dtype, device="cuda")), dict(out=torch.empty(3, 16, 128, device="cuda")),
                dict(lse=torch.empty(3, 8, device="cuda")), dict(q=s.q.float().requires_grad_(), k=s.k.float(), v=s.v.float())):
        x = dict(q=s.q, k=s.k, v=s.v, lens=s.lens, indptr=s.indptr, mask=s.mask)
        kw = {k: bad.pop(k) for k in ("out", "lse") if k in bad}
        x.update(bad)
        with pytest.raises(ValueError):
            kvops.tree_attention(x["q"], x["k"], x["v"], s.cache, x["lens"], x["indptr"], x["mask"], **kw)
    for kw in (dict(layer=1), dict(layer=-1), dict(max_draft=0), dict(max_draft=65), dict(scale=math.nan), dict(work=torch.empty(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(OcrvlError):
            kvops.tree_attention(s.q, s.k, s.v, s.cache, s.lens, s.indptr, s.mask, **kw)
    with pytest.raises(ValueError):
        kvops.attention_mass(s.q, torch.zeros(3, 16, device="cuda"), s.cache, s.lens, s.indptr)
    with pytest.raises(ValueError):
        s.cache.work_bytes(16, 1, torch.int8)
    assert s.cache.work_bytes(16, 20) == max(s.cache.work_bytes(16, 20, t) for t in TYPES.values()) > 0


@pytest.mark.parametrize("name,drafts", [("f32", 1), ("bf16", 1), ("bf16", 64)])
def test_positions_far_inside_a_page(kvops, name, drafts):
    """One page of 2^26 positions: its codes' offsets pass 2^31 bytes at position 2^25.  Keys and values are 0 up to the 100 positions
    there, which are written, read back and attended."""
    dtype, n, D, border = TYPES[name], 100, 128, 1 << 25
    g = torch.Generator().manual_seed(3)
    base = 1.4 * torch.randn(D, generator=g)
    k = (base + 0.1 * torch.randn(1, n, 1, D, generator=g)).to(dtype)
    v = torch.randn(1, n, 1, D, generator=g).to(dtype)
    q = base.to(dtype).expand(drafts, 2, D).contiguous()
    cache = kvops.PackedCache.empty(1, 1, 1, D, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), page_size=1 << 26)
    for at in (border - n // 2, (1 << 26) - n):
        lens, indptr = ints([at]), ints([0, n])
        assert kvops.append(cache, k.cuda(), v.cuda(), lens, indptr).item() == at + n
        kr, vr = (x.cpu().double()[0, :, 0] for x in kvops.read(cache, lens, indptr, n, dtype=torch.float32))
        for x, r in ((k, kr), (v, vr)):  # half a step: 1/7 of a group's largest, rounded to five bits, by 1/2
            assert ((x.double()[0, :, 0] - r).abs() <= x.double().abs().max() / 7 * (1 + 2 ** -5) / 2 + 1e-6).all()
        if at > border:
            break
        none = torch.zeros(drafts, 1, D, dtype=dtype, device="cuda")
        out, lse = kvops.tree_attention(q.cuda(), none, none, cache, ints([at + n]), ints([0, drafts]),
                                        torch.zeros(drafts, dtype=torch.int64, device="cuda"), max_draft=drafts)
        s = kr @ q[0, 0].double() / math.sqrt(D)
        rest = at * math.exp(-s.max().item())  # the positions before them have scores of 0 and values of 0
        w = (s - s.max()).exp()
        want, want_lse = (w @ vr) / (w.sum() + rest), s.max() + (w.sum() + rest).log()
        assert rest < w.sum() / 2
        # f32: a score sums 128 products of |q k| <= 60 in all: 128 2^-24 60 = 5e-4, so a weight's is 1e-3 of it, of values up to 4.5.  bf16:
        # a weight and the output are off by 2^-8 each, and the scores' sums as above: (2^-7 + 1e-3) 4.5.
        tol = 5e-3 if name == "f32" else 4e-2
        assert vr.abs().max() <= 4.5 and (q[0, 0].double().abs() * kr.abs()).sum(1).max() / math.sqrt(D) <= 60
        assert (out.cpu().double() - want).abs().max() <= tol
        assert (lse.cpu().double() - want_lse).abs().max() <= 1e-3
