"""The paged-cache operators (rapidocrvl_b200.kvops) against plain
implementations in 64 bits.

Tolerances: for 16-bit types the output is rounded once to the type (half an
ulp: 2^-9 of the value for bf16, 2^-12 for f16) and the softmax weights once
before the product with v, whose relative error of at most 2^-9 (2^-12) a
weight carries over to the output's scale, the largest |v| seen; both together
stay under 2^-8 (2^-11) of that scale plus 2^-9 (2^-12) of the value.  f32: products keep 22
bits of each factor, so a score is off by at most about 2^-21 sum |q k| scale
plus the rounding of the sums; with |scores| up to 16 that is 1e-5 of a weight.
1e-5 of the largest |v| is allowed, lse 1e-5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
REL = {"f32": (1e-5, 0.0), "f16": (2.0 ** -11, 2.0 ** -12), "bf16": (2.0 ** -8, 2.0 ** -9)}


@pytest.fixture(scope="module")
def kvops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from rapidocrvl_b200 import kvops

    return kvops


class Setup:
    """A cache with `lens` positions a sequence in shuffled pages, garbage
    (NaN) everywhere else, and `counts` drafted tokens a sequence."""

    def __init__(self, kvops, dtype, lens, counts, heads=16, kv_heads=2, dim=128, page=16, layers=1, seed=0, room=0, junk=math.nan):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = TYPES[dtype], heads, kv_heads, dim, page
        self.name, self.lens_h, self.counts = dtype, list(lens), list(counts)
        B, N = len(lens), sum(counts)
        need = [-(-(n + room) // page) for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g).tolist()
        self.table_h = torch.full((B, max(1, max(need)) + 1), -1, dtype=torch.int32)
        pool = torch.full((pages, layers, kv_heads, 2, page, dim), junk)
        for b, n in enumerate(lens):
            for i in range(need[b]):
                p = order.pop()
                self.table_h[b, i] = p
                r = max(0, min(page, n - i * page))
                pool[p, :, :, :, :r] = torch.randn(layers, kv_heads, 2, r, dim, generator=g)
        self.pool = pool.to(self.dtype).cuda()
        self.cache = kvops.PagedCache(self.pool[:, :, :, 0], self.pool[:, :, :, 1], self.table_h.cuda())
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.indptr = torch.tensor([0] + [sum(counts[:b + 1]) for b in range(B)], dtype=torch.int32, device="cuda")
        self.q = (1.5 * torch.randn(N, heads, dim, generator=g)).to(self.dtype).cuda()
        self.k = torch.randn(N, kv_heads, dim, generator=g).to(self.dtype).cuda()
        self.v = torch.randn(N, kv_heads, dim, generator=g).to(self.dtype).cuda()
        bits = []
        for t in counts:  # random trees: each node sees itself and what its parent sees
            seen = []
            for i in range(t):
                up = int(torch.randint(0, max(i, 1), (1,), generator=g))
                seen.append((seen[up] if i else 0) | 1 << i)
            bits += seen
        self.mask = masks(bits)
        self.scale = 1 / math.sqrt(dim)

    def rows(self, b, layer=0, pool=None, n=None):
        """Keys and values of a sequence's cached positions, [n, kv heads, dim] in 64 bits."""
        n = self.lens_h[b] if n is None else n
        t = torch.arange(n)
        pages = self.table_h[b, t // self.page].long()
        x = (self.pool if pool is None else pool).cpu()[pages, layer, :, :, t % self.page].double()
        return x[:, :, 0], x[:, :, 1]

    def want(self, layer=0):
        N, H, D = self.q.shape
        out, lse = torch.zeros(N, H, D, dtype=torch.float64), torch.full((N, H), -math.inf, dtype=torch.float64)
        top = torch.zeros(N, H, 1, dtype=torch.float64)
        q, k, v = (x.cpu().double() for x in (self.q, self.k, self.v))
        for b, t in enumerate(self.counts):
            i0 = int(self.indptr[b])
            ck, cv = self.rows(b, layer)
            for i in range(t):
                m = int(self.mask[i0 + i])
                see = [i0 + j for j in range(t) if m >> j & 1]
                for h in range(H):
                    g = h * self.kv_heads // H
                    keys, values = torch.cat((ck[:, g], k[see, g])), torch.cat((cv[:, g], v[see, g]))
                    if not len(keys):
                        continue
                    s = keys @ q[i0 + i, h] * self.scale
                    lse[i0 + i, h] = torch.logsumexp(s, 0)
                    out[i0 + i, h] = torch.softmax(s, 0) @ values
                    top[i0 + i, h] = values.abs().max()
        return out, lse, top

    def run(self, kvops, **kw):
        return kvops.tree_attention(self.q, self.k, self.v, self.cache, self.lens, self.indptr, self.mask, scale=self.scale, **kw)

    def check(self, out, lse, layer=0):
        w_out, w_lse, top = self.want(layer)
        a, r = REL[self.name]
        off = (out.cpu().double() - w_out).abs()
        assert bool((off <= a * top + r * w_out.abs()).all()), float((off / top.clamp(min=1e-30)).max())
        empty = w_lse == -math.inf
        assert torch.equal(lse.cpu().double() == -math.inf, empty)
        assert float((lse.cpu().double() - w_lse)[~empty].abs().max() if (~empty).any() else 0) <= 1e-5
        assert bool((out.cpu()[empty] == 0).all())


def masks(bits):
    bits = [m & (1 << 64) - 1 for m in bits]
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in bits], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,counts", [
    ([1], [1]), ([0], [1]), ([0], [64]), ([648], [1]), ([15, 16, 17, 0, 129], [1, 2, 3, 4, 5]), ([300, 0, 77], [16, 0, 33]),
    ([1000], [64]), ([127, 128, 2049], [7, 64, 1])])
def test_tree_attention(kvops, dtype, lens, counts):
    s = Setup(kvops, dtype, lens, counts, seed=sum(lens))
    s.check(*s.run(kvops))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (32, 8, 64, 32), (8, 8, 64, 64), (12, 4, 128, 128), (16, 1, 128, 16),
                                                    (3, 3, 64, 16), (7, 1, 128, 1024)])
def test_tree_attention_head_layouts(kvops, dtype, heads, kv_heads, dim, page):
    s = Setup(kvops, dtype, [211, 40], [5, 21], heads, kv_heads, dim, page, seed=heads)
    s.check(*s.run(kvops))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tree_attention_long_cache_is_split(kvops, dtype):
    s = Setup(kvops, dtype, [9001], [2], seed=3)
    s.check(*s.run(kvops))


def test_tree_attention_many_sequences(kvops):
    lens = [(37 * b) % 90 for b in range(150)]
    s = Setup(kvops, "bf16", lens, [b % 4 for b in range(150)], heads=4, dim=64, seed=5)
    s.check(*s.run(kvops))


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("lens,counts,most", [
    ([(29 * b) % 110 for b in range(40)], [64] + [1 + b % 3 for b in range(39)], 64),  # two row blocks, more segments than SMs
    ([(29 * b) % 700 for b in range(8)], [64, 33, 0, 1, 17, 2, 5, 40], 64),  # one wave of segments
    ([9000, 5], [64, 3], 64),  # runs, two row blocks
    ([7000, 12, 900], [9, 1, 16], 16),  # runs, one row block
    ([(29 * b) % 110 for b in range(40)], [1 + b % 9 for b in range(40)], 9)])  # a wave of segments, one row block
def test_tree_attention_shapes_of_many_rows(kvops, dtype, dim, lens, counts, most):
    s = Setup(kvops, dtype, lens, counts, dim=dim, seed=len(lens) + most)
    s.check(*s.run(kvops, max_draft=most))


def test_tree_attention_second_layer_and_strides(kvops):
    s = Setup(kvops, "f32", [50, 33], [3, 9], layers=3, seed=8)
    N = s.q.shape[0]
    fused = torch.full((N, 16 + 4 + 1, 128), math.nan, device="cuda")  # q | k | v side by side, and a gap
    fused[:, :16], fused[:, 16:18], fused[:, 18:20] = s.q, s.k, s.v
    s.q, s.k, s.v = fused[:, :16], fused[:, 16:18], fused[:, 18:20]
    out = torch.full((N, 17, 128), 7.0, device="cuda")
    got, lse = s.run(kvops, layer=2, out=out[:, :16])
    s.check(got, lse, layer=2)
    assert bool((out[:, 16] == 7).all())


def test_tree_attention_masks_that_leave_a_row_empty(kvops):
    for dtype in ("f32", "bf16"):
        s = Setup(kvops, dtype, [0, 40, 0], [3, 2, 40], seed=9)
        m = s.mask.clone()
        m[0] = m[2] = m[3] = 0
        m[10] = 0
        s.mask = m
        s.check(*s.run(kvops))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tree_attention_masked_places_may_hold_anything(kvops, dtype, bad):
    """Drafts that some tokens do not see hold NaN or infinities: those tokens' rows do not change."""
    s = Setup(kvops, dtype, [40, 7], [6, 20], seed=11)
    bits = [1 << i | (1 if i else 0) for i in range(6)] + [1 << i for i in range(20)]
    s.mask = masks(bits)
    s.k[3], s.v[3] = bad, bad            # only token 3 sees draft 3 of the first sequence
    s.v[6 + 17, :, 5] = bad              # and token 17 draft 17 of the second
    out, lse = s.run(kvops)
    clean = [i for i in range(26) if i not in (3, 23)]
    s.k[3], s.v[3], s.v[23, :, 5] = 0.5, 0.5, 0.5
    w_out, w_lse, top = s.want()
    a, r = REL[dtype]
    assert bool(((out.cpu().double() - w_out).abs() <= a * top + r * w_out.abs())[clean].all())
    assert float((lse.cpu().double() - w_lse)[clean].abs().max()) <= 1e-5
    assert not bool(torch.isfinite(out[23, :, 5]).any())
    rest = [d for d in range(128) if d != 5]
    assert bool(((out.cpu().double() - w_out).abs() <= a * top + r * w_out.abs())[23][:, rest].all())


def test_tree_attention_unmapped_pages_are_not_attended(kvops):
    s = Setup(kvops, "f32", [64], [2], seed=13)
    table = s.table_h.clone()
    table[0, 1], table[0, 2] = -1, 1 << 30
    out, lse = kvops.tree_attention(s.q, s.k, s.v, kvops.PagedCache(s.pool[:, :, :, 0], s.pool[:, :, :, 1], table.cuda()),
                                    s.lens, s.indptr, s.mask, scale=s.scale)
    k, v = s.rows(0)
    keep = [t for t in range(64) if t // 16 in (0, 3)]
    s.rows = lambda b, layer=0: (k[keep], v[keep])
    s.check(out, lse)


def test_tree_attention_lengths_past_the_table_and_large_scores(kvops):
    s = Setup(kvops, "f32", [48], [1], seed=14, junk=0.0)
    s.lens = torch.tensor([1 << 30], dtype=torch.int32, device="cuda")  # counts as the table's 64; its 4th page is unmapped
    s.check(*s.run(kvops))
    s = Setup(kvops, "bf16", [200], [4], seed=15)
    s.scale = 12.0  # scores of several hundred: one position takes all
    out, lse = s.run(kvops)
    w_out, w_lse, top = s.want()
    assert float(((lse.cpu().double() - w_lse) / w_lse.abs()).abs().max()) <= 2e-6
    s.scale = 0.0
    s.check(*s.run(kvops))
    s.scale = -0.1
    s.check(*s.run(kvops))


def test_tree_attention_same_bits_every_time_and_on_a_side_stream(kvops):
    s = Setup(kvops, "bf16", [3000, 200], [5, 9], seed=16)
    a, la = s.run(kvops)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = s.run(kvops)
    side.synchronize()
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_tree_attention_in_a_graph(kvops):
    s = Setup(kvops, "f32", [500, 30], [4, 1], seed=17)
    s.run(kvops)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = s.run(kvops)
    s.lens.copy_(torch.tensor([333, 12]))
    s.lens_h = [333, 12]
    graph.replay()
    torch.cuda.synchronize()
    s.check(out, lse)


# -- attention mass -----------------------------------------------------------------

def mass_want(s, lse, counted=None, acc=None, decay=1.0, width=None):
    B = len(s.lens_h)
    out = torch.zeros(B, s.kv_heads, width, dtype=torch.float64)
    for b, n in enumerate(s.lens_h):
        n = min(n, width)
        k, _ = s.rows(b)
        if acc is not None:
            w = min(n, acc.shape[-1])
            out[b, :, :w] = decay * acc[b, :, :w].cpu().double()
        for i in range(s.counts[b]):
            if counted is not None and not counted[b] >> i & 1:
                continue
            tok = int(s.indptr[b]) + i
            for h in range(s.heads):
                l = float(lse[tok, h])
                if l > -math.inf:
                    g = h * s.kv_heads // s.heads
                    out[b, g, :n] += torch.exp(k[:n, g] @ s.q[tok, h].cpu().double() * s.scale - l)
    return out


def mass_check(got, want):
    """Each weight keeps 22 bits of its factors' products in f32 (see above) and
    the sum of up to 1,024 of them rounds at 2^-24 each: 2e-5 of the sum."""
    off = (got.cpu().double() - want).abs()
    assert bool((off <= 2e-5 * want.abs() + 1e-12).all()), float((off / want.abs().clamp(min=1e-12)).max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,counts", [([1], [1]), ([0, 5], [2, 0]), ([648], [1]), ([15, 16, 17, 0, 700], [1, 2, 3, 4, 5]), ([900], [64]),
                                         ([127, 128, 2049], [7, 33, 1])])
def test_attention_mass(kvops, dtype, lens, counts):
    s = Setup(kvops, dtype, lens, counts, seed=sum(lens) + 1)
    _, lse = s.run(kvops)
    width = s.cache.capacity
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale)
    assert got.shape == (len(lens), 2, width)
    mass_check(got, mass_want(s, lse, width=width))


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (32, 8, 64, 32), (8, 8, 64, 64), (16, 1, 128, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_mass_head_layouts_and_sums_so_far(kvops, dtype, heads, kv_heads, dim, page):
    s = Setup(kvops, dtype, [211, 40], [5, 21], heads, kv_heads, dim, page, seed=heads)
    _, lse = s.run(kvops)
    width = s.cache.capacity + 5
    acc = torch.rand(2, kv_heads, 2 * width, device="cuda")[:, :, :100]
    counted = [0b10110, (1 << 64) - 1]
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, counted=masks(counted), acc=acc, decay=0.5,
                               out=torch.full((2, kv_heads, width), math.nan, device="cuda"))
    mass_check(got, mass_want(s, lse, counted, acc, 0.5, width))


def test_attention_mass_in_place_empty_rows_and_nonfinite_queries(kvops):
    s = Setup(kvops, "f32", [100, 0, 33], [4, 2, 3], seed=21)
    s.mask[:] = 0
    _, lse = s.run(kvops)
    assert bool((lse[4:6] == -math.inf).all())
    acc = torch.rand(3, 2, s.cache.capacity, device="cuda")
    want = mass_want(s, lse, [0b1101, 3, 7], acc, 0.9, acc.shape[-1])
    s.q[1] = math.nan  # not counted
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, counted=masks([0b1101, 3, 7]), acc=acc, decay=0.9, out=acc)
    assert got is acc
    mass_check(acc, want)


def test_attention_mass_narrow_sums(kvops):
    """Sums narrower than the cache: positions past them are left out."""
    s = Setup(kvops, "bf16", [500], [3], seed=22)
    _, lse = s.run(kvops)
    out = torch.full((1, 2, 300), math.nan, device="cuda")
    mass_check(kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, out=out), mass_want(s, lse, width=300))


@pytest.mark.parametrize("dtype,dim,group", [("bf16", 128, 8), ("f16", 64, 16), ("f32", 128, 8), ("bf16", 128, 1)])
def test_attention_mass_many_tiles(kvops, dtype, dim, group):
    """Several tiles and segments a block, some without tokens, and more rows than a block
    holds at a time."""
    s = Setup(kvops, dtype, [90000, 33, 700, 12001], [3, 64, 0, 33], 2 * group, 2, dim, 32, seed=23)
    _, lse = s.run(kvops)
    width = s.cache.capacity
    acc = torch.rand(4, 2, width, device="cuda")
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, acc=acc, decay=0.75)
    mass_check(got, mass_want(s, lse, None, acc, 0.75, width))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_mass_one_token_many_tiles(kvops, dtype):
    s = Setup(kvops, dtype, [70000, 0, 31], [1, 1, 1], seed=25)
    _, lse = s.run(kvops, max_draft=1)
    width = s.cache.capacity
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, max_draft=1)
    mass_check(got, mass_want(s, lse, width=width))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_mass_many_rows_empty_nonfinite_and_unmapped(kvops, dtype):
    """As above for many rows: tokens that attended nothing or do not count add nothing whatever
    their queries hold, an unmapped page gets nothing, a key that is not finite reaches its own position alone."""
    s = Setup(kvops, dtype, [300, 0, 140], [40, 12, 17], seed=24)
    _, lse = s.run(kvops)
    lse[5] = -math.inf
    counted = [(1 << 40) - 1 - (1 << 7), (1 << 12) - 1, 0b1011]
    width = s.cache.capacity
    want = mass_want(s, lse, counted, width=width)
    s.q[7] = math.nan
    s.cache.table[0, 3] = -1
    want[0, :, 48:64] = 0
    s.cache.k[s.cache.table[2, 2], 0, 1, 5] = math.nan
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, counted=masks(counted))
    assert bool(got[2, 1, 37].isnan())
    got[2, 1, 37] = want[2, 1, 37]
    mass_check(got, want)


# -- select, compact, evict ------------------------------------------------------------

def select_want(row, n, keep, sinks, recent):
    if n <= keep:
        return list(range(n))
    lowest = [-math.inf if x != x else x for x in row]
    mid = sorted(range(sinks, n - recent), key=lambda t: (-lowest[t], t))[:keep - sinks - recent]
    return sorted(list(range(sinks)) + mid + list(range(n - recent, n)))


def select_check(kvops, acc, lens, keep, sinks, recent):
    L, B, KVH, W = acc.shape
    pool = torch.zeros(1, L, KVH, 2, 16, 64, device="cuda")
    cache = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], torch.zeros(B, -(-W // 16), dtype=torch.int32, device="cuda"))
    idx, sums, new = kvops.select(cache, acc, torch.tensor(lens, dtype=torch.int32, device="cuda"), keep=keep, sinks=sinks, recent=recent)
    host = acc.cpu()
    for l in range(L):
        for b in range(B):
            n = min(max(lens[b], 0), W)
            for h in range(KVH):
                want = select_want(host[l, b, h].tolist(), n, keep, sinks, recent)
                assert idx[l, b, h].tolist() == want + [-1] * (keep - len(want)), (l, b, h)
                w = torch.cat((host[l, b, h, want], torch.zeros(keep - len(want))))
                assert torch.equal(sums[l, b, h].cpu().view(torch.int32), w.view(torch.int32))
    assert new.tolist() == [min(max(n, 0), W, keep) if n > 0 else 0 for n in lens]


@pytest.mark.parametrize("width,lens,keep,sinks,recent", [
    (1, [1], 1, 0, 0), (40, [40, 0, 33, 7], 8, 2, 3), (40, [40, 39, 8, -3], 8, 4, 4), (5000, [5000, 4097, 64, 65], 64, 4, 32),
    (50000, [50000], 1000, 4, 32), (70000, [70000, 50], 3000, 0, 0), (131072, [131072], 4096, 4, 32), (300001, [300001], 17, 1, 1),
    (450000, [450000], 2000, 4, 100)])
def test_select(kvops, width, lens, keep, sinks, recent):
    g = torch.Generator(device="cuda").manual_seed(width)
    acc = torch.empty(2, len(lens), 2, width, device="cuda").normal_(0, 2, generator=g).exp_()
    acc[0] *= torch.rand(acc[0].shape, generator=g, device="cuda") > 0.3  # zeros tie
    select_check(kvops, acc, lens, keep, sinks, recent)


def test_select_ties_signs_and_nonfinite(kvops):
    g = torch.Generator(device="cuda").manual_seed(4)
    acc = torch.randint(-2, 3, (3, 2, 2, 9000), generator=g, device="cuda").float() / 2  # few values
    acc[0, 0, 0, ::3] = -0.0
    acc[1, 0] = 1.0  # all the same
    acc[2, 0, 0, 5::50], acc[2, 0, 1, 7::50], acc[2, 1, 0, 1::2], acc[2, 1, 1, 3::4] = math.nan, math.inf, -math.inf, 1e-42
    for keep, sinks, recent in ((1, 0, 0), (1000, 4, 32), (8000, 0, 7999), (4500, 10, 0)):
        select_check(kvops, acc, [9000, 8999], keep, sinks, recent)


@pytest.mark.parametrize("dtype,dim,page,in_place", [("f32", 128, 16, True), ("f32", 128, 16, False), ("bf16", 64, 32, True), ("f16", 128, 64, False)])
def test_evict_moves_keys_values_and_sums(kvops, dtype, dim, page, in_place):
    lens, keep = [200, 63, 0, 64, 777], 64
    s = Setup(kvops, dtype, lens, [0] * 5, kv_heads=3, heads=3, dim=dim, page=page, layers=2, seed=31)
    g = torch.Generator(device="cuda").manual_seed(1)
    acc = torch.rand(2, 5, 3, s.cache.capacity, generator=g, device="cuda")
    before = s.pool.clone()
    into = None
    if not in_place:
        pool = torch.full((-(-keep // page) * 5, 2, 3, 2, page, dim), 9.0, dtype=s.dtype, device="cuda")
        table = torch.randperm(pool.shape[0], generator=torch.Generator().manual_seed(2)).int().view(5, -1)
        into = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], table.cuda())
    idx, sums, new = kvops.evict(s.cache, acc, s.lens, keep=keep, sinks=4, recent=8, into=into)
    assert new.tolist() == [min(n, keep) for n in lens]
    for b, n in enumerate(lens):
        for layer in range(2):
            k0, v0 = s.rows(b, layer, pool=before)
            if in_place:
                k1, v1 = s.rows(b, layer, n=min(n, keep))
            else:
                t = torch.arange(min(n, keep))
                x = pool.cpu()[table[b, t // page].long(), layer, :, :, t % page].double()
                k1, v1 = x[:, :, 0], x[:, :, 1]
            for h in range(3):
                want = select_want(acc[layer, b, h].tolist(), n, keep, 4, 8)
                assert idx[layer, b, h, :len(want)].tolist() == want
                assert torch.equal(k1[:, h], k0[want, h]) and torch.equal(v1[:, h], v0[want, h])
                assert torch.equal(sums[layer, b, h, :len(want)], acc[layer, b, h, want])


def test_evict_to_more_than_the_cache_moves_nothing(kvops):
    s = Setup(kvops, "bf16", [40, 17], [0, 0], seed=33, junk=3.0)
    before = s.pool.clone()
    idx, sums, new = kvops.evict(s.cache, torch.rand(1, 2, 2, 48, device="cuda"), s.lens, keep=300, sinks=4, recent=8)
    assert torch.equal(before, s.pool) and new.tolist() == [40, 17]
    assert bool((idx[..., 48:] == -1).all())


# -- append ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim,page", [("f32", 128, 16), ("bf16", 64, 32), ("f16", 128, 16)])
def test_append_paths(kvops, dtype, dim, page):
    lens, counts, n_path = [0, 15, 16, 100, 31], [4, 9, 1, 64, 5], [4, 3, 0, 5, 5]
    s = Setup(kvops, dtype, lens, counts, dim=dim, page=page, layers=3, seed=41, room=6, junk=2.0)
    g = torch.Generator().manual_seed(42)
    k = torch.randn(3, sum(counts), 2, dim, generator=g).to(s.dtype).cuda()
    v = torch.randn(3, sum(counts), 2, dim, generator=g).to(s.dtype).cuda()
    path = torch.full((5, 6), 99, dtype=torch.int32)
    for b in range(5):
        path[b, :n_path[b]] = torch.randperm(counts[b], generator=g)[:n_path[b]].sort().values.int()
    before = s.pool.clone()
    new = kvops.append(s.cache, k, v, s.lens, s.indptr, path=path.cuda(), n_path=torch.tensor(n_path, dtype=torch.int32, device="cuda"))
    assert new.tolist() == [a + n for a, n in zip(lens, n_path)]
    want = before.cpu()
    for b in range(5):
        for i in range(n_path[b]):
            t, tok = lens[b] + i, int(s.indptr[b]) + int(path[b, i])
            want[s.table_h[b, t // page].long(), :, :, 0, t % page] = k[:, tok].cpu()
            want[s.table_h[b, t // page].long(), :, :, 1, t % page] = v[:, tok].cpu()
    assert torch.equal(s.pool.cpu(), want)


def test_append_prompt_bad_nodes_and_full_tables(kvops):
    s = Setup(kvops, "f32", [0, 5], [300, 7], layers=2, seed=43, room=0, junk=2.0)
    k, v = torch.randn(2, 307, 2, 128, device="cuda"), torch.randn(2, 307, 2, 128, device="cuda")
    pool = torch.full((40, 2, 2, 2, 16, 128), 2.0, device="cuda")
    table = torch.full((2, 20), -1, dtype=torch.int32)
    table[0, :19] = torch.arange(19).int()
    table[1, :1] = 30
    cache = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], table.cuda())
    assert kvops.append(cache, k, v, s.lens, s.indptr).tolist() == [300, 12]
    t = torch.arange(300)
    assert torch.equal(pool[t // 16, :, :, 0, t % 16].cpu(), k[:, :300].transpose(0, 1).cpu())
    assert torch.equal(pool[t // 16, :, :, 1, t % 16].cpu(), v[:, :300].transpose(0, 1).cpu())
    assert torch.equal(pool[30, :, :, 0, 5:12].cpu(), k[:, 300:].permute(0, 2, 1, 3).cpu())
    assert bool((pool[30, :, :, :, 12:] == 2).all()) and bool((pool[19:30] == 2).all()) and bool((pool[31:] == 2).all())
    # nodes outside the sequence and positions without a page are skipped
    before = pool.clone()
    lens = torch.tensor([318, 14], dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 1, 2, 3], [-1, 7, 2, 6]], dtype=torch.int32, device="cuda")
    new = kvops.append(cache, k, v, lens, s.indptr, path=path, n_path=torch.tensor([4, 9], dtype=torch.int32, device="cuda"))
    assert new.tolist() == [320, 18]
    assert torch.equal(before, pool)


# -- refusals ------------------------------------------------------------------------------

def test_refusals(kvops):
    from rapidocrvl_b200._lib import OcrvlError

    s = Setup(kvops, "f32", [20], [3], seed=51)
    k, v = s.pool[:, :, :, 0], s.pool[:, :, :, 1]
    t = s.cache.table
    with pytest.raises(ValueError):
        kvops.PagedCache(k, v[:1], t)
    with pytest.raises(ValueError):
        kvops.PagedCache(k.cpu(), v.cpu(), t)
    with pytest.raises(ValueError):
        kvops.PagedCache(k, v, t.long())
    for shape in ((2, 1, 2, 2, 8, 128), (2, 1, 2, 2, 24, 128), (2, 1, 2, 2, 16, 96)):
        p = torch.zeros(shape, device="cuda")
        bad = kvops.PagedCache(p[:, :, :, 0], p[:, :, :, 1], t)
        with pytest.raises(OcrvlError):
            kvops.compact(bad, torch.zeros(1, 1, 2, 4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        kvops.tree_attention(s.q.half(), s.k, s.v, s.cache, s.lens, s.indptr, s.mask)
    with pytest.raises(ValueError):
        kvops.tree_attention(s.q, s.k[:2], s.v, s.cache, s.lens, s.indptr, s.mask)
    with pytest.raises(ValueError):
        kvops.tree_attention(s.q, s.k, s.v, s.cache, s.lens.long(), s.indptr, s.mask)
    with pytest.raises(ValueError):
        kvops.tree_attention(s.q, s.k, s.v, s.cache, s.lens, s.indptr[:1], s.mask)
    with pytest.raises(ValueError):
        kvops.tree_attention(s.q.transpose(1, 2).contiguous().transpose(1, 2), s.k, s.v, s.cache, s.lens, s.indptr, s.mask)
    for kw in (dict(layer=1), dict(layer=-1), dict(max_draft=0), dict(max_draft=65), dict(scale=math.nan),
               dict(work=torch.empty(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(OcrvlError):
            s.run(kvops, **kw) if "scale" not in kw else kvops.tree_attention(s.q, s.k, s.v, s.cache, s.lens, s.indptr, s.mask, **kw)
    q = torch.zeros(3, 5, 128, device="cuda")
    with pytest.raises(OcrvlError):  # 5 heads over 2
        kvops.tree_attention(q, s.k, s.v, s.cache, s.lens, s.indptr, s.mask)
    odd = torch.zeros(3 * 16 * 128 + 1, device="cuda")[1:].view(3, 16, 128)
    with pytest.raises(OcrvlError):  # 4-byte aligned
        kvops.tree_attention(odd, s.k, s.v, s.cache, s.lens, s.indptr, s.mask)
    acc = torch.zeros(1, 1, 2, 32, device="cuda")
    for kw in (dict(keep=0), dict(keep=4, sinks=3, recent=2), dict(keep=4, sinks=-1)):
        with pytest.raises(OcrvlError):
            kvops.select(s.cache, acc, s.lens, **kw)
    with pytest.raises(ValueError):
        kvops.select(s.cache, acc[0], s.lens, keep=4)
    with pytest.raises(ValueError):
        kvops.append(s.cache, s.k[None], s.v[None], s.lens, s.indptr, path=torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    out, lse = s.run(kvops)
    with pytest.raises(OcrvlError):
        kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, decay=math.inf)
    with pytest.raises(ValueError):
        kvops.attention_mass(s.q, lse[:2], s.cache, s.lens, s.indptr)
    none = kvops.tree_attention(s.q[:0], s.k[:0], s.v[:0], s.cache, s.lens, torch.zeros(2, dtype=torch.int32, device="cuda"), s.mask[:0])
    assert none[0].shape == (0, 16, 128)
