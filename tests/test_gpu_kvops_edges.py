"""The paged-cache operators (rapidocrvl_b200.kvops) where they can go wrong:
values that are not finite or as large as the type goes, scores that rise
along the context, rows and pages with nothing in them, on every shape of
kernel.  Setup, types and the tolerances' derivation are test_gpu_kvops.py's;
what a test adds to them is said there."""
import math
import threading

import pytest
import torch

from test_gpu_kvops import REL, Setup, kvops, mass_check, mass_want, masks, select_check  # noqa: F401 (kvops: the fixture)

pytestmark = pytest.mark.gpu

# Calls of 16-bit types that take each shape of the tensor-memory kernel (heads 16 / 2): (lens, counts, max_draft).
# Lengths differ by 128 so that the drafts lie in tiles of both streams.
MANY_ROWS = {
    "narrow, runs": ([4000, 4130, 3900], [16, 9, 13], 16),
    "narrow, whole": ([(37 * b) % 300 for b in range(40)], [16, 11] + [1 + b % 5 for b in range(38)], 16),
    "wide, runs": ([4000, 4130], [64, 33], 64),
    "wide, whole": ([(37 * b) % 300 for b in range(37)], [64, 40] + [b % 4 for b in range(35)], 64),
}


def want(s, see_cached=None):
    """(out, lse, largest |v| seen) in 64 bits: of every token over the cached positions (those of see_cached[b], if
    given) and over the drafts that its mask names, nothing else touched."""
    N, H, D = s.q.shape
    out, lse = torch.zeros(N, H, D, dtype=torch.float64), torch.full((N, H), -math.inf, dtype=torch.float64)
    top = torch.zeros(N, H, 1, dtype=torch.float64)
    q, k, v = (x.cpu().double() for x in (s.q, s.k, s.v))
    mask, group = s.mask.tolist(), H // s.kv_heads
    for b, t in enumerate(s.counts):
        if not t:
            continue
        at = slice(int(s.indptr[b]), int(s.indptr[b]) + t)
        ck, cv = s.rows(b)
        if see_cached is not None:
            ck, cv = ck[see_cached[b]], cv[see_cached[b]]
        n = len(ck)
        keys, values = torch.cat((ck, k[at])), torch.cat((cv, v[at]))
        see = torch.ones(t, n + t, dtype=torch.bool)
        see[:, n:] = torch.tensor([[bool(m >> j & 1) for j in range(t)] for m in mask[at]])
        for h in range(H):
            g = h // group
            x = (q[at, h] @ keys[:, g].T * s.scale).masked_fill(~see, -math.inf)
            lse[at, h] = torch.logsumexp(x, 1)
            w = torch.where(see.any(1)[:, None], torch.softmax(x, 1), torch.zeros_like(x))
            out[at, h] = w @ values[:, g]
            top[at, h, 0] = torch.where(see, values[:, g].abs().amax(1)[None], torch.zeros(())).amax(1)
    return out, lse, top


def check(s, got, wanted, extra=0.0):
    """extra: a weight's further relative error, and the lse's."""
    (out, lse), (w_out, w_lse, top) = got, wanted
    out, lse = out.cpu().double(), lse.cpu().double()
    a, r = REL[s.name]
    for same in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(same(out), same(w_out)), same
    fine = torch.isfinite(w_out)
    off = (out - w_out).abs() <= (a + extra) * top + r * w_out.abs()
    assert bool(off[fine].all()), float(((out - w_out).abs() / top.clamp(min=1e-30))[fine].max())
    empty = w_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool(((lse - w_lse).abs() <= 1e-5 + extra)[~empty].all())


# -- values that are not finite -------------------------------------------------------

@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("shape", MANY_ROWS)
def test_many_rows_get_the_values_they_see(kvops, shape, dtype, dim, bad):
    """A draft's value that is not finite, in dims of both halves and of tiles of both streams, reaches every row that
    sees the draft, in those dims alone, and no other row."""
    lens, counts, most = MANY_ROWS[shape]
    s = Setup(kvops, dtype, lens, counts, dim=dim, seed=61)
    starts = s.indptr.tolist()
    for b, t in enumerate(counts):
        if t:
            s.v[starts[b] + t // 2, b % 2, [1, dim // 2 - 1, dim // 2, dim - 2][b % 4]] = bad
    for d in (0, dim // 2 + 1):  # the first sequence's first draft, in both halves
        s.v[starts[0], 1, d] = bad
    check(s, s.run(kvops, max_draft=most), want_nonfinite(s))


def want_nonfinite(s):
    """want() of finite values, then what is not finite added where it is seen: its weight is positive."""
    v = s.v
    s.v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    out, lse, top = want(s)
    s.v = v
    group = s.heads // s.kv_heads
    for i, g, d in torch.nonzero(~torch.isfinite(v)).tolist():
        b = int(torch.searchsorted(s.indptr.cpu(), torch.tensor(i), right=True)) - 1
        i0 = int(s.indptr[b])
        for j in range(i0, i0 + s.counts[b]):
            if int(s.mask[j]) >> (i - i0) & 1:
                out[j, g * group:(g + 1) * group, d] += float(v[i, g, d])
    return out, lse, top


@pytest.mark.parametrize("big", [torch.finfo(torch.float32).min, torch.finfo(torch.float32).max, 3.402e38])
@pytest.mark.parametrize("counts,heads", [([6, 1], 4), ([20, 3], 16), ([64, 3], 16)])  # 8, 16 and 32 rows a block
def test_f32_drafts_as_large_as_the_type_goes(kvops, counts, heads, big):
    """Keys and values filled with the type's lowest or largest value, masked."""
    s = Setup(kvops, "f32", [40, 300], counts, heads=heads, seed=62)
    s.mask = masks([1 << i | (i > 0) for t in counts for i in range(t)])
    s.k[3], s.v[3] = big, big  # only token 3 sees it
    got = s.run(kvops)
    s.k[3], s.v[3] = 0.5, 0.5
    rest = [i for i in range(sum(counts)) if i != 3]
    check(s, [x[rest] for x in got], [x[rest] for x in want(s)])


@pytest.mark.parametrize("big", [torch.finfo(torch.float32).min, torch.finfo(torch.float32).max])
def test_f32_largest_values_seen(kvops, big):
    s = Setup(kvops, "f32", [0, 20], [2, 1], seed=63)
    s.mask = masks([1, 3, 1])
    s.v[0] = big
    s.k[1] = s.k[0]  # token 1 sees both alike
    s.v[1, :, 1:] = 0
    s.pool[s.table_h[1, 0].long(), 0, :, 1, 4] = big / 4
    check(s, s.run(kvops), want(s))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,counts,heads", [
    ([300, 20, 90], [2, 1, 2], 4), ([300, 20, 140], [40, 1, 17], 16), ([9000], [64], 32), ([90000], [1], 16)])
def test_attention_mass_of_tokens_that_attended_nothing(kvops, dtype, lens, counts, heads, bad):
    """A token, or some of its heads, whose lse is -inf adds nothing whatever its query holds."""
    s = Setup(kvops, dtype, lens, counts, heads=heads, seed=64)
    _, lse = s.run(kvops, max_draft=max(counts))
    none = [0, sum(counts) - 1] if sum(counts) > 1 else []
    half = heads // 2 + 1
    lse[none] = -math.inf
    lse[0, half:] = -math.inf
    w = mass_want(s, lse, width=s.cache.capacity)
    s.q[none] = bad
    s.q[0, half:, 7] = bad
    mass_check(kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, max_draft=max(counts)), w)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,counts,heads", [([300, 20], [1, 1], 4), ([300, 140], [40, 3], 16)])
def test_attention_mass_of_infinite_keys(kvops, dtype, lens, counts, heads):
    """A key with an infinity counts with the rows that count: one whose score is -inf weighs nothing."""
    s = Setup(kvops, dtype, lens, counts, heads=heads, seed=68)
    _, lse = s.run(kvops)
    s.q[..., 3] = s.q[..., 3].abs() + 0.5
    s.cache.k[s.cache.table[0, 2], 0, 1, 5, 3] = -math.inf  # position 37: every score is -inf
    s.cache.k[s.cache.table[1, 0], 0, 0, 2, 3] = math.inf   # every score is inf
    got = kvops.attention_mass(s.q, lse, s.cache, s.lens, s.indptr, scale=s.scale, counted=masks([1, 1]))
    w = mass_want(s, lse, [1, 1], width=s.cache.capacity)
    assert float(got[0, 1, 37]) == 0 and float(w[0, 1, 37]) == 0
    assert float(got[1, 0, 2]) == math.inf
    got[1, 0, 2] = w[1, 0, 2] = 0
    mass_check(got, w)


# -- the reference's rise, rows and pages with nothing in them --------------------------

# As MANY_ROWS, with several tiles a group of warps.
MANY_TILES = {
    "narrow, runs": ([40000, 300], [16, 5], 16),
    "narrow, whole": ([(137 * b) % 1000 for b in range(40)], [16, 11] + [1 + b % 3 for b in range(38)], 16),
    "wide, runs": ([20000, 4130], [64, 3], 64),
    "wide, whole": ([(137 * b) % 1000 for b in range(37)], [64, 40] + [b % 3 for b in range(35)], 64),
    "few rows": ([2000, 40], [2, 1], 2),
}


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 128)])
@pytest.mark.parametrize("shape", MANY_TILES)
def test_scores_that_rise_along_the_context(kvops, shape, dtype, dim):
    """Some rows' scores rise by 16 powers of two every 32 positions of some tiles and by 100 at once
    further on, others fall alike.  A score of size x is off by its sum's roundings, at most one of 2^-23 for each
    of eight products of 16 dims: x 2^-20 of a weight."""
    lens, counts, most = MANY_TILES[shape]
    s = Setup(kvops, dtype, lens, counts, dim=dim, seed=71)
    per = 4 * s.scale / math.log(2)  # powers of two a unit of dim 0, whose queries are 4 and -4
    s.q[:, ::2, 0], s.q[:, 1::2, 0] = 4, -4
    for b, n in enumerate(lens):
        t = torch.arange(n)
        steps = torch.cumsum((t % 32 == 0) & (t // 128 % 7 % 3 == 1) & (t < 2300), 0).clamp(max=12) * 16 + (t >= 700) * 100
        pages = s.table_h[b, t // s.page].long().cuda()
        for g in range(2):
            s.pool[pages, 0, g, 0, (t % s.page).cuda(), 0] = (steps / per).to(s.dtype).cuda()
    w = want(s)
    check(s, s.run(kvops, max_draft=most), w, extra=2.0 ** -20 * float(w[1][torch.isfinite(w[1])].abs().max()))


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("shape", MANY_TILES)
def test_many_rows_with_unmapped_pages_and_nothing_to_see(kvops, shape, dtype, dim):
    lens, counts, most = MANY_TILES[shape]
    s = Setup(kvops, dtype, lens, counts, dim=dim, seed=72)
    table, starts = s.table_h.clone(), s.indptr.tolist()
    mapped = [torch.ones(n, dtype=torch.bool) for n in lens]

    def unmap(b, page, entry):
        table[b, page] = entry
        mapped[b][page * 16:(page + 1) * 16] = False

    for page in list(range(17)) + [20, 23, 40, 55]:  # whole tiles at the start, then single pages
        if page * 16 < lens[0]:
            unmap(0, page, -1 if page % 2 else 1 << 30)
    for page in range(-(-lens[1] // 16)):  # the second sequence has nothing cached
        unmap(1, page, table.shape[0] * 10000 if page % 3 else -5)
    bits = s.mask.tolist()
    for i in range(starts[1], starts[2], 2):  # and half of its tokens do not see themselves either
        bits[i] = 0
    for i in range(starts[0], starts[1], 3):
        bits[i] = 0
    s.mask = masks(bits)
    s.cache = kvops.PagedCache(s.pool[:, :, :, 0], s.pool[:, :, :, 1], table.cuda())
    check(s, s.run(kvops, max_draft=most), want(s, see_cached=mapped))


def long_tail(kvops, dtype, n, most):
    """One position far above all others, each of which has 2^-24 to 2^-27 of its weight: together a 400th or a 50th of
    the sum.  Returns (out, lse) and what they should be."""
    B, heads, dim, page = 74, 16, 64, 1024
    pages = n // page
    g = torch.Generator(device="cuda").manual_seed(65)
    pool = torch.zeros(128, 1, 2, 2, page, dim, dtype=dtype, device="cuda")
    pool[:, :, :, 1] = torch.empty(pool[:, :, :, 1].shape, dtype=dtype, device="cuda").uniform_(0.5, 1.0, generator=g)
    pool[0, 0, :, 0, 0, 0], pool[0, 0, :, 1, 0] = 1.0, 0.0  # the strong position
    row = torch.arange(pages, dtype=torch.int32)
    row[128:] = row[128:] % 127 + 1  # long contexts: the pages without it over and over
    cache = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], row.cuda().repeat(B, 1))
    counts = [most] + [1] * (B - 1)
    N = sum(counts)
    q = torch.zeros(N, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = torch.linspace(16.0, 18.0, heads, device="cuda").to(dtype)
    kv = torch.zeros(N, 2, dim, dtype=dtype, device="cuda")
    scale = 25.6 * math.log(2) / 17.0
    out, lse = kvops.tree_attention(q, kv, kv, cache, torch.full((B,), n, dtype=torch.int32, device="cuda"),
                                    torch.tensor([0] + [sum(counts[:b + 1]) for b in range(B)], dtype=torch.int32, device="cuda"),
                                    torch.zeros(N, dtype=torch.int64, device="cuda"), max_draft=most, scale=scale)
    v = pool[row.cuda().long(), 0, :, 1].double().sum((0, 2)).repeat_interleave(heads // 2, 0)  # [heads, dim]
    x = q[0, :, 0].double() * scale
    w = torch.exp(-x)[:, None]
    return out.double(), lse.double(), v * w / (1 + (n - 1) * w), x + torch.log1p((n - 1) * w[:, 0])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,most", [(1 << 17, 8), (1 << 20, 1)])  # many rows, eight rows
def test_long_tails_are_in_the_sum(kvops, n, most, dtype):
    _, lse, _, want = long_tail(kvops, {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype], n, most)
    assert bool(((lse - want).abs() <= 1e-5).all()), float((lse - want).abs().max())


@pytest.mark.parametrize("n,most", [(1 << 17, 8), (1 << 20, 1)])
def test_f16_long_tails_keep_their_weight(kvops, n, most):
    """Weights below f16's smallest numbers reach the values too."""
    out, _, want, _ = long_tail(kvops, torch.float16, n, most)
    a, r = REL["f16"]
    assert bool(((out - want).abs() <= a + r * want).all()), float((out - want).abs().max())


# -- calls with fewer drafts than max_draft ------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("lens,counts,heads,kv_heads,most", [
    ([16779, 9000, 16779, 300, 12000], [17, 9, 17, 1, 3], 32, 8, 64),  # up to 68 rows where 256 may come
    ([32344, 0, 20000, 5], [1, 1, 1, 1], 32, 8, 64),
    ([3000 + 77 * b for b in range(16)], [1 + b % 2 for b in range(16)], 16, 2, 64),
    ([8000, 8000, 8000], [64, 1, 40], 16, 2, 64),  # blocks of 256 rows, of few, of 256 and 64
    ([(613 * b) % 2500 for b in range(50)], [b % 3 for b in range(50)], 16, 2, None)])  # the default: the call's tokens
def test_fewer_drafts_than_the_call_may_have(kvops, lens, counts, heads, kv_heads, most, dtype, dim):
    s = Setup(kvops, dtype, lens, counts, heads, kv_heads, dim, seed=91)
    wanted = want(s)
    for _ in range(3):
        check(s, s.run(kvops, max_draft=most), wanted)


# -- tables -----------------------------------------------------------------------------

def test_tables_whose_rows_overlap_are_refused(kvops):
    s = Setup(kvops, "f32", [100, 100], [1, 2], seed=73)
    k, v, row = s.cache.k, s.cache.v, s.cache.table[:1]
    for bad in (row.expand(2, -1), torch.as_strided(s.cache.table, (2, 6), (1, 1))):
        with pytest.raises(ValueError, match="overlap"):
            kvops.PagedCache(k, v, bad)
    # one row, a copy of it, and rows that lie apart are fine
    kvops.PagedCache(k, v, row.expand(1, -1))
    apart = torch.full((2, 2 * row.shape[1]), 1 << 30, dtype=torch.int32, device="cuda")[:, :row.shape[1]]
    apart.copy_(row.expand(2, -1))
    same = []
    for table in (row.expand(2, -1).contiguous(), apart):
        s.cache = kvops.PagedCache(k, v, table)
        same.append(s.run(kvops))
    assert torch.equal(same[0][0], same[1][0]) and torch.equal(same[0][1], same[1][1])
    s.table_h[1] = s.table_h[0]
    s.check(*same[0])


# -- select -----------------------------------------------------------------------------

def test_select_of_several_widths_from_several_threads(kvops):
    """Calls of the C entry (which takes no lock) on streams of their own, each of another width."""
    from rapidocrvl_b200 import _lib

    L, said = _lib.load(), []

    def calls(acc, lens, idx, stream):
        for _ in range(400):
            if L.ocrvl_op_kv_select(1, 1, 2, acc.data_ptr(), acc.shape[1], acc.shape[1], lens.data_ptr(), 64, 0, 0, idx.data_ptr(), None, None,
                                    stream.cuda_stream):
                return said.append((acc.shape[1], _lib.last_error()))

    work = [(torch.stack([torch.randperm(w, device="cuda").float() for _ in range(2)]), torch.tensor([w], dtype=torch.int32, device="cuda"),
             torch.empty(2, 64, dtype=torch.int32, device="cuda"), torch.cuda.Stream()) for w in (390000, 300000, 200000, 100000)]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=calls, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not said
    for acc, _, idx, _ in work:
        assert torch.equal(idx.long(), acc.topk(64).indices.sort().values)


@pytest.mark.parametrize("width", [9001, 30003, 300001])  # clusters of several sizes
def test_select_of_few_positions_in_wide_unaligned_rows(kvops, width):
    """Most blocks of a row's cluster have nothing to hold, and rows start at each alignment."""
    acc = torch.rand(2, 8, 1, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(width))
    select_check(kvops, acc, [5, 6, 7, 9, 13, 33, 61, 130], 4, 1, 1)
    select_check(kvops, acc[..., :width - 2], [17, 18, 19, 23, 5, 64, 1, 0], 4, 0, 2)


# -- compact and evict ------------------------------------------------------------------

@pytest.mark.parametrize("keep", [65, 200])
def test_evict_into_too_little_room_is_refused(kvops, keep):
    from rapidocrvl_b200._lib import OcrvlError

    s = Setup(kvops, "f32", [200], [0], seed=66)
    pool = torch.full((4, 1, 2, 2, 16, 128), 9.0, device="cuda")
    into = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], torch.arange(4, dtype=torch.int32, device="cuda")[None])
    acc = torch.rand(1, 1, 2, 208, device="cuda")
    with pytest.raises(OcrvlError, match="room"):
        kvops.evict(s.cache, acc, s.lens, keep=keep, into=into)
    idx, _, _ = kvops.select(s.cache, acc, s.lens, keep=keep)
    with pytest.raises(OcrvlError, match="room"):
        kvops.compact(s.cache, idx, into=into)
    assert bool((pool == 9).all())
    _, _, new = kvops.evict(s.cache, acc, s.lens, keep=64, into=into)
    assert new.tolist() == [64] and not bool((pool == 9).any())
    # a cache that holds no more than there is room for may be asked to keep any number
    small = Setup(kvops, "f32", [40], [0], seed=67)
    _, _, new = kvops.evict(small.cache, acc[..., :48].contiguous(), small.lens, keep=keep, into=into)
    assert new.tolist() == [40]


# -- large pools --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_past_32_bits(kvops, dtype):
    """Pages that lie 5 GB behind the start of the pool."""
    s = Setup(kvops, dtype, [700, 3000, 33], [16, 1, 40], heads=8, kv_heads=2, seed=95, room=64, junk=2.0)
    pages, far = s.pool.shape[0], -(-(5 << 30) // s.pool[0].nbytes)
    big = torch.empty((far + pages,) + s.pool.shape[1:], dtype=s.dtype, device="cuda")
    big[far:] = s.pool
    moved = torch.where(s.table_h >= 0, s.table_h + far, s.table_h)
    cache = kvops.PagedCache(big[:, :, :, 0], big[:, :, :, 1], moved.cuda())
    near = s.cache, s.pool
    results = []
    for c, pool in (near, (cache, big[far:])):
        s.cache = c
        out, lse = s.run(kvops)
        mass = kvops.attention_mass(s.q, lse, c, s.lens, s.indptr, scale=s.scale)
        new = kvops.append(c, s.k[None], s.v[None], s.lens, s.indptr)
        kept = kvops.evict(c, mass[None], s.lens, keep=100, sinks=2, recent=5)
        results.append((out, lse, mass, new, *kept, pool))
    for a, b in zip(*results):
        assert torch.equal(a, b)


# -- autograd ---------------------------------------------------------------------------

def _calls(kvops, s, into):
    """Every operator on tensors by name."""
    layers = torch.randn(1, s.q.shape[0], 2, 128, device="cuda")
    _, lse = s.run(kvops)
    x = dict(q=s.q, k=s.k, v=s.v, lse=lse, acc=torch.rand(1, 2, s.cache.capacity, device="cuda"), out=torch.empty_like(s.q),
             new_k=layers, new_v=layers.clone(), idx=torch.arange(8, dtype=torch.int32, device="cuda").expand(1, 1, 2, 8).contiguous())
    seqs = (s.lens, s.indptr)
    return x, {
        "tree_attention": (lambda: kvops.tree_attention(x["q"], x["k"], x["v"], s.cache, *seqs, s.mask, out=x["out"], lse=x["lse"]),
                           ("q", "k", "v"), ("out", "lse")),
        "attention_mass": (lambda: kvops.attention_mass(x["q"], x["lse"], s.cache, *seqs, acc=x["acc"], out=x["acc"]), ("q", "lse", "acc"), ("acc",)),
        "append": (lambda: kvops.append(s.cache, x["new_k"], x["new_v"], *seqs), ("new_k", "new_v"), "cache"),
        "evict": (lambda: kvops.evict(s.cache, x["acc"][None], s.lens, keep=8, into=into), ("acc",), "into"),
        "evict in place": (lambda: kvops.evict(s.cache, x["acc"][None], s.lens, keep=8), ("acc",), "cache"),
        "select": (lambda: kvops.select(s.cache, x["acc"][None], s.lens, keep=8), ("acc",), ()),
        "compact": (lambda: kvops.compact(s.cache, x["idx"], into=into), (), "into"),
    }


def test_tensors_that_require_a_gradient_are_refused_and_writes_are_counted(kvops):
    s = Setup(kvops, "f32", [40], [3], seed=81, room=4)
    pool = torch.zeros(1, 1, 2, 2, 16, 128, device="cuda")
    into = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    x, calls = _calls(kvops, s, into)
    for name, (call, reads, writes) in calls.items():
        for key in reads:
            x[key].requires_grad_()
            with pytest.raises(ValueError, match="gradient"):
                call()
            x[key].requires_grad_(False)
        counted = {"cache": (s.cache.k, s.cache.v), "into": (into.k, into.v)}[writes] if isinstance(writes, str) else [x[w] for w in writes]
        before = [t._version for t in counted]
        call()
        assert all(t._version > b for t, b in zip(counted, before)), name
        with torch.inference_mode():
            call()
    grown = s.pool.clone().requires_grad_()  # a cache that requires one
    s.cache = kvops.PagedCache(grown[:, :, :, 0], grown[:, :, :, 1], s.cache.table)
    for call, _, _ in calls.values():
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        s.run(kvops)
        x["q"].requires_grad_()
        s.run(kvops)


# -- refusals ---------------------------------------------------------------------------

def test_too_many_kv_heads_are_refused_before_anything_runs(kvops):
    from rapidocrvl_b200._lib import OcrvlError

    heads = 70000
    pool = torch.zeros(1, 1, heads, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, 320, dtype=torch.int32, device="cuda")  # long enough to be split and joined
    cache = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], table)
    q = torch.zeros(1, heads, 64, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full((1, heads), 7.0, device="cuda")
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([5000], [0, 1])]
    with pytest.raises(OcrvlError, match="heads"):
        kvops.tree_attention(q, q, q, cache, *ints, torch.ones(1, dtype=torch.int64, device="cuda"), out=out, lse=lse)
    torch.cuda.synchronize()
    assert bool((out == 7).all()) and bool((lse == 7).all())
