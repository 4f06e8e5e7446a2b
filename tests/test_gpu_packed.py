"""The packed cache (rapidocrvl_b200.kvops.PackedCache): tokens quantised as they are
written, and read back, against the format's definition in 64 bits.  Codes, scales
and the numbers they stand for are equal bit by bit: the format leaves no room."""
import math

import numpy as np
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


def quantised(x):
    """Rows [..., dim] as bytes, bf16 scales and the numbers (64 bits) they stand for."""
    x = np.asarray(x, np.float64)
    rows = x.reshape(-1, x.shape[-1])
    n, D = rows.shape
    G = D // 32
    codes, scales, numbers = np.zeros((n, D // 2), np.uint8), np.zeros((n, G)), np.zeros((n, D))
    for j in range(G):
        v = rows[:, 32 * j:32 * j + 32]
        fine = np.isfinite(v).all(1)
        m, e = np.frexp(np.where(fine, np.abs(np.where(fine[:, None], v, 0)).max(1), 0) / 7)
        s = np.ldexp(np.rint(m * 32) / 32, e)
        s[s < 2.0 ** -126] = 0
        c = np.zeros((n, 32))
        np.divide(v, s[:, None], out=c, where=(s > 0)[:, None])
        c = np.rint(c)
        assert np.abs(c).max(initial=0) <= 7
        scales[:, j] = np.where(fine, s, np.nan)
        numbers[:, 32 * j:32 * j + 32] = c * scales[:, j:j + 1]
        for d in range(32):
            nibble = 4 * (d // 4 * G + j) + d % 4
            codes[:, nibble // 2] |= ((c[:, d] + 8).astype(np.uint8) << 4 * (nibble % 2)).astype(np.uint8)
    lead = x.shape[:-1]
    return (torch.from_numpy(codes.reshape(*lead, D // 2)), torch.from_numpy(scales.reshape(*lead, G)).to(torch.bfloat16),
            torch.from_numpy(numbers.reshape(x.shape)))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Store:
    """A cache of shuffled pages whose bytes are known, and tokens to write."""

    def __init__(self, kvops, dtype, lens, counts, kv_heads=2, dim=128, page=16, layers=2, seed=0, most=None):
        g = torch.Generator().manual_seed(seed)
        self.lens_h, self.counts, self.page, self.layers, self.kv_heads, self.dim = lens, counts, page, layers, kv_heads, dim
        B, N = len(lens), sum(counts)
        need = [-(-(n + t) // page) for n, t in zip(lens, counts)]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g).tolist()
        self.table_h = torch.full((B, most or max(1, max(need))), -1, dtype=torch.int32)
        for b in range(B):
            for i in range(min(need[b], self.table_h.shape[1])):
                self.table_h[b, i] = order.pop()
        self.codes = torch.randint(0, 256, (2, pages, layers, kv_heads, page, dim // 2), generator=g, dtype=torch.uint8)
        self.scales = torch.rand(2, pages, layers, kv_heads, page, dim // 32, generator=g).to(torch.bfloat16)
        self.dev, self.dev_s = self.codes.cuda(), self.scales.cuda()
        self.cache = kvops.PackedCache(self.dev[0], self.dev[1], self.dev_s[0], self.dev_s[1], self.table_h.cuda())
        self.lens, self.indptr = ints(lens), ints([0] + [sum(counts[:b + 1]) for b in range(B)])
        self.x = (2 * torch.randn(2, layers, N, kv_heads, dim, generator=g)).to(TYPES[dtype])

    def put(self, b, pos, token):
        """What the cache holds once the token is at the position."""
        codes, scales, _ = quantised(self.x[:, :, token].double())
        p = int(self.table_h[b, pos // self.page])
        if p >= 0:
            self.codes[:, p, :, :, pos % self.page], self.scales[:, p, :, :, pos % self.page] = codes, scales

    def check(self):
        assert torch.equal(self.dev.cpu(), self.codes)
        assert torch.equal(self.dev_s.cpu().view(torch.int16), self.scales.view(torch.int16))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,counts,kv_heads,dim,page,layers", [
    ([0], [1], 2, 128, 16, 1), ([15, 0, 31], [3, 0, 40], 2, 128, 16, 5), ([7], [17], 1, 64, 16, 3), ([100, 3], [1, 64], 8, 64, 32, 4), ([5], [129], 3, 128, 64, 18)])
def test_append_and_read(kvops, dtype, lens, counts, kv_heads, dim, page, layers):
    s = Store(kvops, dtype, lens, counts, kv_heads, dim, page, layers)
    x = s.x.cuda()
    new = kvops.append(s.cache, x[0], x[1], s.lens, s.indptr)
    assert new.tolist() == [n + t for n, t in zip(lens, counts)]
    for b, t in enumerate(counts):
        for i in range(t):
            s.put(b, lens[b] + i, int(s.indptr[b]) + i)
    s.check()
    want = quantised(s.x.double())[2]
    for name, to in TYPES.items():
        k, v = kvops.read(s.cache, s.lens, s.indptr, sum(counts), dtype=to)
        assert torch.equal(k.cpu(), want[0].to(to)) and torch.equal(v.cpu(), want[1].to(to)), name
        if name != "f16":
            assert torch.equal(k.cpu().double(), want[0])  # the numbers are the type's own


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_of_special_values(kvops, dtype):
    """Zeros, borders between codes and between scales, the type's largest and smallest, infinities and NaN."""
    t = TYPES[dtype]
    fin = torch.finfo(t)
    s = Store(kvops, dtype, [0], [40], 1, 128, layers=1)
    x = torch.randn(2, 1, 40, 1, 128, generator=torch.Generator().manual_seed(3)) * 10 ** torch.linspace(-7, 4, 40)[:, None, None]
    rows = x[:, 0, :, 0]
    rows[:, 0] = 0
    rows[:, 1] = -0.0
    rows[:, 2, 0::2] = fin.max
    rows[:, 3] = -fin.max
    rows[:, 4] = fin.tiny
    rows[:, 5] = fin.smallest_normal * torch.arange(128) / 128
    rows[:, 6] = float(fin.smallest_normal) * 2.0 ** -4
    rows[:, 7, 5] = math.inf
    rows[:, 8, 40] = -math.inf
    rows[:, 9, 127] = math.nan
    rows[:, 10] = (torch.arange(128) % 32 - 16) / 2  # borders between codes at a scale of one
    rows[:, 10, ::32] = 7
    rows[:, 11] = (torch.arange(128) % 32 - 16) * 0.75
    rows[:, 12] = 7 * (1 + 1 / 32)  # a scale half way between two of five bits: to the even one
    rows[:, 13] = 7 * (1 + 3 / 32)
    rows[:, 14] = 7 * (1 + 1 / 32) * (1 + fin.eps)
    rows[:, 15] = 7 * (1 + 3 / 32) * (1 - fin.eps)
    rows[:, 16, 1:] = 0
    s.x = x.to(t)
    dev = s.x.cuda()
    kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr)
    for i in range(40):
        s.put(0, i, i)
    s.check()
    k, v = kvops.read(s.cache, s.lens, s.indptr, 40, dtype=torch.float32)
    want = quantised(s.x.double())[2]
    assert torch.equal(k.cpu().double().nan_to_num(nan=-1e300), want[0].nan_to_num(nan=-1e300))
    assert bool(v[0, 7, 0, :32].isnan().all()) and not bool(v[0, 7, 0, 32:].isnan().any())


def test_scales_next_to_the_smallest_normal_number(kvops):
    """Five bits of a number below 2^-126 are counted from its own first bit on: 31/32 of it is 0, from 63/64 on it is 2^-126."""
    s = Store(kvops, "f32", [0], [24], 1, 64, layers=1)
    s.x = torch.zeros(2, 1, 24, 1, 64)
    tiny = 2.0 ** -126
    for i, f in enumerate([0.5, 0.9375, 0.96, 0.96875, 0.975, 0.98, 63 / 64 - 2.0 ** -20, 63 / 64, 63 / 64 + 2.0 ** -20, 0.99, 1, 1.03125, 1.04, 1.1, 1.9, 1.97, 2, 3, 31, 63, 0.1, 1e-6, 0, 0.75]):
        s.x[0, 0, i, 0, i], s.x[1, 0, i, 0, 63 - i] = 7 * f * tiny, -7 * f * tiny
        s.x[:, 0, i, 0, 30] = 3 * f * tiny
    dev = s.x.cuda()
    kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr)
    for i in range(24):
        s.put(0, i, i)
    s.check()


def test_append_of_paths_bad_nodes_and_full_tables(kvops):
    s = Store(kvops, "bf16", [30, 0, 17, 60], [4, 3, 5, 8], layers=4, most=4)
    s.table_h[2, 1] = -1  # no page for positions 16 ..
    s.table_h[1, 0] = 10 ** 6
    s.cache.table.copy_(s.table_h)
    path = ints([[0, 2, 2, 3, 0], [1, 2, 0, 0, 0], [0, 1, 4, 0, 0], [7, -1, 8, 3, 2]])
    dev = s.x.cuda()
    new = kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr, path=path, n_path=ints([4, 3, 3, 9]))
    assert new.tolist() == [34, 3, 20, 64]
    for i, n in enumerate([0, 2, 2, 3]):
        s.put(0, 30 + i, n)
    s.put(3, 60, 12 + 7)  # then a token of no sequence, one past the sequence's, the table's last, nothing
    s.put(3, 63, 12 + 3)
    s.check()


def test_read_strided_unmapped_and_past_the_end(kvops):
    s = Store(kvops, "f32", [0, 40], [20, 30], kv_heads=3, dim=64, layers=3)
    dev = s.x.cuda()
    kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr)
    want = quantised(s.x.double())[2]
    s.table_h[1, 3] = -1  # positions 48 .. 63
    s.cache.table.copy_(s.table_h)
    want[:, :, 20 + 8:20 + 24] = 0
    out = torch.full((3, 2, 70, 5, 64), -7.0, device="cuda")  # [layer][k or v][token][heads and room]
    k, v = out[:, 0, :, 1:4], out[:, 1, :, 1:4]
    got = kvops.read(s.cache, s.lens, s.indptr, 70, k=k, v=v)
    assert got[0].data_ptr() == k.data_ptr()
    o = out.cpu().double()
    for i in range(2):
        assert torch.equal(o[:, i, :50, 1:4], want[i])
    o[:, :, :50, 1:4] = -7
    assert bool((o == -7).all())
    # past the table: zeros
    k, v = kvops.read(s.cache, ints([60, 10 ** 9]), ints([0, 10, 12]), 12, dtype=torch.float16)
    assert not bool(k.any() or v.any())
    k, v = kvops.read(s.cache, s.lens, ints([0, 0, 0]), 0)
    assert k.shape == (3, 0, 3, 64)


def test_append_in_a_graph_and_on_a_side_stream(kvops):
    s = Store(kvops, "bf16", [3, 9], [5, 2], layers=4)
    dev = s.x.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr)
        k0, v0 = kvops.read(s.cache, s.lens, s.indptr, 7)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr)
        k, v = kvops.read(s.cache, s.lens, s.indptr, 7)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, v0) and new.tolist() == [8, 11]
    s.lens += 6  # lengths and tokens are read when it runs
    dev.mul_(-3)
    graph.replay()
    torch.cuda.synchronize()
    want = quantised(dev[0].cpu().double())[2]
    want[:, 6] = 0  # position 16, past the table's one page
    assert new.tolist() == [14, 16] and torch.equal(k.cpu().double(), want)


def test_packed_cache_empty_reads_as_zero(kvops):
    c = kvops.PackedCache.empty(4, 2, 2, 128, ints([[0, 1], [2, 3]]), page_size=32)
    k, v = kvops.read(c, ints([0, 0]), ints([0, 64, 128]), 128, dtype=torch.float32)
    assert k.shape == (2, 128, 2, 128) and not bool(k.any() or v.any())


def test_pages_past_32_bits(kvops):
    """Codes more than 4 GB behind the start of the pool."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 11 GB")
    pages = (5 << 30) // (16 * 64 * 2)  # one layer, two heads of 1 KB
    codes = torch.empty(2, pages, 1, 2, 16, 64, dtype=torch.uint8, device="cuda")
    scales = torch.empty(2, pages, 1, 2, 16, 4, dtype=torch.bfloat16, device="cuda")
    c = kvops.PackedCache(codes[0], codes[1], scales[0], scales[1], ints([[pages - 1, pages - 2]]))
    x = torch.randn(2, 1, 20, 2, 128, generator=torch.Generator().manual_seed(0))
    dev = x.cuda()
    kvops.append(c, dev[0], dev[1], ints([5]), ints([0, 20]))
    k, v = kvops.read(c, ints([5]), ints([0, 20]), 20, dtype=torch.float32)
    want = quantised(x.double())[2]
    assert torch.equal(k.cpu().double(), want[0]) and torch.equal(v.cpu().double(), want[1])


def test_refusals(kvops):
    s = Store(kvops, "bf16", [3], [2])
    dev = s.x.cuda()
    u, sc, t = s.dev, s.dev_s, s.cache.table
    P = kvops.PackedCache
    for bad in (lambda: P(u[0].cpu(), u[1], sc[0], sc[1], t), lambda: P(u[0], u[1].int(), sc[0], sc[1], t), lambda: P(u[0], u[1], sc[0].half(), sc[1].half(), t),
                lambda: P(u[0][..., :48], u[1][..., :48], sc[0][..., :3], sc[1][..., :3], t), lambda: P(u[0], u[1], sc[0][..., :2], sc[1][..., :2], t),
                lambda: P(u[0][:, :, :, ::2], u[1][:, :, :, ::2], sc[0][:, :, :, ::2], sc[1][:, :, :, ::2], t),
                lambda: P(u[0], u[1], sc[0], sc[1], t.long()), lambda: P(u[0], u[1], sc[0], sc[1], t.expand(2, -1)),
                lambda: kvops.append(s.cache, dev[0].double(), dev[1].double(), s.lens, s.indptr), lambda: kvops.append(s.cache, dev[0], dev[1].float(), s.lens, s.indptr),
                lambda: kvops.append(s.cache, dev[0, :1], dev[1, :1], s.lens, s.indptr), lambda: kvops.append(s.cache, dev[0], dev[1], s.lens.long(), s.indptr),
                lambda: kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr, path=ints([[0]])),
                lambda: kvops.read(s.cache, s.lens, s.indptr, -1), lambda: kvops.read(s.cache, s.lens, s.indptr, 2, dtype=torch.int8),
                lambda: kvops.read(s.cache, s.lens, s.indptr, 2, dtype="bf16"), lambda: kvops.read(s.cache, s.lens, s.indptr, 2, k=dev[0]),
                lambda: kvops.read(s.cache, s.lens, s.indptr, 3, k=dev[0], v=dev[1]), lambda: kvops.read(s.cache, s.lens[:0], s.indptr, 2),
                lambda: kvops.append(s.cache, dev[0].float().requires_grad_(), dev[1].float(), s.lens, s.indptr),
                lambda: kvops.select(s.cache, torch.zeros(2, 1, 2, 16, device="cuda"), s.lens, keep=2),
                lambda: kvops.compact(s.cache, ints([[[[0], [0]]]] * 2))):
        with pytest.raises(ValueError):
            bad()
    plain = torch.zeros(4, 2, 2, 16, 128, device="cuda")
    with pytest.raises(ValueError):
        kvops.read(kvops.PagedCache(plain, plain.clone(), t), s.lens, s.indptr, 2)
    s.check()
    k = torch.zeros_like(dev)
    before = (s.cache.k._version, k._version)
    kvops.append(s.cache, dev[0], dev[1], s.lens, s.indptr)
    kvops.read(s.cache, s.lens, s.indptr, 2, k=k[0], v=k[1])
    assert s.cache.k._version > before[0] and k._version > before[1]
