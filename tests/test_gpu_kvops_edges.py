"""The paged-cache operators (rapidocrvl_b200.kvops) where they can go wrong:
values that are not finite or as large as the type goes, scores that rise
along the context, rows and pages with nothing in them, on every shape of
kernel.  Setup, types and the tolerances' derivation are test_gpu_kvops.py's;
what a test adds to them is said there."""
import math

import pytest
import torch

from test_gpu_kvops import REL, Setup, kvops, masks, mass_check, mass_want  # noqa: F401 (kvops: the fixture)

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
    mask, group = s.mask.cpu(), H // s.kv_heads
    for b, t in enumerate(s.counts):
        i0 = int(s.indptr[b])
        ck, cv = s.rows(b)
        if see_cached is not None:
            ck, cv = ck[see_cached[b]], cv[see_cached[b]]
        for i in range(i0, i0 + t):
            see = [i0 + j for j in range(t) if int(mask[i]) >> j & 1]
            if not len(ck) and not see:
                continue
            keys, values = torch.cat((ck, k[see])), torch.cat((cv, v[see]))  # [n, kv heads, D]
            x = torch.einsum("ngd,ghd->ghn", keys, q[i].view(s.kv_heads, group, D)) * s.scale
            lse[i] = torch.logsumexp(x, -1).view(H)
            w = torch.softmax(x, -1)
            o = torch.einsum("ghn,ngd->ghd", w, values)
            out[i] = o.reshape(H, D)
            top[i] = values.abs().amax((0, 2)).repeat_interleave(group)[:, None]
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
