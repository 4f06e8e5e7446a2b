"""What the packed-cache operators compute, and the cases they are measured at.

A decoder that keeps its paged K/V cache in 4 bits calls them one after another:

  rotate   queries and keys of new tokens: a norm of each head (where the model has one) and the rotation by
           positions of one or several axes (time, height, width)
  attend   drafted tokens over a packed cache and over one another; one drafted token is the ordinary decode step
  store    tokens quantised as they are written behind a packed cache, and read back
  read     a stretch of positions of a packed cache, all layers, as numbers again

A packed cache holds 32 consecutive dims of a position's key (or value) as 32 whole numbers c of -7 .. 7 and one
scale s, each dim is c s:
  s = the number of five significant bits nearest to max |x| / 7 (of two the even one), 0 below 2^-126, NaN where
      the 32 values are not all finite
  c = x / s to the nearest whole number (of two the even one), 0 where s is 0
c + 8 lies in the low bits first: a row of D dims is D / 4 halfwords, dim d is nibble d % 4 of halfword
(d / 4 % 8) (D / 32) + d / 32.

`run` computes them in plain torch, or, where `own` is set, by the package's kernels.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def _case(name, op, dtype, batch, context, heads=16, kv_heads=2, dim=128, page=16, layers=1, draft=1, ragged=True):
    c = {"op": op, "dtype": dtype, "batch": batch, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "page": page, "layers": layers, "draft": draft, "ragged": ragged}
    return {"name": name, **c} if name else c


def _rotate(name, dtype, tokens, heads=16, kv_heads=2, dim=128, pairs=64, axes=3, norm=False, neighbours=False, far=32768):
    c = {"op": "rotate", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "pairs": pairs,
         "axes": axes, "norm": norm, "neighbours": neighbours, "far": far}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one sequence, one token, a short document's context: the call whose latency counts
        _case("attend-1x1-f32", "attend", "f32", 1, 700, ragged=False),
        # a full serving batch, one token each, contexts of up to four thousand, in both widths of its other tensors
        _case("attend-64x1-f32", "attend", "f32", 64, 4096),
        _case("attend-64x1-bf16", "attend", "bf16", 64, 4096),
        # a tree of 16 drafts a sequence, prompts of up to 8 thousand
        _case("attend-8x16-bf16", "attend", "bf16", 8, 8448, draft=16),
        # the widest tree over one long document
        _case("attend-1x64-f16-long", "attend", "f16", 1, 131071, draft=64, ragged=False),
        # the accepted paths of a batch after a verified step, all layers
        _case("store-64x18-f32", "store", "f32", 64, 1024, layers=18, draft=16),
        # a document prompt of 1,241 tokens (image patches and text) behind an empty cache
        _case("store-1x18-prompt", "store", "bf16", 1, 0, layers=18, draft=1241, ragged=False),
        # a document's whole cache back to the engine's own type
        _case("read-1x18-f32", "read", "f32", 1, 0, layers=18, draft=1497, ragged=False),
        # stretches of eight sequences, from the middle of their caches, for operators that want 16 bits
        _case("read-8x4-bf16", "read", "bf16", 8, 1000, layers=4, draft=7448),
        # one token's queries and keys
        _rotate("rotate-1-f32", "f32", 1),
        # image patches of a 70 x 70 grid: two axes, as many keys as queries, 72 dims a head
        _rotate("rotate-4900-f16", "f16", 4900, heads=16, kv_heads=16, dim=72, pairs=36, axes=2, far=70),
        # prompts of a batch, normed and rotated in one pass
        _rotate("rotate-9928-bf16", "bf16", 9928, norm=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("attend", "attend", "attend", "store", "store", "read", "rotate", "rotate"))
        heads, kv_heads = rng.choice(((16, 2), (16, 2), (4, 2), (32, 8), (8, 8), (12, 4)))
        dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
        if op == "rotate":
            dim, pairs = rng.choice(((128, 64), (128, 64), (64, 32), (72, 36), (96, 48), (128, 32), (256, 64)))
            c = _rotate(None, dtype, _log(rng, 1, 12000), heads, kv_heads, dim, pairs, rng.choice((1, 2, 3, 3, 4)),
                        rng.random() < 0.5, rng.random() < 0.3, _log(rng, 64, 1 << 20))
        else:
            layers = 1 if op == "attend" else rng.choice((1, 2, 4, 18))
            context, draft = _log(rng, 1, 131072), _log(rng, 1, 64)
            if op != "attend" and rng.random() < 0.5:
                context, draft = rng.choice((0, context)), _log(rng, 64, 4096)
            c = _case(None, op, dtype, _log(rng, 1, 64), context, heads, kv_heads, rng.choice((128, 128, 64)),
                      rng.choice((16, 16, 32, 64)), layers, draft, rng.random() < 0.7)
        numbers = 0 if op == "rotate" else 2 * c["batch"] * (context + draft) * kv_heads * c["dim"] * layers
        if _cost(c) <= most and numbers <= 1 << 29:
            return c


# -- sizes: from the case alone ------------------------------------------------

def _lens(c):
    """Cached positions of each sequence: uneven ones spread over the last fifteen sixteenths of the range."""
    if not c["ragged"]:
        return [c["context"]] * c["batch"]
    lo = c["context"] // 16
    return [lo + int((0.61803398875 * (b + 1)) % 1.0 * (c["context"] - lo + 1)) for b in range(c["batch"])]


def _counts(c):
    """Drafted tokens of each sequence, or the positions that are read."""
    if not c["ragged"]:
        return [c["draft"]] * c["batch"]
    return [1 + int((0.75487766625 * (b + 1)) % 1.0 * c["draft"]) for b in range(c["batch"])]


def _moved(c):
    """Tokens of each sequence that are written or read: all, or a path of up to five drafts."""
    if c["op"] == "read" or c["draft"] > 64:
        return _counts(c)
    return [min(t, 1 + (5 * b + 2) % 5) for b, t in enumerate(_counts(c))]


def work(case):
    c, size = case, SIZES[case["dtype"]]
    if c["op"] == "rotate":
        rows, d = c["tokens"] * (c["heads"] + c["kv_heads"]), c["dim"]
        # rows read and written, positions; four products a pair, and the norm's square, sum and two products a value
        return {"bytes": 2.0 * rows * d * size + 4.0 * c["axes"] * c["tokens"],
                "flops": rows * (6.0 * c["pairs"] + (4.0 * d if c["norm"] else 0.0))}
    full = c["kv_heads"] * c["dim"] * size  # one position's keys (or values) of one layer
    packed = c["kv_heads"] * (c["dim"] // 2 + c["dim"] // 16)
    if c["op"] in ("store", "read"):
        # what is stored is read in full width, written packed and given back in full width
        return {"bytes": 2.0 * c["layers"] * sum(_moved(c)) * (packed + full * (2 if c["op"] == "store" else 1)), "flops": 0.0}
    lens, counts = _lens(c), _counts(c)
    q = c["heads"] * c["dim"] * size
    return {"bytes": float(2 * packed * sum(lens) + (2 * q + 2 * full + 4 * c["heads"] + 8) * sum(counts)),
            "flops": 4.0 * c["dim"] * c["heads"] * sum((n + t) * t for n, t in zip(lens, counts))}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


# -- packing, plainly ------------------------------------------------------------

def _halfword(dim, device):
    """Where the halfwords of a row's groups are: [group, halfword of the group]."""
    groups = dim // 32
    return torch.arange(8, device=device) * groups + torch.arange(groups, device=device)[:, None]


def _pack(x):
    """[..., dim] as bytes [..., dim / 2] and scales [..., dim / 32]."""
    groups = x.shape[-1] // 32
    x = x.double().unflatten(-1, (groups, 32))
    m, e = torch.frexp(x.abs().amax(-1) / 7)
    s = torch.ldexp(torch.round(m * 32) / 32, e)
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    s = torch.where(torch.isfinite(x).all(-1), s, math.nan)
    c = torch.where(s[..., None] > 0, torch.round(x / s[..., None]), 0.0).to(torch.int32) + 8
    c = c.unflatten(-1, (8, 4))
    half = c[..., 0] | c[..., 1] << 4 | c[..., 2] << 8 | c[..., 3] << 12
    row = torch.empty(half.shape[:-2] + (groups * 8,), dtype=torch.int32, device=x.device)
    row[..., _halfword(groups * 32, x.device).flatten()] = half.flatten(-2)
    return torch.stack((row & 255, row >> 8), -1).flatten(-2).to(torch.uint8), s.to(torch.bfloat16)


def _unpack(rows, scales):
    """The numbers that packed rows stand for, in 32 bits (exactly)."""
    b = rows.to(torch.int32).unflatten(-1, (-1, 2))
    half = (b[..., 0] | b[..., 1] << 8)[..., _halfword(rows.shape[-1] * 2, rows.device)]  # [..., groups, 8]
    c = torch.stack([(half >> 4 * i & 15) - 8 for i in range(4)], -1).flatten(-2).float()
    return (c * scales.float()[..., None]).flatten(-2)


# -- inputs ----------------------------------------------------------------------

def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    dtype = TYPES[c["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, scale, generator=g)

    if c["op"] == "rotate":
        N, H, KVH, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        qkv = normal(N, (H + 2 * KVH) * D, scale=1.5)  # one projection's output: queries and keys are views of it
        s = {"case": c, "q": qkv[:, :H * D].view(N, H, D), "k": qkv[:, H * D:(H + KVH) * D].view(N, KVH, D),
             "pos": torch.randint(0, c["far"], (N, c["axes"]), generator=g, device=dev, dtype=torch.int32)}
        each = c["pairs"] // c["axes"]
        first = c["pairs"] - each * (c["axes"] - 1)
        s["sections"] = [first] + [each] * (c["axes"] - 1)
        s["freq"] = BASE ** (-torch.arange(c["pairs"], dtype=torch.float64, device=dev) / c["pairs"])
        s["axis"] = torch.repeat_interleave(torch.arange(c["axes"], device=dev), torch.tensor(s["sections"], device=dev))
        s["qw"], s["kw"] = (normal(D, scale=0.2) + 1, normal(D, scale=0.2) + 1) if c["norm"] else (None, None)
        if own:
            from rapidocrvl_b200 import kvops

            s["rotary"] = kvops.Rotary(D, theta=BASE, pairs=c["pairs"], sections=s["sections"], neighbours=c["neighbours"])
        return s

    B, L, KVH, D, page = c["batch"], c["layers"], c["kv_heads"], c["dim"], c["page"]
    lens, counts = _lens(c), _counts(c)
    N = sum(counts)
    room = [n + (t if c["op"] != "attend" else 0) for n, t in zip(lens, _moved(c))]
    pages = [-(-n // page) for n in room]
    total = max(1, sum(pages))
    order = torch.randperm(total, generator=h)
    table = torch.full((B, max(1, max(pages))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": c, "scale": 1.0 / math.sqrt(D), "table": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
         "most": max(lens), "indptr": torch.tensor([0] + [sum(counts[:b + 1]) for b in range(B)], dtype=torch.int32, device=dev)}
    for x in ("k", "v"):
        s[x] = torch.empty(total, L, KVH, page, D // 2, dtype=torch.uint8, device=dev)
        s[x + "s"] = torch.empty(total, L, KVH, page, D // 32, dtype=torch.bfloat16, device=dev)
        step = max(1, (1 << 25) // (L * KVH * page * D))
        # a few dims of all keys lie off zero, as they do in models
        off = torch.empty(L, KVH, 1, D, device=dev).normal_(0.0, 1.0, generator=g)
        off = torch.where(off.abs() > 1.7, 2 * off, 0.0) if x == "k" else 0 * off
        for i in range(0, total, step):  # a part at a time: packing takes room
            part = torch.empty(min(step, total - i), L, KVH, page, D, device=dev).normal_(0.0, 1.0, generator=g)
            s[x][i:i + step], s[x + "s"][i:i + step] = _pack(part + off)
    if c["op"] == "attend":
        s["q"] = normal(N, c["heads"], D, scale=1.5)
        s["dk"], s["dv"] = normal(N, KVH, D), normal(N, KVH, D)
        masks = []
        for t in counts:  # a node sees itself and what its parent sees; parents are drawn
            up = torch.rand(t, generator=h).tolist()
            seen = []
            for i in range(t):
                seen.append((seen[int(up[i] * i)] if i else 0) | 1 << i)
            masks += [m - (1 << 64) if m >> 63 else m for m in seen]
        s["mask"] = torch.tensor(masks, dtype=torch.int64, device=dev)
    else:
        moved = _moved(c)
        s["moved"] = torch.tensor([0] + [sum(moved[:b + 1]) for b in range(B)], dtype=torch.int32, device=dev)
        s["tokens"] = sum(moved)
    if c["op"] == "store":
        s["dk"], s["dv"] = normal(L, N, KVH, D), normal(L, N, KVH, D)
        path = torch.zeros(B, max(moved), dtype=torch.int32)
        for b, (n, t) in enumerate(zip(moved, counts)):
            path[b, :n] = torch.randperm(t, generator=h)[:n].sort().values
        s["path"], s["n_path"] = path.to(dev), torch.tensor(moved, dtype=torch.int32, device=dev)
    if own:
        from rapidocrvl_b200 import kvops

        s["cache"] = kvops.PackedCache(s["k"], s["v"], s["ks"], s["vs"], s["table"])
    return s


BASE = 500000.0  # of the rotation's frequencies
EPS = 1e-5       # of the norms


# -- the operators, plainly --------------------------------------------------------

def _rows(s, which):
    """Keys ("k") or values ("v") by position: [batch, kv heads, positions, dim]."""
    at = s["table"].clamp(min=0).long()
    t = _unpack(s[which][at, 0], s[which + "s"][at, 0])  # [batch, pages, kv heads, page, dim]
    return t.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :s["most"]]


def _padded(s, x):
    """A flat [tokens, heads, dim] as [batch, heads, draft, dim], and where the tokens are in it."""
    n = s["indptr"].long()
    token = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(n, token, right=True) - 1
    out = torch.zeros(n.numel() - 1, s["case"]["draft"], *x.shape[1:], device=x.device)
    out[seq, token - n[seq]] = x.float()
    return out.transpose(1, 2), seq, token - n[seq]


def _attend(s):
    c = s["case"]
    B, H, KVH, D, T = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["draft"]
    q, seq, place = _padded(s, s["q"])
    dk, dv = _padded(s, s["dk"])[0], _padded(s, s["dv"])[0]
    q = q.reshape(B, KVH, H // KVH * T, D)
    cached = (torch.arange(s["most"], device=q.device) < s["lens"][:, None])[:, None, None, None]
    bits = torch.zeros(B, T, dtype=torch.int64, device=q.device)
    bits[seq, place] = s["mask"]
    seen = (bits[:, :, None] >> torch.arange(T, device=q.device) & 1).bool()[:, None, None]
    a = (q @ _rows(s, "k").transpose(-1, -2) * s["scale"]).view(B, KVH, H // KVH, T, -1).masked_fill(~cached, -math.inf)
    d = (q @ dk.transpose(-1, -2) * s["scale"]).view(B, KVH, H // KVH, T, T).masked_fill(~seen, -math.inf)
    both = torch.cat((a, d), -1)
    top = both.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(both - top)
    total = w.sum(-1, keepdim=True)
    w = w.reshape(B, KVH, -1, w.shape[-1])
    out = w[..., :s["most"]] @ _rows(s, "v") + w[..., s["most"]:] @ dv
    out = out.view(B, KVH, H // KVH, T, D) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total))[..., 0]
    out, lse = out.reshape(B, H, T, D), lse.reshape(B, H, T)
    return out[seq, :, place].to(s["q"].dtype), lse[seq, :, place].contiguous()


def _read(s):
    n = s["moved"].long()
    token = torch.arange(s["tokens"], device=n.device)
    seq = torch.searchsorted(n, token, right=True) - 1
    at, page = s["lens"][seq] + token - n[seq], s["case"]["page"]
    where = s["table"][seq, at // page].long()
    return tuple(_unpack(s[x][where, :, :, at % page], s[x + "s"][where, :, :, at % page]).transpose(0, 1).contiguous()
                 .to(TYPES[s["case"]["dtype"]]) for x in ("k", "v"))


def _store(s):
    n, page = s["n_path"], s["case"]["page"]
    there = torch.arange(s["path"].shape[1], device=n.device) < n[:, None]
    seq, i = torch.nonzero(there, as_tuple=True)
    token = s["indptr"][seq] + s["path"][seq, i]
    at = s["lens"][seq] + i
    where = s["table"][seq, at // page].long()
    for x in ("k", "v"):
        rows, scales = _pack(s["d" + x][:, token].transpose(0, 1))
        s[x][where, :, :, at % page] = rows
        s[x + "s"][where, :, :, at % page] = scales
    return (*_read(s), s["lens"] + n)


def _rotated(s):
    c, P = s["case"], s["case"]["pairs"]
    angle = s["pos"].double()[:, s["axis"]] * s["freq"]  # far positions: 32 bits would lose their last turns
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        r = y[..., :2 * P]
        u, v = (r[..., 0::2], r[..., 1::2]) if c["neighbours"] else (r[..., :P], r[..., P:])
        u, v = u * cos - v * sin, v * cos + u * sin
        r = torch.stack((u, v), -1).flatten(-2) if c["neighbours"] else torch.cat((u, v), -1)
        out.append(torch.cat((r, y[..., 2 * P:]), -1).to(x.dtype))
    return tuple(out)


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"attend": _attend, "store": _store, "read": _read, "rotate": _rotated}[op](s)
    from rapidocrvl_b200 import kvops

    if op == "rotate":
        return kvops.rotate(s["q"], s["k"], s["pos"], s["rotary"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
    if op == "attend":
        return kvops.tree_attention(s["q"], s["dk"], s["dv"], s["cache"], s["lens"], s["indptr"], s["mask"],
                                    max_draft=s["case"]["draft"], scale=s["scale"])
    dtype = TYPES[s["case"]["dtype"]]
    if op == "read":
        return kvops.read(s["cache"], s["lens"], s["moved"], s["tokens"], dtype=dtype)
    lens = kvops.append(s["cache"], s["dk"], s["dv"], s["lens"], s["indptr"], path=s["path"], n_path=s["n_path"])
    return (*kvops.read(s["cache"], s["lens"], s["moved"], s["tokens"], dtype=dtype), lens)


# -- the operators, from their definitions in 64 bits ------------------------------

def _exact_numbers(rows, scales):
    """What packed rows [n, dim / 2] stand for, dim by dim."""
    D = rows.shape[-1] * 2
    out = torch.empty(rows.shape[0], D, dtype=torch.float64, device=rows.device)
    for d in range(D):
        nibble = 4 * ((d // 4 % 8) * (D // 32) + d // 32) + d % 4
        byte = rows[:, nibble // 2].long()
        out[:, d] = ((byte // 16 if nibble % 2 else byte % 16) - 8) * scales[:, d // 32].double()
    return out


def _exact_rounded(x):
    """What a row [n, dim] becomes by being packed and read."""
    out = np.empty(x.shape)
    for j in range(0, x.shape[1], 32):
        v = x[:, j:j + 32]
        top = np.abs(v).max(1) / 7
        with np.errstate(divide="ignore"):
            unit = np.exp2(np.floor(np.log2(top)) - 4)  # of the fifth bit
        unit = np.where(top > 0, unit, 1.0)
        unit = np.where(top / unit >= 32, 2 * unit, np.where(top / unit < 16, unit / 2, unit))  # log2 is rounded itself
        s = np.rint(top / unit) * unit
        s = np.where(s < 2.0 ** -126, 0.0, s)[:, None]
        # the whole number by counting the borders below |x|: (i + 1/2) s itself goes to the even one
        c = np.zeros(v.shape)
        for i in range(7):
            border = (i + 0.5) * s
            c += (np.abs(v) > border) | ((np.abs(v) == border) & (i % 2 == 1))
        out[:, j:j + 32] = np.where(s > 0, np.sign(v) * c * s, 0.0)
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotate":
        P, out = c["pairs"], []
        turn = [np.float64(BASE) ** (-i / P) for i in range(P)]
        axis = [a for a, n in enumerate(s["sections"]) for _ in range(n)]
        pos = s["pos"].cpu().numpy().astype(np.float64)
        z = np.stack([np.exp(1j * pos[:, axis[i]] * turn[i]) for i in range(P)], 1)
        z = torch.from_numpy(z).cuda()[:, None]
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            y = x.double()
            if w is not None:
                y = w.double() * y / torch.sqrt(y.square().sum(-1, keepdim=True) / c["dim"] + EPS)
            y = y.clone()
            u, v = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if c["neighbours"] else (slice(0, P), slice(P, 2 * P))
            r = torch.complex(y[..., u], y[..., v]) * z
            y[..., u], y[..., v] = r.real, r.imag
            out.append(y)
        return tuple(out)
    lens, counts, moved = _lens(c), _counts(c), _moved(c)
    B, H, KVH, page, L, D = c["batch"], c["heads"], c["kv_heads"], c["page"], c["layers"], c["dim"]
    if c["op"] == "store":
        if 2 * L * KVH * D * sum(moved) > 1 << 26:
            return None
        out = []
        for x in ("dk", "dv"):
            token = [sum(counts[:b]) + t for b, n in enumerate(moved) for t in s["path"][b, :n].tolist()]
            y = s[x][:, token].double().cpu().numpy()
            out.append(torch.from_numpy(_exact_rounded(y.reshape(-1, D)).reshape(y.shape)))
        return (*out, torch.tensor([n + a for n, a in zip(lens, moved)], dtype=torch.int32))
    if c["op"] == "read":
        out = []
        for x in ("k", "v"):
            parts = []
            for b, n in enumerate(moved):
                at = lens[b] + torch.arange(n, device="cuda")
                pages = s["table"][b, at // page].long()
                rows, scales = s[x][pages, :, :, at % page], s[x + "s"][pages, :, :, at % page]  # [n, layers, kv heads, ...]
                y = _exact_numbers(rows.flatten(0, 2), scales.flatten(0, 2))
                parts.append(y.view(n, L, KVH, D).transpose(0, 1))
            out.append(torch.cat(parts, 1))
        return tuple(out)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, t) in enumerate(zip(lens, counts)):
        at = torch.arange(n, device="cuda")
        pages = s["table"][b, at // page].long()
        of = slice(first, first + t)
        see = torch.tensor([[bool(m >> j & 1) for j in range(t)] for m in s["mask"][of].tolist()], device="cuda")
        for k in range(KVH):
            keys = _exact_numbers(s["k"][pages, 0, k, at % page], s["ks"][pages, 0, k, at % page])
            values = _exact_numbers(s["v"][pages, 0, k, at % page], s["vs"][pages, 0, k, at % page])
            values = torch.cat((values, s["dv"][of, k].double()))
            for hd in range(k * H // KVH, (k + 1) * H // KVH):
                q = s["q"][of, hd].double() / math.sqrt(D)
                x = torch.cat((q @ keys.T, torch.where(see, q @ s["dk"][of, k].double().T, -math.inf)), 1)
                lse[of, hd] = torch.logsumexp(x, 1)
                out[of, hd] = torch.softmax(x, 1) @ values
        first += t
    return out, lse
