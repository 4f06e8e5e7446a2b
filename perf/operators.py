"""What the paged-cache operators compute, and the cases they are measured at.

Four operators on a paged K/V cache, as a decoder that drafts tokens and drops cache positions uses them:

  tree    attention of drafted tokens (a tree given by one bit mask a token) over a cache and over one another;
          one drafted token is the ordinary decode step
  mass    the attention weight that cached positions received from the drafted tokens, added to a running sum
  evict   the positions with the largest sums, the first and the last ones are kept: their indices, and the cache
          and the sums moved together
  append  accepted drafts written behind the cache

`run` computes them in plain torch, or, where `own` is set, by the package's kernels.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def _case(name, op, dtype, batch, context, heads=16, kv_heads=2, dim=128, page=16, layers=1, draft=1, ragged=True, keep=0):
    c = {"op": op, "dtype": dtype, "batch": batch, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "page": page, "layers": layers, "draft": draft, "ragged": ragged, "keep": keep}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one sequence, one token, a short document's context: the call whose latency counts
        _case("tree-1x1-f32", "tree", "f32", 1, 648, ragged=False),
        # a full serving batch, one token each, contexts of one to four thousand
        _case("tree-64x1-f32", "tree", "f32", 64, 4096),
        # a few drafts a sequence over an f32 cache, eight sequences of uneven length
        _case("tree-8x12-f32", "tree", "f32", 8, 4095, draft=12),
        # a tree of 16 drafts a sequence, 16-bit cache, prompts of up to 8 thousand
        _case("tree-8x16-bf16", "tree", "bf16", 8, 8448, draft=16),
        # the widest tree over one long document
        _case("tree-1x64-bf16-long", "tree", "bf16", 1, 131071, draft=64, ragged=False),
        # sums kept up at every decode step of a batch
        _case("mass-64x1-f32", "mass", "f32", 64, 4096),
        # a window of 32 last prompt tokens votes on what to keep
        _case("mass-4x32-bf16", "mass", "bf16", 4, 8448, draft=32),
        # one document's whole cache (18 layers) cut to 512 positions
        _case("evict-1x18-f32", "evict", "f32", 1, 1257, layers=18, keep=512, ragged=False),
        # eight sequences cut to a budget, some of them already under it
        _case("evict-8x4-bf16", "evict", "bf16", 8, 8448, layers=4, keep=1024),
        # one very long context in grouped heads: choosing is most of the work
        _case("evict-1x2-f16-long", "evict", "f16", 1, 131072, heads=32, kv_heads=8, layers=2, keep=4096, ragged=False),
        # the accepted paths of a batch after a verified step, all layers
        _case("append-64x18-f32", "append", "f32", 64, 1024, layers=18, draft=16),
        # a document prompt of 1,241 tokens (image patches and text) behind an empty cache
        _case("append-1x18-prompt", "append", "bf16", 1, 0, layers=18, draft=1241, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("tree", "tree", "tree", "mass", "mass", "evict", "evict", "append"))
        heads, kv_heads = rng.choice(((16, 2), (16, 2), (4, 2), (32, 8), (8, 8), (12, 4)))
        dim = rng.choice((128, 128, 64))
        layers = 1 if op in ("tree", "mass") else rng.choice((1, 2, 4, 18))
        context = _log(rng, 1, 131072)
        draft = 0 if op == "evict" else _log(rng, 1, 64)
        if op == "append" and rng.random() < 0.3:
            context, draft = rng.choice((0, context)), _log(rng, 64, 2048)
        c = _case(None, op, rng.choice(("f32", "bf16", "bf16", "f16")), _log(rng, 1, 64), context, heads, kv_heads, dim,
                  rng.choice((16, 16, 32, 64)), layers, draft, rng.random() < 0.7,
                  min(context, max(64, _log(rng, max(1, context // 32), context))) if op == "evict" else 0)
        pool = 2 * c["batch"] * (context + draft) * kv_heads * dim * layers * SIZES[c["dtype"]]
        if _cost(c) <= most and pool <= 3 << 30:
            return c


# -- sizes: from the case alone ------------------------------------------------

def _lens(c):
    """Cached positions of each sequence: uneven ones spread over the last fifteen sixteenths of the range."""
    if not c["ragged"]:
        return [c["context"]] * c["batch"]
    lo = c["context"] // 16
    return [lo + int((0.61803398875 * (b + 1)) % 1.0 * (c["context"] - lo + 1)) for b in range(c["batch"])]


def _counts(c):
    """Drafted tokens of each sequence."""
    if not c["ragged"]:
        return [c["draft"]] * c["batch"]
    return [1 + int((0.75487766625 * (b + 1)) % 1.0 * c["draft"]) for b in range(c["batch"])]


def _accepted(c):
    """Tokens of each sequence that are appended: a prompt whole, or a path of up to five drafts."""
    return [t if c["draft"] > 64 else min(t, 1 + (5 * b + 2) % 5) for b, t in enumerate(_counts(c))]


def work(case):
    c, size = case, SIZES[case["dtype"]]
    row = c["kv_heads"] * c["dim"] * size  # one position's keys (or values) of one layer
    lens = _lens(c)
    if c["op"] == "evict":
        kept = [min(n, c["keep"]) for n in lens]
        rows = c["layers"] * c["kv_heads"]
        # sums read, indices and kept sums written, kept keys and values read and written
        return {"bytes": 4.0 * rows * sum(lens) + 8.0 * rows * sum(kept) + 4.0 * c["layers"] * row * sum(kept), "flops": 0.0}
    if c["op"] == "append":
        return {"bytes": 4.0 * c["layers"] * row * sum(_accepted(c)), "flops": 0.0}
    counts = _counts(c)
    q = c["heads"] * c["dim"] * size
    if c["op"] == "mass":
        return {"bytes": float(row * sum(lens) + (q + 4 * c["heads"]) * sum(counts) + 8 * c["kv_heads"] * sum(lens)),
                "flops": 2.0 * c["dim"] * c["heads"] * sum(n * t for n, t in zip(lens, counts))}
    return {"bytes": float(2 * row * sum(lens) + (2 * q + 2 * row + 4 * c["heads"] + 8) * sum(counts)),
            "flops": 4.0 * c["dim"] * c["heads"] * sum((n + t) * t for n, t in zip(lens, counts))}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


# -- inputs ----------------------------------------------------------------------

def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    B, L, KVH, D, page = c["batch"], c["layers"], c["kv_heads"], c["dim"], c["page"]
    lens, counts = _lens(c), _counts(c)
    N = sum(counts)

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, scale, generator=g)

    room = [n + (t if c["op"] == "append" else 0) for n, t in zip(lens, _accepted(c))]
    pages = [-(-n // page) for n in room]
    total = max(1, sum(pages))
    order = torch.randperm(total, generator=h)
    table = torch.full((B, max(1, max(pages))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": c, "scale": 1.0 / math.sqrt(D), "table": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
         "most": max(lens), "pool": normal(total, L, KVH, 2, page, D),
         "indptr": torch.tensor([0] + [sum(counts[:b + 1]) for b in range(B)], dtype=torch.int32, device=dev)}
    if c["op"] in ("tree", "mass"):
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
    if c["op"] == "mass":
        s["lse"] = _tree(s)[1]
        s["acc"] = torch.rand(B, KVH, table.shape[1] * page, generator=g, device=dev)
    if c["op"] == "evict":
        width = table.shape[1] * page
        acc = torch.empty(L, B, KVH, width, device=dev).normal_(0.0, 2.0, generator=g).exp_()
        # some positions were never attended: their sums are 0 and tie
        s["acc"] = acc * (torch.rand(acc.shape, generator=g, device=dev) > 0.1)
        kept = [-(-min(n, c["keep"]) // page) for n in lens]
        new = torch.full((B, max(1, max(kept))), -1, dtype=torch.int32)
        order, at = torch.randperm(max(1, sum(kept)), generator=h), 0
        for b, n in enumerate(kept):
            new[b, :n] = order[at:at + n]
            at += n
        s["new_table"] = new.to(dev)
        s["new_pool"] = torch.zeros(max(1, sum(kept)), L, KVH, 2, page, D, dtype=dtype, device=dev)
        s["sinks"], s["recent"] = min(4, c["keep"]), min(32, max(0, c["keep"] - 4))
    if c["op"] == "append":
        s["dk"], s["dv"] = normal(L, N, KVH, D), normal(L, N, KVH, D)
        n_path = _accepted(c)
        path = torch.zeros(B, max(n_path), dtype=torch.int32)
        for b, (n, t) in enumerate(zip(n_path, counts)):
            path[b, :n] = torch.randperm(t, generator=h)[:n].sort().values
        s["path"], s["n_path"] = path.to(dev), torch.tensor(n_path, dtype=torch.int32, device=dev)
    if own:
        from rapidocrvl_b200 import kvops

        s["cache"] = kvops.PagedCache(s["pool"][:, :, :, 0], s["pool"][:, :, :, 1], s["table"])
        if c["op"] == "evict":
            s["new_cache"] = kvops.PagedCache(s["new_pool"][:, :, :, 0], s["new_pool"][:, :, :, 1], s["new_table"])
    return s


# -- the operators, plainly --------------------------------------------------------

def _rows(s, which):
    """Layer 0's keys (0) or values (1) by position, in 32 bits: [batch, kv heads, positions, dim]."""
    t = s["pool"][:, 0, :, which][s["table"].clamp(min=0).long()]  # [batch, pages, kv heads, page, dim]
    return t.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :s["most"]].float()


def _padded(s, x):
    """A flat [tokens, heads, dim] as [batch, heads, draft, dim], and where the tokens are in it."""
    n = s["indptr"].long()
    token = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(n, token, right=True) - 1
    out = torch.zeros(n.numel() - 1, s["case"]["draft"], *x.shape[1:], device=x.device)
    out[seq, token - n[seq]] = x.float()
    return out.transpose(1, 2), seq, token - n[seq]


def _tree(s):
    c = s["case"]
    B, H, KVH, D, T = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["draft"]
    q, seq, place = _padded(s, s["q"])
    dk, dv = _padded(s, s["dk"])[0], _padded(s, s["dv"])[0]
    q = q.reshape(B, KVH, H // KVH * T, D)
    cached = (torch.arange(s["most"], device=q.device) < s["lens"][:, None])[:, None, None, None]
    bits = torch.zeros(B, T, dtype=torch.int64, device=q.device)
    bits[seq, place] = s["mask"]
    seen = (bits[:, :, None] >> torch.arange(T, device=q.device) & 1).bool()[:, None, None]
    a = (q @ _rows(s, 0).transpose(-1, -2) * s["scale"]).view(B, KVH, H // KVH, T, -1).masked_fill(~cached, -math.inf)
    d = (q @ dk.transpose(-1, -2) * s["scale"]).view(B, KVH, H // KVH, T, T).masked_fill(~seen, -math.inf)
    both = torch.cat((a, d), -1)
    top = both.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(both - top)
    total = w.sum(-1, keepdim=True)
    w = w.reshape(B, KVH, -1, w.shape[-1])
    out = w[..., :s["most"]] @ _rows(s, 1) + w[..., s["most"]:] @ dv
    out = out.view(B, KVH, H // KVH, T, D) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total))[..., 0]
    out, lse = out.reshape(B, H, T, D), lse.reshape(B, H, T)
    return out[seq, :, place].to(s["q"].dtype), lse[seq, :, place].contiguous()


def _mass(s):
    c = s["case"]
    B, H, KVH, D, T = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["draft"]
    q, seq, place = _padded(s, s["q"])
    lse = torch.full((B, T, H), math.inf, device=q.device)
    lse[seq, place] = s["lse"]
    a = q.reshape(B, KVH, -1, D) @ _rows(s, 0).transpose(-1, -2) * s["scale"]
    w = torch.exp(a - lse.transpose(1, 2).reshape(B, KVH, -1, 1)).sum(2)
    there = torch.arange(s["acc"].shape[-1], device=q.device) < s["lens"][:, None]
    acc = s["acc"] * DECAY
    acc[:, :, :s["most"]] += w
    return acc.masked_fill(~there[:, None], 0.0)


def _evict(s):
    c, acc, lens = s["case"], s["acc"], s["lens"][:, None, None]
    t = torch.arange(acc.shape[-1], device=acc.device)
    always = (t < s["sinks"]) | (t >= lens - s["recent"])
    order = torch.where(always, math.inf, acc).masked_fill(t >= lens, -math.inf)
    chosen = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    fine = torch.arange(chosen.shape[-1], device=acc.device) < torch.clamp(lens, max=c["keep"])
    idx = torch.where(fine, chosen, acc.shape[-1]).sort(-1).values  # [layers, batch, kv heads, kept]
    fine = fine.expand(idx.shape)
    sums = torch.where(fine, acc.gather(-1, idx.clamp(max=acc.shape[-1] - 1)), 0.0)
    layer, seq, head, new = torch.nonzero(fine, as_tuple=True)
    old, page = idx[layer, seq, head, new], c["page"]
    s["new_pool"][s["new_table"][seq, new // page].long(), layer, head, :, new % page] = \
        s["pool"][s["table"][seq, old // page].long(), layer, head, :, old % page]
    idx = torch.where(fine, idx, -1).int()
    width = c["keep"] - idx.shape[-1]
    if width > 0:
        idx, sums = torch.nn.functional.pad(idx, (0, width), value=-1), torch.nn.functional.pad(sums, (0, width))
    return idx, sums, s["new_pool"], torch.clamp(s["lens"], max=c["keep"])


def _append(s):
    c, n, page = s["case"], s["n_path"], s["case"]["page"]
    there = torch.arange(s["path"].shape[1], device=n.device) < n[:, None]
    seq, i = torch.nonzero(there, as_tuple=True)
    token = s["indptr"][seq] + s["path"][seq, i]
    at = s["lens"][seq] + i
    where = s["table"][seq, at // page].long()
    s["pool"][where, :, :, 0, at % page] = s["dk"][:, token].transpose(0, 1)
    s["pool"][where, :, :, 1, at % page] = s["dv"][:, token].transpose(0, 1)
    return s["pool"], s["lens"] + n


DECAY = 0.97  # how much of the sums so far stays at each step


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"tree": _tree, "mass": _mass, "evict": _evict, "append": _append}[op](s)
    from rapidocrvl_b200 import kvops

    if op == "tree":
        return kvops.tree_attention(s["q"], s["dk"], s["dv"], s["cache"], s["lens"], s["indptr"], s["mask"],
                                    max_draft=s["case"]["draft"], scale=s["scale"])
    if op == "mass":
        return kvops.attention_mass(s["q"], s["lse"], s["cache"], s["lens"], s["indptr"], max_draft=s["case"]["draft"],
                                    scale=s["scale"], acc=s["acc"], decay=DECAY)
    if op == "evict":
        idx, sums, lens = kvops.evict(s["cache"], s["acc"], s["lens"], keep=s["case"]["keep"], sinks=s["sinks"],
                                      recent=s["recent"], into=s["new_cache"])
        return idx, sums, s["new_pool"], lens
    lens = kvops.append(s["cache"], s["dk"], s["dv"], s["lens"], s["indptr"], path=s["path"], n_path=s["n_path"])
    return s["pool"], lens


# -- the operators, from their definitions in 64 bits, one sequence and head at a time ----

def exact(case, seed):
    c, s = case, prepare(case, seed)
    lens, counts = _lens(c), _counts(c)
    B, H, KVH, page, L = c["batch"], c["heads"], c["kv_heads"], c["page"], c["layers"]
    if c["op"] == "append":
        pool = s["pool"].clone()
        for b, n in enumerate(_accepted(c)):
            first = sum(counts[:b])
            at = lens[b] + torch.arange(n, device="cuda")
            pages, tokens = s["table"][b, at // page].long(), first + s["path"][b, :n].long()
            for l in range(L):
                pool[pages, l, :, 0, at % page] = s["dk"][l, tokens]
                pool[pages, l, :, 1, at % page] = s["dv"][l, tokens]
        return pool, torch.tensor([n + a for n, a in zip(lens, _accepted(c))], dtype=torch.int32)
    if c["op"] == "evict":
        keep, host = c["keep"], s["acc"].cpu()
        idx = torch.full((L, B, KVH, keep), -1, dtype=torch.int32)
        sums, pool = torch.zeros(L, B, KVH, keep, dtype=torch.float64), s["new_pool"].clone()
        for b, n in enumerate(lens):
            held = min(n, keep)
            new = torch.arange(held, device="cuda")
            for l in range(L):
                for k in range(KVH):
                    row = host[l, b, k, :n].double().numpy()
                    lo, hi = s["sinks"], n - s["recent"]
                    kept = np.arange(n)
                    if n > keep:  # the largest of the middle; a stable order puts the lower position first
                        top = lo + np.argsort(-row[lo:hi], kind="stable")[:keep - s["sinks"] - s["recent"]]
                        kept = np.sort(np.concatenate((kept[:lo], top, kept[hi:])))
                    idx[l, b, k, :held] = torch.from_numpy(kept).int()
                    sums[l, b, k, :held] = torch.from_numpy(row[kept])
                    old = torch.from_numpy(kept).cuda()
                    pool[s["new_table"][b, new // page].long(), l, k, :, new % page] = \
                        s["pool"][s["table"][b, old // page].long(), l, k, :, old % page]
        return idx, sums, pool, torch.tensor([min(n, keep) for n in lens], dtype=torch.int32)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    acc = torch.zeros(s["acc"].shape, dtype=torch.float64, device="cuda") if c["op"] == "mass" else None
    first = 0
    for b, (n, t) in enumerate(zip(lens, counts)):
        at = torch.arange(n, device="cuda")
        pages = s["table"][b, at // page].long()
        of = slice(first, first + t)
        if c["op"] == "tree":
            see = torch.tensor([[bool(m >> j & 1) for j in range(t)] for m in s["mask"][of].tolist()], device="cuda")
        for hd in range(H):
            k = hd * KVH // H
            keys = s["pool"][pages, 0, k, 0, at % page].double()
            x = s["q"][of, hd].double() @ keys.T / math.sqrt(c["dim"])
            if c["op"] == "mass":
                acc[b, k, :n] += torch.exp(x - s["lse"][of, hd].double()[:, None]).sum(0)
                continue
            y = s["q"][of, hd].double() @ s["dk"][of, k].double().T / math.sqrt(c["dim"])
            x = torch.cat((x, torch.where(see, y, -math.inf)), 1)
            lse[of, hd] = torch.logsumexp(x, 1)
            values = torch.cat((s["pool"][pages, 0, k, 1, at % page], s["dv"][of, k])).double()
            out[of, hd] = torch.softmax(x, 1) @ values
        if c["op"] == "mass":
            acc[b, :, :n] += DECAY * s["acc"][b, :, :n].double()
        first += t
    return acc if c["op"] == "mass" else (out, lse)
