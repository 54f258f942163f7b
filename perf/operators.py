"""Operators of a cache that many sequences share and that forgets, as cases that can be timed and compared.

Three operators over the paged cache (pages of 64 positions, [pages, key/value heads, 64, head size]):

* ``prefix``: attention of one new token a sequence where groups of sequences have their first pages in common.
  out[b, h] = sum_j softmax_j(q[b, h] . k[j]) v[j] over the shared positions and the sequence's own, its newest included.
* ``weighed``: causal attention of runs of new tokens that also keeps, for every cached position and key/value head, the
  sum of the softmax weights it has been given: w[j] <- (w[j] if j was cached before this call, else 0) + sum of p[i, h, j]
  over the run's queries i (all, or the last so many) and the query heads h of the head.
* ``evict``: each key/value head of a sequence keeps its first and its most recent positions and, of those between, the ones
  with the largest sums; their keys, values and sums move, in order, to the head of the sequence's new pages.

``run`` with ``own`` false states them with elementary torch operations in 32 bits; ``exact`` states them again in 64 bits.
"""
import math
import random

import torch

own = False

PAGE = 64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # two answers to one short question: the smallest call, where launches are all there is
        dict(name="prefix: two answers", op="prefix", dtype="bfloat16", heads=32, kv=32, hd=64, batch=2, groups=1, shared=128, low=1, high=40),
        # four applications, each with instructions of its own length in front of its users' questions
        dict(name="prefix: four preambles", op="prefix", dtype="bfloat16", heads=32, kv=8, hd=128, batch=64, groups=4, shared=8192, low=1, high=700),
        # a crowd of questions to one long document: the shared products are work for the tensor cores
        dict(name="prefix: one document", op="prefix", dtype="bfloat16", heads=32, kv=8, hd=128, batch=128, groups=1, shared=16384, low=1, high=64),
        # the same in 32 bits, at the sizes of a small model
        dict(name="prefix: 32 bits", op="prefix", dtype="float32", heads=32, kv=32, hd=64, batch=12, groups=2, shared=1024, low=1, high=100),
        # one user's next token behind a short conversation
        dict(name="weighed: one token", op="weighed", dtype="bfloat16", heads=32, kv=32, hd=64, batch=1, run=1, last=0, low=100, high=100),
        # a server's step: eight conversations of up to two thousand positions, one token each
        dict(name="weighed: eight tokens", op="weighed", dtype="bfloat16", heads=32, kv=32, hd=80, batch=8, run=1, last=0, low=300, high=2047),
        # two long documents, one token each
        dict(name="weighed: long", op="weighed", dtype="bfloat16", heads=32, kv=8, hd=128, batch=2, run=1, last=0, low=32000, high=32767),
        # a whole prompt, every token's weights counted
        dict(name="weighed: prompt", op="weighed", dtype="bfloat16", heads=32, kv=32, hd=80, batch=1, run=2048, last=0, low=0, high=0),
        # a step in 32 bits
        dict(name="weighed: 32 bits", op="weighed", dtype="float32", heads=32, kv=32, hd=64, batch=4, run=1, last=0, low=50, high=700),
        # one layer of four conversations cut to half
        dict(name="evict: one layer", op="evict", dtype="bfloat16", heads=32, kv=32, hd=80, batch=4, layers=1, keep=512, recent=128, first=4, low=700, high=1100),
        # every layer of a model at once
        dict(name="evict: all layers", op="evict", dtype="bfloat16", heads=32, kv=32, hd=64, batch=4, layers=24, keep=1024, recent=256, first=4, low=1800, high=2047),
        # long documents cut to an eighth
        dict(name="evict: long", op="evict", dtype="bfloat16", heads=32, kv=8, hd=128, batch=2, layers=4, keep=4096, recent=1024, first=0, low=30000, high=32767),
    ]


#: (query heads, key/value heads, head size): what the listed cases have, and others between
HEADS = [(32, 32, 64), (32, 32, 80), (32, 8, 128), (16, 4, 128), (8, 2, 32), (16, 1, 64), (12, 4, 48), (16, 2, 256), (6, 3, 16)]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most = [(max(w["bytes"] for w in v), max(w["flops"] for w in v))
            for v in ([work(c) for c in listed() if c["op"] == op] for op in ("prefix", "weighed", "evict"))]
    while True:
        n = rng.randrange(3)
        op = ("prefix", "weighed", "evict")[n]
        heads, kv, hd = rng.choice(HEADS)
        dtype = "float32" if rng.random() < 0.25 else "bfloat16"
        c = dict(op=op, dtype=dtype, heads=heads, kv=kv, hd=hd)
        if op == "prefix":
            batch = _spread(rng, 2, 128)
            high = _spread(rng, 1, 700)
            c.update(batch=batch, groups=rng.randint(1, min(4, max(1, batch // 2))), shared=PAGE * _spread(rng, 1, 256),
                     low=rng.randint(1, high), high=high)
        elif op == "weighed":
            long = rng.random() < 0.4
            batch = _spread(rng, 1, 4 if long else 16)
            high = rng.randint(0, 500) if long else _spread(rng, 1, 32767)
            c.update(batch=batch, run=_spread(rng, 2, 2048) if long else 1, last=rng.choice((0, 32)) if long else 0, low=rng.randint(0, high), high=high)
        else:
            high = _spread(rng, 200, 32767)
            keep = rng.randint(64, max(65, high // 2))
            recent = rng.randint(0, keep // 2)
            c.update(batch=_spread(rng, 1, 8), layers=rng.choice((1, 1, 2, 8)), keep=keep, recent=recent, first=min(rng.choice((0, 4)), keep - recent),
                     low=rng.randint(high // 2, high), high=high)
        w = work(c)
        if w["bytes"] <= most[n][0] and w["flops"] <= max(most[n][1], 1):
            return c


def _lengths(c):
    """Positions cached before the call, sequence by sequence (behind the shared ones, for a shared prefix): the case's two ends, and evenly between."""
    n = c["batch"]
    return [c["low"] + (c["high"] - c["low"]) * i // max(1, n - 1) for i in range(n)]


def _groups(c):
    """[(sequences, shared positions)]: the sequences shared out unevenly, each group's prefix shorter than the one before; with two groups or more
    the last sequence belongs to none."""
    n, g = c["batch"] - (1 if c["groups"] > 1 and c["batch"] > 2 * c["groups"] else 0), c["groups"]
    cuts = [n * i * (i + 1) // (g * (g + 1)) for i in range(g + 1)]
    return [(list(range(cuts[i], cuts[i + 1])), max(PAGE, c["shared"] // (i + 1) // PAGE * PAGE)) for i in range(g) if cuts[i + 1] > cuts[i]]


def _runs(c):
    """New tokens, sequence by sequence: the case's longest, and shorter ones beside it."""
    return [max(1, c["run"] * (c["batch"] - i) // c["batch"]) for i in range(c["batch"])]


def _pages(order, counts, at=0):
    """A table with counts[b] pages of ``order`` for sequence b, and the tail of each row on pages of the last one taken."""
    most = max(counts)
    index = torch.zeros(len(counts), most, dtype=torch.int64)
    for b, n in enumerate(counts):
        index[b, :n] = torch.arange(at, at + n)
        at += n
    return order[index], at


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(c)

    def cache(pages, *layers):
        return torch.randn((*layers, pages, c["kv"], PAGE, c["hd"]), generator=g, device="cuda", dtype=dtype)

    def queries(tokens):
        return (torch.randn(tokens, c["heads"] * c["hd"], generator=g, device="cuda") * (2 * c["hd"] ** -0.5)).to(dtype)

    def order(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32).cpu()

    lengths = _lengths(c)
    random.Random(seed).shuffle(lengths)
    if c["op"] == "prefix":
        groups = _groups(c)
        shared = [0] * c["batch"]
        for members, n in groups:
            for b in members:
                shared[b] = n
        mine = [-(-n // PAGE) for n in lengths]
        total = sum(mine) + sum(n // PAGE for _, n in groups)
        ids = order(total)
        table = torch.zeros(c["batch"], max(a + n // PAGE for a, n in zip(mine, shared)), dtype=torch.int32)
        at = 0
        for members, n in groups:
            table[members, :n // PAGE] = ids[at:at + n // PAGE]
            at += n // PAGE
        for b, n in enumerate(mine):
            table[b, shared[b] // PAGE:shared[b] // PAGE + n] = ids[at:at + n]
            at += n
        s.update(k=cache(total), v=cache(total), q=queries(c["batch"]), pages=table.cuda(), ctx=i32([a + n - 1 for a, n in zip(lengths, shared)]))
        if own:
            # made once for a batch of sequences and kept for all of their steps
            from gopherllm_b200 import ops
            s["plan"] = ops.prefix_plan(groups, c["batch"], c["heads"], c["kv"], c["hd"], dtype, max(lengths), "cuda")
    elif c["op"] == "weighed":
        runs = _runs(c)
        most = -(-max(a + n for a, n in zip(lengths, runs)) // PAGE)      # a page table as reserved: every sequence may grow to the longest
        ids = order(c["batch"] * most)
        s.update(k=cache(ids.numel()), v=cache(ids.numel()), q=queries(sum(runs)), pages=ids.view(c["batch"], most).cuda(),
                 ctx=i32(lengths), qlen=i32(runs), qstart=i32([sum(runs[:b]) for b in range(c["batch"])]),
                 rows=sum(runs), longest=max(runs), reach=max(a + n for a, n in zip(lengths, runs)),
                 sums=torch.rand(ids.numel(), c["kv"], PAGE, generator=g, device="cuda") * 0.05)
    else:
        most = -(-max(lengths) // PAGE)
        fresh = -(-c["keep"] // PAGE)
        ids = order(c["batch"] * (most + fresh))
        s.update(k=cache(ids.numel(), c["layers"]), v=cache(ids.numel(), c["layers"]), pages=ids[:c["batch"] * most].view(c["batch"], most).cuda(),
                 to=ids[c["batch"] * most:].view(c["batch"], fresh).cuda(), length=i32(lengths),
                 # a few positions carry most of the weight
                 sums=torch.rand(c["layers"], ids.numel(), c["kv"], PAGE, generator=g, device="cuda").pow(8) * 100)
    return s


def run(state):
    if own:
        return _own(state)
    return {"prefix": _plain_prefix, "weighed": _plain_weighed, "evict": _plain_evict}[state["op"]](state)


def _own(s):
    from gopherllm_b200 import ops
    if s["op"] == "prefix":
        out = torch.empty_like(s["q"])
        ops.attention_prefix(s["q"], out, s["k"], s["v"], s["ctx"], s["pages"], s["plan"], s["heads"], s["kv"], s["hd"])
        return out
    if s["op"] == "weighed":
        out = torch.empty_like(s["q"])
        ops.attention_weighed(s["q"], out, s["k"], s["v"], s["sums"], s["qstart"], s["qlen"], s["ctx"], s["pages"], s["heads"], s["kv"], s["hd"],
                              max_qlen=s["longest"], max_len=s["reach"], last=s["last"])
        return out, s["sums"]
    kept = ops.cache_evict(s["k"], s["v"], s["sums"], s["length"], s["pages"], s["keep"], recent=s["recent"], first=s["first"], to_pages=s["to"])
    return kept, s["k"], s["v"], s["sums"]


# -- the plain forms ----------------------------------------------------------
def _plain_prefix(s):
    B, H, G, D = s["batch"], s["heads"], s["kv"], s["hd"]
    rows = s["pages"].long()
    k, v = (t[rows].transpose(2, 3).reshape(B, -1, G, D).float() for t in (s["k"], s["v"]))
    q = s["q"].float().view(B, G, H // G, D)
    score = torch.matmul(q, k.permute(0, 2, 3, 1))                                       # [B, G, H / G, positions]
    seen = torch.arange(k.shape[1], device=q.device) <= s["ctx"][:, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, v.transpose(1, 2)).reshape(B, H * D).to(s["q"].dtype)


def _plain_weighed(s):
    B, H, G, D, T = s["batch"], s["heads"], s["kv"], s["hd"], s["longest"]
    rows = s["pages"].long()
    k, v = (t[rows].transpose(2, 3).reshape(B, -1, G, D).float() for t in (s["k"], s["v"]))
    L = k.shape[1]
    step = torch.arange(T, device=k.device)
    real = step < s["qlen"][:, None]                                                      # [B, T]
    place = torch.where(real, s["qstart"][:, None] + step, 0)
    q = s["q"].float()[place].view(B, T, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * T, D)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).view(B, G, H // G, T, L)
    at = torch.arange(L, device=k.device)
    seen = at <= (s["ctx"][:, None] + step)[..., None]                                    # [B, T, L]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, G, -1, L), v.transpose(1, 2)).view(B, G, H // G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H * D)
    put = torch.arange(s["rows"], device=k.device)
    seq = (put[:, None] >= s["qstart"]).sum(-1) - 1
    out = o[seq, put - s["qstart"][seq]].to(s["q"].dtype)
    counted = real & (step >= s["qlen"][:, None] - s["last"]) if s["last"] else real
    given = (p * counted[:, None, None, :, None]).sum((2, 3))                             # [B, G, L]
    had = s["sums"][rows].transpose(1, 2).reshape(B, G, L)
    old, new = at < s["ctx"][:, None], at < (s["ctx"] + s["qlen"])[:, None]
    now = torch.where(new[:, None], torch.where(old[:, None], had, 0.0) + given, had)
    s["sums"][rows] = now.view(B, G, -1, PAGE).transpose(1, 2)
    return out, s["sums"]


def _plain_evict(s):
    N, B, G, D, keep = s["layers"], s["batch"], s["kv"], s["hd"], s["keep"]
    rows, to = s["pages"].long(), s["to"].long()
    sums = s["sums"][:, rows].transpose(2, 3).reshape(N, B, G, -1)
    at = torch.arange(sums.shape[-1], device=sums.device)
    n = s["length"][:, None].long()
    always = (at < s["first"]) | (at >= n - s["recent"])
    rank = torch.where(always[:, None], math.inf, sums)
    rank = torch.where((at < n)[:, None], rank, -math.inf)
    top = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    pad = keep - top.shape[-1]
    if pad > 0:
        top = torch.cat([top, top[..., :1].expand(N, B, G, pad)], -1)
    left = torch.arange(keep, device=at.device) < n                                       # [B, keep]
    kept = torch.sort(torch.where(left[:, None], top, at.numel()), dim=-1).values
    kept = torch.where(left[:, None], kept, -1)
    src = kept.clamp(min=0)
    layer, head = torch.arange(N, device=at.device)[:, None, None, None], torch.arange(G, device=at.device)[:, None]
    page = rows[torch.arange(B, device=at.device)[:, None, None], src // PAGE]            # [N, B, G, keep]
    slot = torch.arange(keep, device=at.device)
    goes = to[:, None, slot // PAGE]                                                      # [B, 1, keep]
    for name in ("k", "v", "sums"):
        t = s[name]
        moved = t[layer, page, head, src % PAGE]
        stays = t[layer, goes, head, slot % PAGE]
        mask = left[:, None] if name == "sums" else left[:, None, :, None]
        t[layer, goes, head, slot % PAGE] = torch.where(mask, moved, stays)
    return kept.to(torch.int32), s["k"], s["v"], s["sums"]


# -- the definitions in 64 bits ----------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    H, G, D, B = s["heads"], s["kv"], s["hd"], s["batch"]
    ctx = (s["length"] if s["op"] == "evict" else s["ctx"]).tolist()
    if s["op"] == "prefix":
        out = torch.empty(B, H, D, dtype=torch.float64, device="cuda")
        for b in range(B):
            k, v = (_rows64(t, s["pages"][b], ctx[b] + 1).repeat_interleave(H // G, 1) for t in (s["k"], s["v"]))
            p = torch.softmax(torch.einsum("hd,jhd->hj", s["q"][b].double().view(H, D), k), -1)
            out[b] = torch.einsum("hj,jhd->hd", p, v)
        return out.view(B, H * D)
    if s["op"] == "weighed":
        out, sums = torch.empty(s["rows"], H, D, dtype=torch.float64, device="cuda"), s["sums"].double()
        start, runs = s["qstart"].tolist(), s["qlen"].tolist()
        for b in range(B):
            n = ctx[b] + runs[b]
            q = s["q"][start[b]:start[b] + runs[b]].double().view(runs[b], H, D)
            page, slot = s["pages"][b].long()[torch.arange(n, device="cuda") // PAGE], torch.arange(n, device="cuda") % PAGE
            k, v = _rows64(s["k"], s["pages"][b], n), _rows64(s["v"], s["pages"][b], n)
            late = torch.arange(n, device="cuda") > torch.arange(ctx[b], n, device="cuda")[:, None]
            for h in range(H):
                score = q[:, h] @ k[:, h * G // H].T
                p = torch.softmax(score.masked_fill(late, -math.inf), -1)
                out[start[b]:start[b] + runs[b], h] = p @ v[:, h * G // H]
                if h % (H // G) == 0:
                    sums[page[ctx[b]:], h * G // H, slot[ctx[b]:]] = 0.0
                sums[page, h * G // H, slot] += (p[-s["last"]:] if s["last"] else p).sum(0)
        return out.view(-1, H * D), sums
    k, v, sums = s["k"].double(), s["v"].double(), s["sums"].double()
    kept = torch.full((s["layers"], B, G, s["keep"]), -1, dtype=torch.int32, device="cuda")
    for b in range(B):
        n, m = ctx[b], min(ctx[b], s["keep"])
        page, slot = s["pages"][b].long()[torch.arange(n, device="cuda") // PAGE], torch.arange(n, device="cuda") % PAGE
        goes = s["to"][b].long()[torch.arange(m, device="cuda") // PAGE]
        for layer in range(s["layers"]):
            for g in range(G):
                if n <= s["keep"]:
                    chosen = torch.arange(n, device="cuda")
                else:
                    first, recent = s["first"], n - s["recent"]
                    between = sums[layer, page, g, slot][first:recent]
                    best = torch.argsort(-between, stable=True)[:m - first - s["recent"]] + first
                    chosen = torch.cat([torch.arange(first, device="cuda"), best.sort().values, torch.arange(recent, n, device="cuda")])
                kept[layer, b, g, :m] = chosen
                for t in (k, v, sums):
                    t[layer, goes, g, torch.arange(m, device="cuda") % PAGE] = t[layer, page[chosen], g, slot[chosen]]
    return kept, k, v, sums


def _rows64(cache, pages, n):
    """The first n positions of one sequence, [n, heads, head size] in 64 bits."""
    return cache[pages[:-(-n // PAGE)].long()].double().transpose(1, 2).reshape(-1, *cache.shape[1::2])[:n]


# -- what a pass cannot do without ----------------------------------------------------
def work(case):
    c = case
    size = 2 if c["dtype"] == "bfloat16" else 4
    row = c["kv"] * c["hd"] * size                            # a position's keys, or its values
    lengths = _lengths(c)
    if c["op"] == "prefix":
        groups = _groups(c)
        shared = {b: n for members, n in groups for b in members}
        read = sum(lengths) + sum(n for _, n in groups)
        pairs = sum(lengths) + sum(shared.values())
        return {"bytes": 2 * row * read + 2 * c["batch"] * c["heads"] * c["hd"] * size, "flops": 4 * c["heads"] * c["hd"] * pairs}
    if c["op"] == "weighed":
        runs = _runs(c)
        after = sum(a + n for a, n in zip(lengths, runs))
        pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(lengths, runs))
        return {"bytes": 2 * row * after + 4 * c["kv"] * (after + sum(lengths)) + 2 * sum(runs) * c["heads"] * c["hd"] * size,
                "flops": 4 * c["heads"] * c["hd"] * pairs}
    stays = sum(min(n, c["keep"]) for n in lengths)
    return {"bytes": c["layers"] * (4 * row * stays + 4 * c["kv"] * (sum(lengths) + 2 * stays)), "flops": 0}
