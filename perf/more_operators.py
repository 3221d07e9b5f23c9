"""Cases for windowed attention, drafted trees and sampling, each with a plain form in elementary torch operations.

Four operators:

* ``window``  attention over the paged cache with a sliding window and a few first tokens that stay visible
  (``megaqwen_b200.paged.window_attend``);
* ``tree``    attention of a tree of drafted tokens over the paged cache (``paged.tree_attend``);
* ``accept``  room for a drafted tree, the walk along the tokens that were chosen at its nodes, and the cache cut down to
  the accepted path (``paged.reserve``, ``paged.accept``);
* ``sample``  a token for each row of logits by temperature, top-k, top-p and min-p from given random numbers
  (``megaqwen_b200.sampling.sample``).

Where ``own`` is false, ``run`` computes them in their plain form: attention in 32 bits, sampling in 64 (its sums are long
and its choices are borders between them); where it is true it calls the package.  Lengths are functions of the case alone,
so ``work`` is exact; page numbers, trees and values come from the seed.
"""
from types import SimpleNamespace

import math

import numpy as np
import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    qwen = {"hq": 16, "hkv": 8, "d": 128, "dtype": "bf16"}
    return [
        # one conversation far past its window, one token: latency
        {"name": "window_decode_1", "op": "window", **qwen, "page": 64, "seqs": 1, "q_len": 1, "ctx": 20001, "window": 1024,
         "sinks": 4},
        # a decode batch of long conversations
        {"name": "window_decode_64", "op": "window", **qwen, "page": 64, "seqs": 64, "q_len": 1, "ctx": 12000,
         "window": 4096, "sinks": 16},
        # prompts prefilled from their first token, twice as long as the window
        {"name": "window_prompts_8x2000", "op": "window", **{**qwen, "dtype": "fp16"}, "page": 64, "seqs": 8, "q_len": 2000,
         "ctx": 2000, "window": 1024, "sinks": 4},
        # a piece of a long prompt on what came before it, small pages, odd sizes
        {"name": "window_piece_3001", "op": "window", **qwen, "page": 16, "seqs": 1, "q_len": 3001, "ctx": 16411,
         "window": 2000, "sinks": 128},
        # one conversation with a small tree: latency
        {"name": "tree_1x16", "op": "tree", **qwen, "page": 64, "seqs": 1, "nodes": 16, "ctx": 1000},
        # a batch of a chat server, uneven contexts
        {"name": "tree_16x31", "op": "tree", **{**qwen, "dtype": "fp16"}, "page": 16, "seqs": 16, "nodes": 31, "ctx": 6000},
        # wide trees on long contexts
        {"name": "tree_32x64", "op": "tree", **qwen, "page": 64, "seqs": 32, "nodes": 64, "ctx": 8192},
        # two conversations accept a few tokens of a small model's cache: latency
        {"name": "accept_2x8", "op": "accept", **qwen, "page": 16, "layers": 2, "seqs": 2, "nodes": 8, "ctx": 90, "depth": 3},
        # a batch, all layers
        {"name": "accept_32x64", "op": "accept", **qwen, "page": 16, "layers": 28, "seqs": 32, "nodes": 64, "ctx": 40,
         "depth": 8},
        # one conversation's next token: latency
        {"name": "sample_1", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "fp32", "rule": "all"},
        # a batch of requests, each with parameters of its own, a few of them constrained to a grammar's tokens
        {"name": "sample_64_mixed", "op": "sample", "rows": 64, "vocab": 151936, "dtype": "fp32", "rule": "mixed"},
        # the nodes of a batch of trees, logits in 16 bits (many equal ones)
        {"name": "sample_256_nucleus", "op": "sample", "rows": 256, "vocab": 151936, "dtype": "bf16", "rule": "top_p"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(["window", "window", "tree", "tree", "accept", "sample", "sample"])
    c = {"op": op}
    if op == "sample":
        c["vocab"] = rng.choice([151936, 151936, log(100, 262144), log(1000, 151936)])
        c["rows"] = log(1, min(256, 256 * 151936 // c["vocab"]))
        c["dtype"] = rng.choice(["fp32", "fp32", "bf16", "fp16"])
        if c["dtype"] == "fp32":
            c["rows"] = min(c["rows"], 128)
        c["rule"] = rng.choice(["all", "mixed", "mixed", "top_p", "top_k", "min_p", "plain"])
        return c
    hkv, g = rng.choice([(8, 2), (8, 2), (8, 4), (4, 7), (2, 5), (1, 8), (8, 1), (4, 8)])
    c.update(hq=hkv * g, hkv=hkv, d=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
             page=rng.choice([16, 32, 64, 128]))
    wide = max(1.0, c["hq"] * c["d"] / 2048)   # relative width of a token
    if op == "window":
        c["seqs"] = log(1, 64)
        c["window"] = log(16, 4096)
        c["sinks"] = rng.choice([0, 4, 4, log(1, 128)])
        most = 8 * 2000 * 1024 / wide          # (query, key) pairs of a head
        if rng.random() < 0.5:
            c["q_len"] = rng.choice([1, 1, 2, 5])
            c["ctx"] = c["q_len"] + log(1, 16000)
        else:
            c["q_len"] = log(8, min(4000, most / (c["seqs"] * c["window"]) + 8))
            c["ctx"] = c["q_len"] + rng.choice([0, log(1, 16000)])
        while c["seqs"] > 1 and c["seqs"] * (c["ctx"] + c["q_len"]) * c["hkv"] * c["d"] > 64 * 12000 * 1024:
            c["seqs"] //= 2
    elif op == "tree":
        c["nodes"] = rng.choice([1, log(2, 64), log(4, 64), log(16, 200)])
        c["ctx"] = log(1, 16000)
        most = 32 * 64 * 8192 / wide
        c["seqs"] = log(1, min(64, most / (c["nodes"] * c["ctx"]) + 1))
        while c["seqs"] > 1 and c["seqs"] * c["ctx"] * c["hkv"] * c["d"] > 32 * 8192 * 1024:
            c["seqs"] //= 2
    else:
        c["layers"] = log(1, 28)
        c["seqs"] = log(1, 32)
        c["nodes"] = log(1, 64)
        c["ctx"] = log(1, 300)
        c["depth"] = rng.randint(1, 8)
        while c["seqs"] * (c["ctx"] + c["nodes"] + 2 * c["page"]) * c["layers"] * c["hkv"] * c["d"] > 32 * 136 * 28 * 1024:
            if c["seqs"] > 1:
                c["seqs"] //= 2
            else:
                c["layers"] = max(1, c["layers"] // 2)
    return c


# ------------------------------------------------------------------------------------------------------------------
# sizes that follow from a case

def _ceil(a, b):
    return -(-a // b)


def _sizes(c):
    """(query tokens, positions in the cache with them) of each sequence."""
    out = []
    for b in range(c["seqs"]):
        if c["op"] == "window":
            n = max(1, c["q_len"] - (c["q_len"] * (b * 19 % 23)) // 92)      # the longest three quarters, ragged
            before = c["ctx"] - c["q_len"]
            out.append((n, n + before - (before * (b * 37 % 41)) // 82))     # of ctx, the upper half
        else:
            n = max(1, c["nodes"] - (c["nodes"] * (b * 11 % 13)) // 26)
            out.append((n, n + c["ctx"] - (c["ctx"] * (b * 29 % 61)) // 122))
    return out


def _depth(nodes, depth):
    """Most nodes that a walk accepts: the ones behind the root are chosen among the nodes from there on."""
    return max(1, min(depth, nodes // 2))


# ------------------------------------------------------------------------------------------------------------------
# inputs

def _ints(v):
    return torch.as_tensor(v, dtype=torch.int32).to(DEV)


def _normal(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    x.normal_(0.0, scale, generator=g)
    return x


def _tree(gc, n):
    """Parents of a tree of n nodes, the root first, each node on one of the twelve before it."""
    if n == 1:
        return [-1]
    r = torch.rand(n, generator=gc).tolist()
    return [-1] + [max(0, i - 12) + int(r[i] * min(i, 12)) for i in range(1, n)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    gc = torch.Generator().manual_seed(int(seed))
    dt = TYPES[c["dtype"]]
    s = SimpleNamespace(c=dict(c))
    if c["op"] == "sample":
        n, v = c["rows"], c["vocab"]
        # a language model's logits: a broad middle, a few dozen candidates that stand out
        x = _normal(g, (n, v), torch.float32, 2.0)
        some = min(v, 60)
        at = torch.randint(0, v, (n, some), generator=g, device=DEV)
        x.scatter_add_(1, at, torch.empty(n, some, device=DEV).exponential_(0.25, generator=g))
        if c["rule"] == "mixed":   # rows of constrained requests: all but a few tokens are ruled out
            for r in range(3, n, 8):
                keep = x[r, at[r, :5]].clone()
                x[r] = -math.inf
                x[r, at[r, :5]] = keep
        s.logits = x.to(dt)
        s.u = torch.rand(n, generator=g, device=DEV)
        s.temperature, s.top_k, s.top_p, s.min_p = {
            "plain": (1.0, 0, 1.0, 0.0), "all": (0.7, 50, 0.95, 0.02), "top_k": (0.8, 40, 1.0, 0.0),
            "top_p": (1.0, 0, 0.9, 0.0), "min_p": (1.2, 0, 1.0, 0.05), "mixed": (None,) * 4}[c["rule"]]
        if c["rule"] == "mixed":
            def among(values, dtype):
                return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (n,), generator=gc)].to(DEV)
            s.temperature = among([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32)
            s.top_k = among([0, 0, 1, 20, 50, 1000], torch.int32)
            s.top_p = among([0.5, 0.9, 0.95, 1.0], torch.float32)
            s.min_p = among([0.0, 0.0, 0.02, 0.1], torch.float32)
        return s
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    sizes = _sizes(c)
    s.page, s.scale = page, 1.0 / math.sqrt(d)
    if c["op"] == "accept":
        s.layers = c["layers"]
        have = [_ceil(t - n, page) for n, t in sizes]
        pages = sum(_ceil(t, page) for _, t in sizes) + 3
    else:
        s.layers = 1
        have = [_ceil(t, page) for _, t in sizes]
        pages = sum(have) + 2
    cols = max(_ceil(t, page) for _, t in sizes) + 1
    perm = torch.randperm(pages, generator=gc).int()
    order = torch.randperm(c["seqs"] + 1, generator=gc)[:c["seqs"]]
    table = torch.full((c["seqs"] + 1, cols), -1, dtype=torch.int32)
    lengths = torch.zeros(c["seqs"] + 1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for b, k in enumerate(have):
        table[order[b], :k] = perm[at:at + k]
        refs[perm[at:at + k].long()] = 1
        lengths[order[b]] = sizes[b][1] - (sizes[b][0] if c["op"] == "accept" else 0)
        at += k
    s.table, s.lengths, s.refs, s.slots = table.to(DEV), lengths.to(DEV), refs.to(DEV), order.int().to(DEV)
    s.k = _normal(g, (pages, s.layers, hkv, page, d), dt)
    s.v = _normal(g, (pages, s.layers, hkv, page, d), dt)
    starts = [0]
    for n, _ in sizes:
        starts.append(starts[-1] + n)
    s.q_starts = None if c["op"] == "window" and c["q_len"] == 1 else _ints(starts)
    if c["op"] != "accept":
        s.q = _normal(g, (starts[-1], hq, d), dt, 2.0)   # scores of standard deviation 2
    if c["op"] != "window":
        trees = [_tree(gc, n) for n, _ in sizes]
        s.parents = _ints(sum(trees, []))
    if c["op"] == "accept":
        # tokens drafted and chosen: the walk takes a child that lies behind the places the accepted rows move to, or one
        # that is in its place, so that another pass over the same pages finds its rows where this one did
        s.tokens = torch.randint(0, 50000, (starts[-1],), generator=gc).int()
        s.chosen = torch.randint(50000, 100000, (starts[-1],), generator=gc).int()
        for b, tree in enumerate(trees):
            most, at = _depth(len(tree), c["depth"]), 0
            for step in range(1, most):
                kids = [i for i in range(1, len(tree)) if tree[i] == at and (i >= most or i == step)]
                if not kids:
                    break
                s.chosen[starts[b] + at] = s.tokens[starts[b] + kids[-1]]
                at = kids[-1]
        s.tokens, s.chosen = s.tokens.to(DEV), s.chosen.to(DEV)
        s.grown = _ints([t for _, t in sizes])
    return s


# ------------------------------------------------------------------------------------------------------------------
# the plain forms

def _attention(q, k, v, seen, scale):
    """q [n, hkv, grp, d], k and v [hkv, l, d] in 32 bits, seen [n, l]; rows that see nothing are zero."""
    score = torch.einsum("nhgd,hld->hgnl", q, k) * scale
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    out = torch.einsum("hgnl,hld->nhgd", w, v)
    total = w.sum(-1).permute(2, 0, 1)[..., None]
    return torch.where(total > 0, out / total, 0.0)


def _gather(pages, ids, lo, hi):
    """Positions lo .. hi - 1 of a sequence whose pages are ids: [hkv, positions, d] in 32 bits."""
    page = pages.shape[3]
    p0, p1 = lo // page, _ceil(hi, page)
    x = pages[ids[p0:p1].long(), 0].transpose(0, 1).flatten(1, 2)
    return x[:, lo - p0 * page:hi - p0 * page].float()


def _plain_window(s):
    c = s.c
    hkv, grp, d = c["hkv"], c["hq"] // c["hkv"], c["d"]
    out = torch.empty_like(s.q)
    r0 = 0
    for b, (n, t) in enumerate(_sizes(c)):
        ids = s.table[s.slots[b].long()]
        for i in range(0, n, 512):
            m = min(512, n - i)
            first, last = t - n + i, t - n + i + m - 1
            lo = max(0, first - c["window"] + 1)
            head = min(c["sinks"], lo)
            k = torch.cat([_gather(s.k, ids, 0, head), _gather(s.k, ids, lo, last + 1)], 1) if head else _gather(s.k, ids, lo, last + 1)
            v = torch.cat([_gather(s.v, ids, 0, head), _gather(s.v, ids, lo, last + 1)], 1) if head else _gather(s.v, ids, lo, last + 1)
            key = torch.cat([torch.arange(head, device=DEV), torch.arange(lo, last + 1, device=DEV)])
            pos = torch.arange(first, last + 1, device=DEV)[:, None]
            seen = (key <= pos) & ((key < c["sinks"]) | (key > pos - c["window"]))
            q = s.q[r0 + i:r0 + i + m].float().view(m, hkv, grp, d)
            out[r0 + i:r0 + i + m] = _attention(q, k, v, seen, s.scale).reshape(m, hkv * grp, d).to(out.dtype)
        r0 += n
    return out


def _plain_tree(s):
    c = s.c
    hkv, grp, d = c["hkv"], c["hq"] // c["hkv"], c["d"]
    out = torch.empty_like(s.q)
    r0 = 0
    for b, (n, t) in enumerate(_sizes(c)):
        ids = s.table[s.slots[b].long()]
        parent = s.parents[r0:r0 + n].long()
        node = torch.arange(n, device=DEV)
        seen = torch.zeros(n, n + 1, dtype=torch.bool, device=DEV)   # the last column takes the roots' parent
        at = node.clone()
        for _ in range(n):
            seen[node, at] = True
            at = torch.where(at < n, parent[at.clamp(max=n - 1)], n)
            at = torch.where(at < 0, n, at)
        seen = torch.cat([torch.ones(n, t - n, dtype=torch.bool, device=DEV), seen[:, :n]], 1)
        q = s.q[r0:r0 + n].float().view(n, hkv, grp, d)
        o = _attention(q, _gather(s.k, ids, 0, t), _gather(s.v, ids, 0, t), seen, s.scale)
        out[r0:r0 + n] = o.reshape(n, hkv * grp, d).to(out.dtype)
        r0 += n
    return out


def _plain_accept(s):
    c, page, dev = s.c, s.page, s.k.device
    sizes = _sizes(c)
    n_seq, width = len(sizes), max(n for n, _ in sizes)
    slots = s.slots.long()
    pages, cols = s.k.shape[0], s.table.shape[1]
    col = torch.arange(cols, device=dev)
    # room for the trees: the lowest free pages, in the order of the sequences
    have = (s.lengths[slots] + page - 1) // page
    want = (s.grown + page - 1) // page
    free = torch.argsort(s.refs > 0, stable=True)                     # the free ones first, lowest first
    new = (col >= have[:, None]) & (col < want[:, None])
    rank = torch.cumsum(new.flatten(), 0).view(n_seq, cols) - 1
    rows = torch.where(new, free[rank.clamp(min=0, max=pages - 1)].int(), s.table[slots])
    s.table[slots] = rows
    s.refs.index_add_(0, torch.where(new, rows, 0).flatten().long(), new.flatten().int())
    # the walks, all sequences side by side
    n = torch.tensor([n for n, _ in sizes], device=dev)
    at = torch.cumsum(n, 0) - n
    node = torch.arange(width, device=dev)
    inside = node < n[:, None]
    flat = torch.where(inside, at[:, None] + node, 0)
    parents = torch.where(inside, s.parents[flat], -2).long()
    tokens, chosen = s.tokens[flat], s.chosen[flat]
    path = torch.full((n_seq, width), -1, dtype=torch.long, device=dev)
    here, alive = torch.zeros(n_seq, dtype=torch.long, device=dev), torch.ones(n_seq, dtype=torch.bool, device=dev)
    path[:, 0] = 0
    for i in range(1, width):
        hit = (parents == here[:, None]) & (tokens == chosen.gather(1, here[:, None])) & (node > 0)
        child = torch.where(hit, node, width).amin(1)
        alive = alive & (child < width)
        here = torch.where(alive, child, here)
        path[:, i] = torch.where(alive, here, -1)
    count = (path >= 0).sum(1)
    # accepted rows to their places (the others onto themselves)
    base = s.grown - n.int()
    src = base[:, None] + torch.where(path >= 0, path, torch.where(inside, node, 0))
    dst = base[:, None] + torch.where(inside, node, 0)
    sp, dp = rows.gather(1, (src // page).long()).long(), rows.gather(1, (dst // page).long()).long()
    for x in (s.k, s.v):
        x[dp, :, :, (dst % page).long()] = x[sp, :, :, (src % page).long()]
    # the sequences end behind the accepted ones; pages past that are free again
    length = base + count.int()
    gone = (col >= ((length + page - 1) // page)[:, None]) & (col < want[:, None])
    s.refs.index_add_(0, torch.where(gone, rows, 0).flatten().long(), -gone.flatten().int())
    s.table[slots] = torch.where(gone, -1, rows)
    s.lengths[slots] = length
    emitted = torch.where(path >= 0, chosen.gather(1, path.clamp(min=0)), -1)
    return _accept_outputs(s, path[inside].int(), emitted[inside].int(), count.int())


def _accept_outputs(s, path, emitted, count):
    return {"path": path, "emitted": emitted, "count": count, "table": s.table, "lengths": s.lengths, "refs": s.refs,
            "k_pages": s.k, "v_pages": s.v}


def _per_row(x, n, dtype):
    return (x.to(dtype) if torch.is_tensor(x) else torch.full((n,), x, dtype=torch.float32, device=DEV).to(dtype))[:, None]


def _plain_sample(s):
    n, v = s.logits.shape
    t, p, lowest = (_per_row(x, n, torch.float64) for x in (s.temperature, s.top_p, s.min_p))
    k, u = _per_row(s.top_k, n, torch.int64), s.u.double()[:, None]
    out = torch.empty(n, dtype=torch.int32, device=DEV)
    for r in range(0, n, 64):
        some = slice(r, r + 64)
        x, at = torch.sort(s.logits[some].double(), dim=-1, descending=True, stable=True)
        w = torch.exp((x - x[:, :1]) / torch.where(t[some] > 0, t[some], 1.0))
        rank = torch.arange(v, device=DEV)
        w = torch.where((k[some] > 0) & (rank >= k[some]), 0.0, w)
        before = torch.cumsum(w, -1) - w
        keep = (p[some] >= 1) | (before < p[some] * w.sum(-1, keepdim=True)) | (rank == 0)
        w = torch.where(keep & (w >= lowest[some]), w, 0.0)
        w = torch.zeros_like(w).scatter_(1, at, w)                    # in the order of the tokens
        sums = torch.cumsum(w, -1)
        pick = (sums <= u[some] * sums[:, -1:]).sum(-1)
        out[some] = torch.where(t[some, 0] > 0, pick, at[:, 0]).int()
    return out


def run(s):
    c = s.c
    if not own:
        return {"window": _plain_window, "tree": _plain_tree, "accept": _plain_accept, "sample": _plain_sample}[c["op"]](s)
    from megaqwen_b200 import paged, sampling
    if c["op"] == "window":
        return paged.window_attend(s.q, s.k, s.v, s.table, s.lengths, s.slots, layer=0, window=c["window"],
                                   sinks=c["sinks"], q_starts=s.q_starts, scale=s.scale)
    if c["op"] == "tree":
        return paged.tree_attend(s.q, s.k, s.v, s.table, s.lengths, s.slots, s.parents, layer=0, q_starts=s.q_starts,
                                 scale=s.scale)
    if c["op"] == "accept":
        paged.reserve(s.table, s.lengths, s.refs, s.slots, s.grown, s.page)
        return _accept_outputs(s, *paged.accept(s.k, s.v, s.table, s.lengths, s.refs, s.slots, s.parents, s.tokens,
                                                s.chosen, q_starts=s.q_starts))
    return sampling.sample(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    c = case
    if c["op"] == "sample":
        n, v = c["rows"], c["vocab"]
        return {"bytes": n * (v * (4 if c["dtype"] == "fp32" else 2) + 8), "flops": 4 * n * v}   # scale, exp, sum, compare
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    row = 2 * hkv * d * 2                       # bytes of one position's keys and values in one layer
    sizes = _sizes(c)
    if c["op"] == "accept":
        moved = sum(_depth(n, c["depth"]) - 1 for n, _ in sizes)   # the root stays where it is
        return {"bytes": moved * 2 * row * c["layers"] + sum(n for n, _ in sizes) * 5 * 4 + len(sizes) * 16, "flops": 0}
    pairs = keys = 0
    for n, t in sizes:
        if c["op"] == "tree":
            keys += t
            pairs += n * (t - n) + n            # at least itself
            continue
        w, sinks = c["window"], c["sinks"]
        lo = max(0, t - n - w + 1)
        keys += t - lo + min(sinks, lo)
        for p in range(t - n, t):
            first = max(0, p - w + 1)
            pairs += p - first + 1 + min(sinks, first)
    tokens = sum(n for n, _ in sizes)
    return {"bytes": keys * row + tokens * hq * d * 2 * 2 + keys // page * 4, "flops": pairs * hq * d * 4}


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits

def _sample64(x, u, t, k, p, lowest):
    """One row, numpy in 64 bits."""
    best = int(np.argmax(x))
    if t <= 0:
        return best
    w = np.exp((x - x[best]) / t)
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        acc = np.cumsum(w[order])
        order = order[:1 + int(np.searchsorted(acc, p * acc[-1], side="left"))]
    keep = np.sort(order[w[order] >= lowest])
    acc = np.cumsum(w[keep])
    return int(keep[min(int(np.searchsorted(acc, u * acc[-1], side="right")), len(keep) - 1)])


def exact(case, seed):
    c = case
    if c["op"] == "accept":
        return None   # copies and whole numbers only
    s = prepare(case, seed)
    if c["op"] == "sample":
        n = c["rows"]

        def each(x):
            return x.cpu().double().tolist() if torch.is_tensor(x) else [float(np.float32(x))] * n

        t, k, p, lowest, u = (each(x) for x in (s.temperature, s.top_k, s.top_p, s.min_p, s.u))
        got = [_sample64(s.logits[i].double().cpu().numpy(), u[i], t[i], int(k[i]), p[i], lowest[i]) for i in range(n)]
        return torch.tensor(got, dtype=torch.int32, device=DEV)
    out = torch.empty(s.q.shape, dtype=torch.float64, device=DEV)
    grp, r0 = c["hq"] // c["hkv"], 0
    parents = s.parents.tolist() if c["op"] == "tree" else None
    for b, (n, t) in enumerate(_sizes(c)):
        ids = s.table[s.slots[b].long(), :_ceil(t, c["page"])].long()
        k, v = (x[ids, 0].permute(0, 2, 1, 3).reshape(-1, c["hkv"], c["d"])[:t].double() for x in (s.k, s.v))
        base = t - n
        if parents:
            seen = torch.zeros(n, t, dtype=torch.bool)
            seen[:, :base] = True
            for i in range(n):
                if parents[r0 + i] >= 0:
                    seen[i, base:] = seen[parents[r0 + i], base:]
                seen[i, base + i] = True
            seen = seen.to(DEV)
        for h in range(c["hq"]):
            for i in range(0, n, 1000):
                m = min(1000, n - i)
                if parents:
                    view = seen[i:i + m]
                else:
                    gap = torch.arange(base + i, base + i + m, device=DEV)[:, None] - torch.arange(t, device=DEV)
                    view = (gap >= 0) & ((gap < c["window"]) | (torch.arange(t, device=DEV) < c["sinks"]))
                z = (s.q[r0 + i:r0 + i + m, h].double() @ k[:, h // grp].T) * s.scale
                z = torch.softmax(z.masked_fill(~view, -math.inf), -1)
                out[r0 + i:r0 + i + m, h] = z @ v[:, h // grp]
        r0 += n
    return out
