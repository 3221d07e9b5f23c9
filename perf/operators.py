"""Cases for the operators of the paged KV cache, each with a plain form in elementary torch operations.

Four operators, reached through ``megaqwen_b200.paged``:

* ``rope``    rotary positions fused with the write of K and V into the pages (and of the pages' score index);
* ``fork``    sequences released, forked from a common prompt and grown again; ``compact`` a pool gathered into another;
* ``shared``  attention of a batch whose sequences share a long prefix, the prefix read once per group;
* ``sparse``  attention over the pages that a cheap score selects for each query token.

Where ``own`` is false, ``run`` computes them in their plain form, in 32 bits; where it is true it calls the package.
Lengths are functions of the case alone, so ``work`` is exact; page numbers and values come from the seed.
"""
from types import SimpleNamespace

import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PAD = 16   # bytes of an index record after its two bounds: the exponent and padding


def listed():
    qwen = {"hq": 16, "hkv": 8, "d": 128, "dtype": "bf16"}
    return [
        # one decode step of a few conversations: latency
        {"name": "rope_decode_8", "op": "rope", **qwen, "seqs": 8, "q_len": 1, "ctx": 2048, "page": 16, "rot": 128,
         "interleaved": False, "yarn": 1.0, "index": False},
        # a prefill of eight long prompts under a scaled table, with the index kept for sparse attention
        {"name": "rope_prefill_8x4001", "op": "rope", **qwen, "seqs": 8, "q_len": 4001, "ctx": 64, "page": 64,
         "rot": 64, "interleaved": True, "yarn": 4.0, "index": True},
        # a beam search's step on a small pool: latency
        {"name": "fork_beams_6", "op": "fork", **qwen, "layers": 2, "pages": 256, "page": 16, "parents": 2,
         "children": 6, "length": 203, "grow": 1},
        # one prompt forked into 64 samples over all 28 layers
        {"name": "fork_samples_64", "op": "fork", **qwen, "layers": 28, "pages": 256, "page": 64, "parents": 1,
         "children": 64, "length": 2088, "grow": 65},
        # a pool at 60 % gathered into a smaller one
        {"name": "compact_28_layers", "op": "compact", **qwen, "layers": 28, "pages": 256, "page": 32, "live": 0.6,
         "out_pages": 160, "index": True},
        # four chats behind a short system prompt: latency
        {"name": "shared_4_prefix_512", "op": "shared", **qwen, "page": 16, "groups": 1, "per_group": 4, "uneven": False,
         "prefix": 32, "own": 48, "q_len": 1},
        # a serving batch behind one long document, ragged own parts
        {"name": "shared_64_prefix_8k", "op": "shared", **qwen, "page": 64, "groups": 1, "per_group": 64,
         "uneven": False, "prefix": 128, "own": 512, "q_len": 1},
        # several system prompts, groups of uneven size, four tokens a step (speculation), smaller heads, groups of three
        {"name": "shared_6_groups_q4_d64", "op": "shared", "hq": 24, "hkv": 8, "d": 64, "dtype": "fp16", "page": 32,
         "groups": 6, "per_group": 16, "uneven": True, "prefix": 65, "own": 333, "q_len": 4},
        # the largest: 128 questions about one book
        {"name": "shared_128_prefix_32k", "op": "shared", **qwen, "page": 64, "groups": 1, "per_group": 128,
         "uneven": False, "prefix": 512, "own": 256, "q_len": 1},
        # one conversation at 32k, small pages: latency
        {"name": "sparse_1_32k", "op": "sparse", **qwen, "page": 16, "seqs": 1, "q_len": 1, "ctx": 32768, "top_k": 64},
        # a decode batch at up to 64k
        {"name": "sparse_16_64k", "op": "sparse", **qwen, "page": 64, "seqs": 16, "q_len": 1, "ctx": 65536,
         "top_k": 32},
        # a chunk of prompt on a context of 16k, every token with its own choice
        {"name": "sparse_chunk_2x250", "op": "sparse", **{**qwen, "dtype": "fp16"}, "page": 64, "seqs": 2, "q_len": 250,
         "ctx": 16384, "top_k": 16},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rope", "fork", "compact", "shared", "shared", "sparse", "sparse"])
    hkv, g = rng.choice([(8, 2), (8, 2), (8, 4), (4, 7), (2, 5), (1, 8), (8, 1), (4, 8)])
    c = {"op": op, "hq": hkv * g, "hkv": hkv, "d": rng.choice([64, 128, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
         "page": rng.choice([16, 32, 64, 128])}
    wide = c["hq"] * c["d"] / 2048   # relative width of a token
    if op == "rope":
        n = log(1, 32000 / max(1.0, wide))
        c["seqs"] = min(n, log(1, 128))
        c["q_len"] = max(1, n // c["seqs"])
        c["ctx"] = log(1, 30000)
        c["rot"] = rng.choice([c["d"], c["d"], c["d"] // 2, c["d"] // 4])
        c["interleaved"] = rng.random() < 0.5
        c["yarn"] = rng.choice([1.0, 1.0, 4.0])
        c["index"] = rng.random() < 0.5
    elif op == "fork":
        c["layers"] = log(1, 28)
        c["parents"] = rng.randint(1, 3)
        c["children"] = log(1, 64)
        c["length"] = log(1, 2100)
        c["grow"] = log(1, 65)
        need = c["parents"] * -(-c["length"] // c["page"]) + c["children"] * (2 + -(-c["grow"] // c["page"]))
        c["pages"] = need + log(4, 100)
        while c["pages"] * c["page"] * c["layers"] > 256 * 64 * 28 and c["layers"] > 1:
            c["layers"] -= 1
        if c["pages"] * c["page"] * c["layers"] > 256 * 64 * 28:
            c["children"] = 8
            c["pages"] = c["parents"] * -(-c["length"] // c["page"]) + 8 * (2 + -(-c["grow"] // c["page"])) + 5
    elif op == "compact":
        c["layers"] = log(1, 28)
        c["pages"] = log(3, max(4, 256 * 32 * 28 // (c["page"] * c["layers"])))
        c["pages"] = min(c["pages"], 4096)
        c["live"] = rng.choice([0.2, 0.5, 0.6])
        c["out_pages"] = max(1, int(c["pages"] * 0.65))
        c["index"] = rng.random() < 0.5
    elif op == "shared":
        c["groups"] = rng.choice([1, 1, 2, log(2, 12)])
        n = log(1, 128 / max(1.0, wide))
        c["per_group"] = max(1, n // c["groups"])
        c["uneven"] = rng.random() < 0.5
        c["q_len"] = rng.choice([1, 1, 1, 2, 5]) if n <= 32 else 1
        c["prefix"] = max(1, log(64, 32768 / max(1, c["groups"])) // c["page"])
        c["own"] = log(1, 256)
    else:
        c["seqs"] = log(1, 16)
        c["q_len"] = rng.choice([1, 1, 1, 3, log(8, 200)])
        if c["q_len"] > 3:
            c["seqs"] = min(c["seqs"], 2)
        c["ctx"] = log(100, 65536 if c["q_len"] == 1 else 16384)
        c["ctx"] = max(c["ctx"], c["q_len"])
        c["top_k"] = max(1, log(16, 1024 if c["q_len"] > 3 else 2048) // c["page"])
    return c


# ------------------------------------------------------------------------------------------------------------------
# sizes that follow from a case

def _ceil(a, b):
    return -(-a // b)


def _rope_starts(c):
    """First position of each sequence's new tokens."""
    return [(c["ctx"] * (b * 37 % 101)) // 101 for b in range(c["seqs"])]


def _group_sizes(c):
    n = c["per_group"]
    return [max(1, n - (g * 5) % n) if c["uneven"] else n for g in range(c["groups"])]


def _shared_sizes(c):
    """(group starts, prefix pages per group, sequence lengths)."""
    sizes = _group_sizes(c)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    prefix = [max(1, c["prefix"] - g * 3 % c["prefix"]) for g in range(c["groups"])]
    lens = []
    for g, n in enumerate(sizes):
        for b in range(n):
            lens.append(prefix[g] * c["page"] + c["q_len"] + (c["own"] * (b * 53 % 97)) // 97)
    return starts, prefix, lens


def _sparse_lens(c):
    """The context of each sequence, its new tokens included."""
    return [max(c["q_len"], c["ctx"] - (c["ctx"] * (b * 29 % 61)) // 122) for b in range(c["seqs"])]


# ------------------------------------------------------------------------------------------------------------------
# inputs

def _tables(max_pos, rot, factor, theta=1_000_000.0, trained=40960):
    """fp32 cos and sin [max_pos, rot / 2]; factor > 1 scales the slow channels for a longer context (YaRN)."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    inv = theta ** (-2.0 * i / rot)
    mult = 1.0
    if factor > 1.0:
        def at(turns):
            return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(0.0, math.floor(at(32.0))), min(rot - 1.0, math.ceil(at(1.0)))
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
        mult = 0.1 * math.log(factor) + 1.0
    a = torch.outer(torch.arange(max_pos, dtype=torch.float64), inv)
    return (a.cos() * mult).float().to(DEV), (a.sin() * mult).float().to(DEV)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pool(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    x.normal_(0.0, scale, generator=g)
    return x


def _refs(table, pages):
    t = table.reshape(-1)
    return torch.zeros(pages + 1, dtype=torch.int32, device=DEV).index_add_(
        0, torch.where(t >= 0, t, pages).long(), torch.ones_like(t))[:pages].contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    gc = torch.Generator().manual_seed(int(seed))
    dt = TYPES[c["dtype"]]
    s = SimpleNamespace(c=dict(c), page=c["page"], scale=1.0 / math.sqrt(c["d"]), index=None)
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]

    if c["op"] == "rope":
        starts = _rope_starts(c)
        n = c["q_len"]
        cols = [_ceil(p + n, page) for p in starts]
        pages, layers = sum(cols) + 3, 2
        s.layer = 1
        perm = torch.randperm(pages, generator=gc).int()
        table = torch.full((c["seqs"], max(cols) + 1), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(cols):
            table[b, :k] = perm[at:at + k]
            at += k
        s.table = table.to(DEV)
        s.k = _pool(g, (pages, layers, hkv, page, d), dt)
        s.v = _pool(g, (pages, layers, hkv, page, d), dt)
        if c["index"]:
            s.index = torch.zeros(pages, layers, hkv, 2 * d + PAD, dtype=torch.int8, device=DEV)
        # q, k and v as a projection leaves them: side by side in one row
        qkv = _pool(g, (c["seqs"] * n, (hq + 2 * hkv) * d), dt)
        s.q_in = qkv[:, :hq * d].unflatten(1, (hq, d))
        s.k_in = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        s.v_in = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        s.slots = torch.arange(c["seqs"], device=DEV).repeat_interleave(n).int()
        s.positions = (torch.tensor(starts, device=DEV)[:, None] + torch.arange(n, device=DEV)).reshape(-1).int()
        s.cos, s.sin = _tables(c["ctx"] + n, c["rot"], c["yarn"])

    elif c["op"] == "fork":
        pages = c["pages"]
        pp = _ceil(c["length"], page)
        cols = _ceil(c["length"] + c["grow"], page) + 1
        perm = torch.randperm(pages, generator=gc).int()
        table = torch.full((c["parents"] + c["children"] + 1, cols), -1, dtype=torch.int32)
        for b in range(c["parents"]):
            table[b, :pp] = perm[b * pp:(b + 1) * pp]
        s.table = table.to(DEV)
        s.lengths = torch.zeros(table.shape[0], dtype=torch.int32)
        s.lengths[:c["parents"]] = c["length"]
        s.lengths = s.lengths.to(DEV)
        s.refs = _refs(s.table, pages)
        s.k = _pool(g, (pages, c["layers"], hkv, page, d), dt)
        s.v = _pool(g, (pages, c["layers"], hkv, page, d), dt)
        kids = torch.randperm(c["children"], generator=gc).int() + c["parents"]
        s.children = kids.to(DEV)
        s.parents = torch.randint(0, c["parents"], (c["children"],), generator=gc).int().to(DEV)
        s.new_lengths = _ints([c["length"] + 1 + i * 31 % c["grow"] for i in range(c["children"])])

    elif c["op"] == "compact":
        pages = c["pages"]
        live = max(1, int(pages * c["live"]))
        rows = min(16, live)
        per = _ceil(live, rows)
        perm = torch.randperm(pages, generator=gc).int()[:live]
        flat = torch.full((rows * per,), -1, dtype=torch.int32)
        flat[:live] = perm
        table = flat.view(rows, per)
        if rows > 1 and per > 2:
            table[1, 0] = table[0, 0]   # a shared first page
        s.table = table.to(DEV)
        s.refs = _refs(s.table, pages)
        s.k = _pool(g, (pages, c["layers"], hkv, page, d), dt)
        s.v = _pool(g, (pages, c["layers"], hkv, page, d), dt)
        s.out_k = torch.zeros((c["out_pages"],) + s.k.shape[1:], dtype=dt, device=DEV)
        s.out_v = torch.zeros_like(s.out_k)
        s.out_table = torch.empty_like(s.table)
        s.out_refs = torch.empty(c["out_pages"], dtype=torch.int32, device=DEV)
        s.out_index = None
        if c["index"]:
            s.index = torch.randint(-127, 128, (pages, c["layers"], hkv, 2 * d + PAD), dtype=torch.int8, device=DEV,
                                    generator=g)
            s.out_index = torch.zeros((c["out_pages"],) + s.index.shape[1:], dtype=torch.int8, device=DEV)

    elif c["op"] == "shared":
        starts, prefix, lens = _shared_sizes(c)
        n, s.layer = len(lens), 0
        own_cols = [_ceil(lens[b], page) - prefix[gi] for gi in range(c["groups"]) for b in range(starts[gi], starts[gi + 1])]
        pages = sum(prefix) + sum(own_cols) + 2
        perm = torch.randperm(pages, generator=gc).int()
        table = torch.full((n + 1, max(_ceil(x, page) for x in lens) + 1), -1, dtype=torch.int32)
        order = torch.randperm(n + 1, generator=gc)[:n]
        at = 0
        for gi in range(c["groups"]):
            head = perm[at:at + prefix[gi]]
            at += prefix[gi]
            for b in range(starts[gi], starts[gi + 1]):
                table[order[b], :prefix[gi]] = head
                table[order[b], prefix[gi]:prefix[gi] + own_cols[b]] = perm[at:at + own_cols[b]]
                at += own_cols[b]
        s.table = table.to(DEV)
        s.slots = order.int().to(DEV)
        lengths = torch.zeros(n + 1, dtype=torch.int32)
        lengths[order] = torch.tensor(lens, dtype=torch.int32)
        s.lengths = lengths.to(DEV)
        s.group_starts, s.prefix = _ints(starts), _ints(prefix)
        s.q_starts = None if c["q_len"] == 1 else _ints([b * c["q_len"] for b in range(n + 1)])
        s.k = _pool(g, (pages, 1, hkv, page, d), dt)
        s.v = _pool(g, (pages, 1, hkv, page, d), dt)
        s.q = _pool(g, (n * c["q_len"], hq, d), dt, 2.0)   # logits of standard deviation 2
        s.max_group, s.max_prefix = max(_group_sizes(c)), max(prefix)
        s.max_own = max(own_cols)

    else:
        lens = _sparse_lens(c)
        s.layer = 0
        cols = [_ceil(x, page) for x in lens]
        pages = sum(cols) + 2
        perm = torch.randperm(pages, generator=gc).int()
        table = torch.full((c["seqs"], max(cols) + 1), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(cols):
            table[b, :k] = perm[at:at + k]
            at += k
        s.table = table.to(DEV)
        # keys that lean page by page to a direction of their own, as neighbouring tokens do
        s.k = _pool(g, (pages, 1, hkv, page, d), dt, 0.8)
        s.k += _pool(g, (pages, 1, hkv, 1, d), dt, 0.6)
        s.v = _pool(g, (pages, 1, hkv, page, d), dt)
        s.index = torch.zeros(pages, 1, hkv, 2 * d + PAD, dtype=torch.int8, device=DEV)
        for lo in range(0, pages, 2048):
            s.index[lo:lo + 2048] = _index_of(s.k[lo:lo + 2048])
        s.q = _pool(g, (c["seqs"] * c["q_len"], hq, d), dt, 1.5)
        s.slots = torch.arange(c["seqs"], device=DEV).repeat_interleave(c["q_len"]).int()
        s.positions = (torch.tensor([x - c["q_len"] for x in lens], device=DEV)[:, None]
                       + torch.arange(c["q_len"], device=DEV)).reshape(-1).int()
        s.max_pages = max(cols)
    return s


# ------------------------------------------------------------------------------------------------------------------
# plain forms

def _quantise(x):
    """Whole numbers of magnitude up to 127 and the power of two they count in, along the last dimensions of x."""
    return _quantise_by(x, x.abs().amax(-1, keepdim=True))


def _two_to(e):
    """2^e in fp32, from its bits (a power function may be off by a unit)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise_by(x, a):
    e = torch.frexp(a)[1] - 7   # floor(log2 a) - 6
    e = torch.where(a > 0, e.clamp(-60, 40), torch.zeros_like(e))
    return (x * _two_to(-e)).round().clamp(-127, 127), e


def _index_of(k):
    """Index records [..., 2 d + 16] of full pages k [..., page, d]."""
    k = k.float()
    hi, lo = k.amax(-2), k.amin(-2)
    both = torch.cat([hi, lo], -1)
    q, e = _quantise_by(both, both.abs().amax(-1, keepdim=True))
    return torch.cat([q, e.float(), torch.zeros_like(q[..., :PAD - 1])], -1).to(torch.int8)


def _plain_rope(s):
    page, rot = s.page, s.c["rot"]
    cos, sin = s.cos[s.positions.long()][:, None], s.sin[s.positions.long()][:, None]

    def turn(x):
        x = x.float()
        r, rest = x[..., :rot], x[..., rot:]
        if s.c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
        else:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
        y0, y1 = a * cos - b * sin, b * cos + a * sin
        y = torch.stack([y0, y1], -1).flatten(-2) if s.c["interleaved"] else torch.cat([y0, y1], -1)
        return torch.cat([y, rest], -1)

    q = turn(s.q_in).to(s.q_in.dtype)
    pos = s.positions.long()
    pages, rows = s.table[s.slots.long(), pos // page].long(), pos % page
    s.k[pages, s.layer, :, rows] = turn(s.k_in).to(s.k.dtype)
    s.v[pages, s.layer, :, rows] = s.v_in
    out = {"q": q, "k_pages": s.k, "v_pages": s.v}
    if s.index is not None:
        done = pages[rows == page - 1]
        s.index[done, s.layer] = _index_of(s.k[done, s.layer])
        out["index"] = s.index
    return out


def _plain_free(table, lengths, refs, slots, page):
    slots = slots.long()
    rows = table[slots]
    used = torch.arange(table.shape[1], device=DEV) < ((lengths[slots] + page - 1) // page)[:, None]
    refs.index_add_(0, torch.where(used, rows, 0).reshape(-1).long(), -used.reshape(-1).int())
    table[slots] = -1
    lengths[slots] = 0


def _free_pages(refs):
    """All pages, the free ones first, in ascending order."""
    return torch.sort((refs > 0).int(), stable=True).indices


def _plain_fork(s):
    page, kids, parents = s.page, s.children.long(), s.parents.long()
    table, lengths, refs = s.table, s.lengths, s.refs
    _plain_free(table, lengths, refs, kids, page)
    # fork: whole pages shared, the part page copied into the lowest free pages, in the children's order
    col = torch.arange(table.shape[1], device=DEV)
    full, part = lengths[parents] // page, lengths[parents] % page
    shared = col < full[:, None]
    rows = torch.where(shared, table[parents], -1)
    refs.index_add_(0, torch.where(shared, rows, 0).reshape(-1).long(), shared.reshape(-1).int())
    need = part > 0
    dst = _free_pages(refs)[(need.cumsum(0) - 1).clamp(min=0)]
    src = table[parents, full.long().clamp(max=table.shape[1] - 1)].long()
    refs.index_add_(0, torch.where(need, dst, 0), need.int())
    rows = torch.where((col == full[:, None]) & need[:, None], dst[:, None].int(), rows)
    src, to = torch.where(need, src, 0), torch.where(need, dst, 0)
    keep = (torch.arange(page, device=DEV) >= part[:, None])[:, None, None, :, None]
    s.k[to] = torch.where(keep, s.k[to], s.k[src])
    s.v[to] = torch.where(keep, s.v[to], s.v[src])
    table[kids] = rows.int()
    lengths[kids] = lengths[parents]
    # reserve: the children's new pages, the lowest free ones in the children's order
    have = (lengths[kids] + page - 1) // page
    want = (s.new_lengths + page - 1) // page
    first = (want - have).cumsum(0) - (want - have)
    new = (col >= have[:, None]) & (col < want[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, refs.numel() - 1)
    ids = _free_pages(refs)[at.long()].int()
    refs.index_add_(0, torch.where(new, ids, 0).reshape(-1).long(), new.reshape(-1).int())
    table[kids] = torch.where(new, ids, table[kids])
    lengths[kids] = s.new_lengths


def _plain_compact(s):
    live = s.refs > 0
    new = live.cumsum(0) - 1
    order = torch.sort(live.int(), descending=True, stable=True).indices[:s.out_refs.numel()]
    there = (torch.arange(s.out_refs.numel(), device=DEV) < live.sum())
    wide = there[:, None, None, None, None]
    s.out_k.copy_(torch.where(wide, s.k[order], s.out_k))
    s.out_v.copy_(torch.where(wide, s.v[order], s.out_v))
    if s.index is not None:
        s.out_index.copy_(torch.where(wide[..., 0], s.index[order], s.out_index))
    s.out_table.copy_(torch.where(s.table >= 0, new[s.table.long().clamp(min=0)], -1))
    s.out_refs.copy_(torch.where(there, s.refs[order], 0))


def _gather(pages, layer, ids):
    """Rows of the pages ids [n, m] as fp32 [n, hkv, m * page, d]."""
    x = pages[:, layer][ids.long().clamp(0, pages.shape[0] - 1)]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _part(score, seen, v, expr):
    score = torch.where(seen, score, -math.inf)
    m = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(m.isinf(), 0.0, m))
    return m[..., 0], p.sum(-1), torch.einsum(expr, p, v)


def _plain_shared(s):
    c, page, n = s.c, s.page, s.slots.numel()
    hkv, grp, d, ql = c["hkv"], c["hq"] // c["hkv"], c["d"], c["q_len"]
    q = s.q.float().view(n, ql, hkv, grp, d)
    lens = s.lengths[s.slots.long()]
    pos = lens[:, None] - ql + torch.arange(ql, device=DEV)
    seq = torch.arange(n, device=DEV)
    group = torch.bucketize(seq, s.group_starts[1:].long(), right=True)
    # the prefix: the rows of a group side by side, its keys once
    lead = s.group_starts[:-1].long()
    ids = s.table[s.slots[lead].long(), :s.max_prefix]
    kp, vp = _gather(s.k, s.layer, ids), _gather(s.v, s.layer, ids)
    member = (lead[:, None] + torch.arange(s.max_group, device=DEV)).clamp(max=n - 1)
    score = torch.einsum("gbqhrd,ghld->gbqhrl", q[member], kp) * s.scale
    seen = (torch.arange(kp.shape[2], device=DEV) < s.prefix[:, None] * page)[:, None, None, None, None]
    m0, l0, a0 = _part(score, seen, vp, "gbqhrl,ghld->gbqhrd")
    m0, l0, a0 = (x[group, seq - lead[group]] for x in (m0, l0, a0))
    # each sequence's own part
    col = s.prefix[group][:, None] + torch.arange(s.max_own, device=DEV)
    ids = s.table[s.slots.long()[:, None], col.long().clamp(max=s.table.shape[1] - 1)]
    ko, vo = _gather(s.k, s.layer, ids), _gather(s.v, s.layer, ids)
    at = s.prefix[group][:, None] * page + torch.arange(ko.shape[2], device=DEV)
    score = torch.einsum("bqhrd,bhld->bqhrl", q, ko) * s.scale
    m1, l1, a1 = _part(score, (at[:, None] <= pos[..., None])[:, :, None, None], vo, "bqhrl,bhld->bqhrd")
    m = torch.maximum(m0, m1)
    e0, e1 = torch.exp(m0 - m), torch.exp(m1 - m)
    out = (a0 * e0[..., None] + a1 * e1[..., None]) / (l0 * e0 + l1 * e1)[..., None]
    return out.reshape(n * ql, hkv * grp, d).to(s.q.dtype)


def _plain_sparse(s):
    c, page, n, ql, top = s.c, s.page, s.c["seqs"], s.c["q_len"], s.c["top_k"]
    hkv, grp, d = c["hkv"], c["hq"] // c["hkv"], c["d"]
    q = s.q.float().view(n, ql, hkv, grp, d)
    pos = s.positions.view(n, ql)
    ids = s.table[:, :s.max_pages]
    rec = s.index[:, s.layer][ids.long().clamp(min=0)].float()          # [n, pages, hkv, 2 d + 16]
    qi, qe = _quantise(q)
    two = torch.cat([qi.clamp(min=0), qi.clamp(max=0)], -1)
    score = torch.einsum("bqhrd,bphd->bqhrp", two, rec[..., :2 * d])     # whole numbers below 2^24
    score = (score * _two_to(qe)).amax(3) * _two_to(rec[..., 2 * d]).permute(0, 2, 1)[:, None]
    own_page = (pos // page)[:, :, None, None]
    col = torch.arange(s.max_pages, device=DEV)
    score = torch.where(col < own_page, score, -math.inf)
    score = torch.where(col == own_page, math.inf, score)
    best, pick = torch.sort(score, dim=-1, descending=True, stable=True)
    some = min(top, s.max_pages)
    pick = torch.where(best[..., :some] > -math.inf, pick[..., :some], s.max_pages).sort(-1).values
    sel = torch.full((n, ql, hkv, top), -1, dtype=torch.int32, device=DEV)
    sel[..., :some] = torch.where(pick < s.max_pages, pick, -1).int()
    # the chosen pages' rows, for each token and kv head
    page_id = torch.gather(ids.long()[:, None, None].expand(n, ql, hkv, -1), 3, sel.long().clamp(min=0)).clamp(min=0)
    head = torch.arange(hkv, device=DEV)[None, None, :, None]
    k = s.k[:, s.layer][page_id, head].flatten(3, 4).float()             # [n, ql, hkv, top * page, d]
    v = s.v[:, s.layer][page_id, head].flatten(3, 4).float()
    at = (sel[..., None] * page + torch.arange(page, device=DEV)).flatten(3)
    seen = (at <= pos[:, :, None, None]) & (sel >= 0).repeat_interleave(page, -1)
    sc = torch.einsum("bqhrd,bqhld->bqhrl", q, k) * s.scale
    m, l, a = _part(sc, seen[:, :, :, None], v, "bqhrl,bqhld->bqhrd")
    out = (a / l[..., None]).reshape(n * ql, hkv * grp, d).to(s.q.dtype)
    return {"out": out, "selected": sel.view(n * ql, hkv, top)}


def _fork_state(s):
    return {"table": s.table, "lengths": s.lengths, "refs": s.refs, "k_pages": s.k, "v_pages": s.v}


def _compact_state(s):
    got = {"table": s.out_table, "refs": s.out_refs, "k_pages": s.out_k, "v_pages": s.out_v}
    if s.index is not None:
        got["index"] = s.out_index
    return got


def run(s):
    op = s.c["op"]
    if not own:
        if op == "rope":
            return _plain_rope(s)
        if op == "fork":
            _plain_fork(s)
            return _fork_state(s)
        if op == "compact":
            _plain_compact(s)
            return _compact_state(s)
        return _plain_shared(s) if op == "shared" else _plain_sparse(s)
    from megaqwen_b200 import paged
    if op == "rope":
        q = paged.rope_append(s.q_in, s.k_in, s.v_in, s.k, s.v, s.table, s.slots, s.positions, s.cos, s.sin,
                              layer=s.layer, interleaved=s.c["interleaved"], index=s.index)
        out = {"q": q, "k_pages": s.k, "v_pages": s.v}
        return out if s.index is None else {**out, "index": s.index}
    if op == "fork":
        paged.free(s.table, s.lengths, s.refs, s.children, s.page)
        paged.fork(s.k, s.v, s.table, s.lengths, s.refs, s.parents, s.children)
        paged.reserve(s.table, s.lengths, s.refs, s.children, s.new_lengths, s.page)
        return _fork_state(s)
    if op == "compact":
        paged.compact(s.k, s.v, s.table, s.refs, s.out_k, s.out_v, s.out_table, s.out_refs, index=s.index,
                      out_index=s.out_index)
        return _compact_state(s)
    if op == "shared":
        return paged.attend(s.q, s.k, s.v, s.table, s.lengths, s.slots, layer=s.layer, q_starts=s.q_starts,
                            group_starts=s.group_starts, prefix_pages=s.prefix, scale=s.scale)
    out, sel = paged.sparse_attend(s.q, s.k, s.v, s.index, s.table, s.slots, s.positions, layer=s.layer,
                                   top_k=s.c["top_k"], scale=s.scale)
    return {"out": out, "selected": sel}


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    c = case
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    row = hkv * d * 2                       # bytes of one token's keys in one layer
    if c["op"] == "rope":
        n = c["seqs"] * c["q_len"]
        b = n * ((hq + 2 * hkv) * d * 2 * 2 + 8)
        b += len({p + i for p in _rope_starts(c) for i in range(c["q_len"])}) * c["rot"] * 4
        if c["index"]:
            b += sum((p + c["q_len"]) // page - p // page for p in _rope_starts(c)) * hkv * (2 * d + 1)
        return {"bytes": b, "flops": n * (hq + hkv) * c["rot"] * 3}
    if c["op"] == "fork":
        part = c["length"] % page
        moved = 2 * c["layers"] * part * row
        cols = _ceil(c["length"], page)
        return {"bytes": moved * (c["parents"] if c["children"] >= c["parents"] else c["children"])
                + moved * c["children"] + c["children"] * (3 * cols + 4) * 4 + c["pages"] * 4, "flops": 0}
    if c["op"] == "compact":
        live = max(1, int(c["pages"] * c["live"]))
        if min(16, live) > 1 and _ceil(live, min(16, live)) > 2:
            live -= 1
        one = 2 * c["layers"] * page * row + (c["layers"] * hkv * (2 * d + PAD) if c["index"] else 0)
        return {"bytes": 2 * live * one + c["pages"] * 4, "flops": 0}
    if c["op"] == "shared":
        starts, prefix, lens = _shared_sizes(c)
        keys, pairs = sum(prefix) * page, 0
        for gi in range(c["groups"]):
            for b in range(starts[gi], starts[gi + 1]):
                keys += lens[b] - prefix[gi] * page
                pairs += sum(lens[b] - i for i in range(c["q_len"]))
        return {"bytes": keys * 2 * row + len(lens) * c["q_len"] * hq * d * 2 * 2 + keys // page * 4,
                "flops": pairs * hq * d * 4}
    lens, t = _sparse_lens(c), c["q_len"]
    b, f = len(lens) * t * hq * d * 4, 0
    for n in lens:
        old = (n - 1) // page
        read = sum(min(c["top_k"] - 1, (n - t + i) // page) * page + (n - t + i) % page + 1 for i in range(t))
        b += old * hkv * (2 * d + 1) + min(read, n) * 2 * row + t * hkv * c["top_k"] * 4
        f += read * hq * d * 4 + t * old * hq * d * 2
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits

def _softmax64(q, k, v, seen, scale):
    """q [t, hq, d], k and v [l, hkv, d], seen [t, hq, l], all in 64 bits."""
    grp = q.shape[1] // k.shape[1]
    k, v = k.permute(1, 2, 0), v.permute(1, 0, 2)
    out = torch.empty_like(q)
    for h in range(k.shape[0]):
        z = torch.matmul(q[:, h * grp:(h + 1) * grp], k[h]) * scale
        z = z.masked_fill(~seen[:, h * grp:(h + 1) * grp], -math.inf)
        out[:, h * grp:(h + 1) * grp] = torch.matmul(torch.softmax(z, -1), v[h])
    return out


def _rows64(pages, layer, ids, count):
    return torch.cat([pages[int(i), layer].transpose(0, 1) for i in ids])[:count].double()


def exact(case, seed):
    c = case
    if c["op"] in ("fork", "compact"):
        return None   # copies and whole numbers only
    s = prepare(case, seed)
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    if c["op"] == "rope":
        pos = s.positions.long()
        ang = torch.complex(s.cos.double()[pos], s.sin.double()[pos])[:, None]

        def turn(x):
            x = x.double().clone()
            half = c["rot"] // 2
            i = torch.arange(half, device=DEV)
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
            z = torch.complex(x[..., a], x[..., b]) * ang
            x[..., a], x[..., b] = z.real, z.imag
            return x

        k = s.k.double()
        v = s.v.double()
        to = s.table[s.slots.long(), pos // page].long()
        k[to, s.layer, :, pos % page] = turn(s.k_in)
        v[to, s.layer, :, pos % page] = s.v_in.double()
        out = {"q": turn(s.q_in), "k_pages": k, "v_pages": v}
        # the index holds the rounded keys' bounds as whole numbers: no value of its own in 64 bits
        return out if s.index is None else {**out, "index": None}
    if c["op"] == "shared":
        _, _, lens = _shared_sizes(c)
        slots, table, t = s.slots.tolist(), s.table.cpu(), c["q_len"]
        out = torch.empty(len(lens) * t, hq, d, dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            ids = table[slots[b], :_ceil(n, page)].tolist()
            k, v = (_rows64(x, 0, ids, n) for x in (s.k, s.v))
            at = n - t + torch.arange(t, device=DEV)
            seen = (torch.arange(n, device=DEV) <= at[:, None])[:, None].expand(t, hq, n)
            out[b * t:(b + 1) * t] = _softmax64(s.q[b * t:(b + 1) * t].double(), k, v, seen, s.scale)
        return out
    lens, t, table = _sparse_lens(c), c["q_len"], s.table.cpu()
    out = torch.empty(len(lens) * t, hq, d, dtype=torch.float64, device=DEV)
    chosen = torch.full((len(lens) * t, hkv, c["top_k"]), -1, dtype=torch.int32, device=DEV)

    power = torch.tensor([2.0 ** i for i in range(-60, 41)], dtype=torch.float64, device=DEV)

    def whole(x):
        a = x.abs().amax(-1, keepdim=True)
        e = (torch.frexp(a).exponent - 7).clamp(-60, 40).long()
        unit = power[torch.where(a > 0, e, 0) + 60]
        return torch.round(x / unit).clamp(-127, 127), unit

    for b, n in enumerate(lens):
        m = _ceil(n, page)
        ids = table[b, :m].tolist()
        k, v = (_rows64(x, 0, ids, n) for x in (s.k, s.v))
        q = s.q[b * t:(b + 1) * t].double()
        at = n - t + torch.arange(t, device=DEV)
        own_page = at // page
        score = torch.full((t, hkv, m), -math.inf, dtype=torch.float64, device=DEV)
        full = n // page
        if full:
            kk = k[:full * page].view(full, page, hkv, d)
            both = torch.stack([kk.amax(1), kk.amin(1)], -2)                # [pages, hkv, 2, d]
            w, unit = whole(both.flatten(-2))
            hi, lo = w[..., :d], w[..., d:]
            qi, q_unit = whole(q)
            for h in range(hkv):
                x = qi.view(t, hkv, -1, d)[:, h]
                y = torch.matmul(x.clamp(min=0), hi[:, h].T) + torch.matmul(x.clamp(max=0), lo[:, h].T)
                y = (y * q_unit.view(t, hkv, -1, 1)[:, h]).amax(1) * unit[:, h, 0]
                score[:, h, :full] = y
        col = torch.arange(m, device=DEV)
        score = score.masked_fill(col >= own_page[:, None, None], -math.inf)
        score = score.masked_fill(col == own_page[:, None, None], math.inf)
        got = torch.sort(score, dim=-1, descending=True, stable=True)
        some = min(c["top_k"], m)
        ok = got.values[..., :some] > -math.inf
        take = torch.zeros(t, hkv, m + 1, dtype=torch.bool, device=DEV)
        take.scatter_(2, torch.where(ok, got.indices[..., :some], m), True)
        take = take[..., :m]
        pick = torch.where(take, col, m).sort(-1).values[..., :some]
        chosen[b * t:(b + 1) * t, :, :some] = torch.where(pick < m, pick, -1).int()
        seen = take.repeat_interleave(page, -1)[..., :n] & (torch.arange(n, device=DEV) <= at[:, None])[:, None]
        seen = seen.repeat_interleave(hq // hkv, 1)
        out[b * t:(b + 1) * t] = _softmax64(q, k, v, seen, s.scale)
    return {"out": out, "selected": chosen}
