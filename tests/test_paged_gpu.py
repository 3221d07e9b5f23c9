"""Paged KV cache: every operator against a plain implementation in 64 bits
(bookkeeping: against a Python model of it, exactly).

Tolerances.  An output is rounded once to its type: half a unit is 2^-8 of the
value for bf16 and 2^-11 for fp16.  Attention adds the error of the weights:
scores are fp32 sums of 16-bit products (at most ~3e-5 off for the magnitudes
drawn here, sum |q k| scale < 40), and the weights enter the second product in
two 16-bit pieces (2^-16); together below 2^-13 of the largest value.
Rotations round two products and a sum in fp32: 2^-22 of the pair's magnitudes.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


def dev(x, dtype=torch.int32):
    return torch.as_tensor(x, dtype=dtype, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


class Pool:
    """A pool with sequences of given lengths on shuffled pages."""

    def __init__(self, lens, page, hkv, d, dtype, layers=2, seed=0, extra_slots=1, share=None):
        g = gen(seed)
        self.page, self.lens, self.dtype = page, list(lens), dtype
        cols = [-(-n // page) for n in lens]
        shared = {}
        if share:   # {sequence: (leader, pages)}
            shared = share
        need = sum(c - (shared[b][1] if b in shared else 0) for b, c in enumerate(cols)) + 3
        perm = torch.randperm(need, generator=torch.Generator().manual_seed(seed)).tolist()
        self.rows = []
        for b, c in enumerate(cols):
            row = []
            if b in shared:
                row = self.rows[shared[b][0]][:shared[b][1]]
            row = row + [perm.pop() for _ in range(c - len(row))]
            self.rows.append(row)
        self.spare = perm
        n = len(lens) + extra_slots
        width = max([1] + cols) + 1
        self.table = torch.full((n, width), -1, dtype=torch.int32)
        self.lengths = torch.zeros(n, dtype=torch.int32)
        order = torch.randperm(n, generator=torch.Generator().manual_seed(seed + 1)).tolist()
        self.slots = order[:len(lens)]
        for b, row in enumerate(self.rows):
            self.table[self.slots[b], :len(row)] = torch.tensor(row, dtype=torch.int32)
            self.lengths[self.slots[b]] = lens[b]
        self.table, self.lengths = self.table.cuda(), self.lengths.cuda()
        self.k = normal(g, need, layers, hkv, page, d, dtype=dtype)
        self.v = normal(g, need, layers, hkv, page, d, dtype=dtype)
        self.g = g

    def kv(self, b, layer):
        """Keys and values [len, hkv, d] of sequence b."""
        n = self.lens[b]
        ids = torch.tensor(self.rows[b], dtype=torch.long, device="cuda")
        k, v = (x[ids, layer].permute(0, 2, 1, 3).reshape(-1, x.shape[2], x.shape[4])[:n] for x in (self.k, self.v))
        return k.double(), v.double()


def softmax_rows(q, k, v, seen, scale):
    """q [hq, d] of one token, k/v [len, hkv, d], seen [len] or [hkv, len]: the output row in 64 bits."""
    hq, hkv = q.shape[0], k.shape[1]
    out = torch.zeros(hq, q.shape[1], dtype=torch.float64, device=q.device)
    for h in range(hq):
        j = h // (hq // hkv)
        s = seen if seen.dim() == 1 else seen[j]
        idx = torch.nonzero(s).flatten()
        if idx.numel():
            w = torch.softmax((k[idx, j] @ q[h].double()) * scale, 0)
            out[h] = w @ v[idx, j]
    return out


def close(got, ref, vmax):
    tol = ROUND[got.dtype] * ref.abs() + 2.0 ** -13 * vmax + 2.0 ** -24
    bad = (got.double() - ref).abs() - tol
    assert bool((bad <= 0).all()), f"over by {bad.max().item():.3e} (vmax {vmax:.3f})"


# ---- rotary positions --------------------------------------------------------------------------------------------

def rope_ref(x, pos, cos, sin, inter, inverse=False):
    x = x.double().clone()
    half = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None] * (-1 if inverse else 1)
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + half)
    x0, x1 = x[..., a].clone(), x[..., b].clone()
    mag = torch.zeros_like(x)
    mag[..., a] = mag[..., b] = x0.abs() + x1.abs()
    x[..., a], x[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    return x, mag


def rope_close(got, ref, mag):
    tol = ROUND[got.dtype] * ref.abs() + 2.0 ** -22 * mag + 2.0 ** -24
    assert bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 48), (128, 34), (64, 2), (128, 0)])
def test_rope(paged, dtype, inter, d, rot):
    g = gen(rot + d)
    n, heads = 37, 5
    cos, sin = (paged.rope_tables(300, max(rot, 2)))
    cos, sin = cos[:, :rot // 2].contiguous(), sin[:, :rot // 2].contiguous()
    x = normal(g, n, heads, d, dtype=dtype)
    pos = torch.randint(0, 300, (n,), device="cuda", generator=g).int()
    got = paged.rope(x, pos, cos, sin, interleaved=inter)
    ref, mag = rope_ref(x, pos.long(), cos, sin, inter)
    rope_close(got, ref, mag)
    assert torch.equal(got[..., rot:], x[..., rot:])
    # strided and unaligned views give the same bits
    wide = torch.zeros(n, heads, d + 7, dtype=dtype, device="cuda")
    for lo in (0, 1):
        wide[..., lo:lo + d] = x
        assert torch.equal(paged.rope(wide[..., lo:lo + d], pos, cos, sin, interleaved=inter), got)
    # the other way round
    back = paged.rope(x, pos, cos, sin, interleaved=inter, inverse=True)
    ref, mag = rope_ref(x, pos.long(), cos, sin, inter, inverse=True)
    rope_close(back, ref, mag)


@pytest.mark.parametrize("inter", [False, True])
def test_rope_gradient(paged, inter):
    """d <g, rope(x)> / dx is the inverse rotation of g: against autograd of the formula and against differences,
    both in 64 bits (the map is linear, so a difference is exact up to the rounding of the sums)."""
    g = gen(5)
    n, heads, d = 3, 2, 64
    cos, sin = paged.rope_tables(50, 32)
    pos = dev([0, 7, 49])
    x, grad = normal(g, n, heads, d), normal(g, n, heads, d)
    got = paged.rope(grad, pos, cos, sin, interleaved=inter, inverse=True)
    xd = x.double().requires_grad_(True)
    i = torch.arange(16, device="cuda")
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + 16)
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    y = xd.clone()
    y[..., a], y[..., b] = xd[..., a] * c - xd[..., b] * s, xd[..., b] * c + xd[..., a] * s
    (y * grad.double()).sum().backward()
    _, mag = rope_ref(grad, pos.long(), cos, sin, inter, inverse=True)
    rope_close(got, xd.grad, mag)

    def loss(z):
        return (rope_ref(z, pos.long(), cos, sin, inter)[0] * grad.double()).sum()
    for at in [(0, 0, 0), (1, 1, 17), (2, 0, 31), (1, 0, 40)]:
        e = torch.zeros(n, heads, d, dtype=torch.float64, device="cuda")
        e[at] = 0.5
        diff = loss(x.double() + e) - loss(x.double() - e)
        assert abs(diff.item() - got[at].item()) <= ROUND[got.dtype] * abs(diff.item()) + 2.0 ** -22 * mag[at].item() + 1e-9


def test_rope_tables(paged):
    cos, sin = paged.rope_tables(100, 64, theta=1e4, device="cpu")
    a = torch.outer(torch.arange(100).double(), 1e4 ** (-torch.arange(32).double() / 32))
    assert torch.equal(cos, a.cos().float()) and torch.equal(sin, a.sin().float())
    lin, _ = paged.rope_tables(100, 64, theta=1e4, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.allclose(lin[::4], cos[:25], atol=1e-6)
    for kind in ("yarn", "llama3"):
        c2, s2 = paged.rope_tables(100, 64, theta=1e4, scaling={"type": kind, "factor": 1.0, "trained": 4096}, device="cpu")
        assert torch.allclose(c2, cos, atol=1e-6) and torch.allclose(s2, sin, atol=1e-6)
        c2, s2 = paged.rope_tables(100, 64, theta=1e4, scaling={"type": kind, "factor": 8.0, "trained": 4096}, device="cpu")
        m = 0.1 * math.log(8.0) + 1.0 if kind == "yarn" else 1.0
        assert torch.allclose(c2[:, 0], cos[:, 0] * m, atol=1e-6)           # the fastest pair is kept
        ang = torch.atan2(s2[8, -1], c2[8, -1])
        assert math.isclose(ang.item(), a[1, -1].item(), rel_tol=1e-4)      # the slowest is divided by 8
    ntk, sn = paged.rope_tables(100, 64, theta=1e4, scaling={"type": "ntk", "factor": 8.0}, device="cpu")
    assert math.isclose(torch.atan2(sn[8, -1], ntk[8, -1]).item(), a[1, -1].item(), rel_tol=1e-4)
    assert torch.allclose(ntk[:, 0], cos[:, 0], atol=1e-6)
    for bad in ({"type": "nope"}, {"type": "linear", "factor": 0.5}, {"type": "linear", "factor": 2.0, "x": 1}):
        with pytest.raises(ValueError):
            paged.rope_tables(10, 64, scaling=bad)


def index_ref(k):
    """Records of full pages k [n, page, d] (16-bit): HI, LO, e from the definition, in 64 bits."""
    k = k.double()
    hi, lo = k.amax(1), k.amin(1)
    a = torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True)
    e = (torch.frexp(a).exponent - 7).clamp(-60, 40)
    e = torch.where(a > 0, e, torch.zeros_like(e))
    unit = torch.tensor([2.0 ** i for i in range(-60, 41)], dtype=torch.float64, device=k.device)[(e + 60).long()]
    return torch.cat([torch.round(hi / unit).clamp(-127, 127), torch.round(lo / unit).clamp(-127, 127), e.double()], -1).to(torch.int8)


@pytest.mark.parametrize("dtype,d,page,rot,inter,index", [
    (torch.bfloat16, 128, 16, 128, False, True), (torch.bfloat16, 128, 64, 64, True, True),
    (torch.float16, 64, 32, 64, False, True), (torch.float16, 128, 128, 32, True, True),
    (torch.bfloat16, 64, 128, 18, False, True), (torch.float16, 64, 16, 64, True, False)])
@pytest.mark.parametrize("news", [[1], [1, 1, 1], [5, 0, 130], [64, 16, 1, 33]])
def test_rope_append(paged, dtype, d, page, rot, inter, index, news):
    hkv, hq, layer = 3, 6, 1
    starts = [(b * 61) % 150 for b in range(len(news))]
    p = Pool([s + n for s, n in zip(starts, news)], page, hkv, d, dtype, seed=page + len(news))
    n = sum(news)
    cos, sin = paged.rope_tables(400, rot)
    qkv = normal(p.g, n, (hq + 2 * hkv) * d, dtype=dtype)
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
    slots = dev([p.slots[b] for b, c in enumerate(news) for _ in range(c)])
    pos = dev([s + i for s, c in zip(starts, news) for i in range(c)])
    idx = torch.full((p.k.shape[0], 2, hkv, 2 * d + 16), 99, dtype=torch.int8, device="cuda") if index else None
    k0, v0 = p.k.clone(), p.v.clone()
    status = dev([0])
    out = paged.rope_append(q, k, v, p.k, p.v, p.table, slots, pos, cos, sin, layer=layer, interleaved=inter, index=idx,
                            status=status)
    assert status.item() == 0
    ref, mag = rope_ref(q, pos.long(), cos, sin, inter)
    rope_close(out, ref, mag)
    ref, mag = rope_ref(k, pos.long(), cos, sin, inter)
    touched = torch.zeros(p.k.shape[0], page, dtype=torch.bool, device="cuda")
    at = 0
    for b, c in enumerate(news):
        for i in range(c):
            x = starts[b] + i
            pg, row = p.rows[b][x // page], x % page
            rope_close(p.k[pg, layer, :, row], ref[at], mag[at])
            assert torch.equal(p.v[pg, layer, :, row], v[at])
            touched[pg, row] = True
            at += 1
    keep = ~touched[:, None, None, :, None]
    other = torch.ones_like(p.k, dtype=torch.bool)
    other[:, layer] = keep[:, 0].expand_as(other[:, layer])
    assert torch.equal(p.k[other], k0[other]) and torch.equal(p.v[other], v0[other])
    if index:
        full = [p.rows[b][(starts[b] + i) // page] for b, c in enumerate(news) for i in range(c) if (starts[b] + i) % page == page - 1]
        want = torch.full_like(idx, 99)
        for pg in full:
            for h in range(hkv):
                rec = index_ref(p.k[pg:pg + 1, layer, h])[0]
                want[pg, layer, h, :2 * d + 1] = rec
                want[pg, layer, h, 2 * d + 1:] = 0
        assert torch.equal(idx, want)


def test_index_of_odd_keys(paged):
    """Zeros, one huge channel, infinities and NaN in a page's keys."""
    d, page = 64, 16
    p = Pool([16] * 5, page, 1, d, torch.bfloat16, layers=1)
    idx = torch.zeros(p.k.shape[0], 1, 1, 2 * d + 16, dtype=torch.int8, device="cuda")
    cos, sin = paged.rope_tables(16, 2)
    cos, sin = cos[:, :0].contiguous(), sin[:, :0].contiguous()   # no rotation: the keys go in as they are
    k = normal(p.g, 5, page, 1, d)
    k[0] = 0
    k[1, 3, 0, 5] = 2.0 ** 100
    k[2, 2, 0, 7] = math.inf
    k[2, 4, 0, 8] = -math.inf
    k[3, :, 0, 9] = math.nan
    k[4] *= 2.0 ** -90
    kk = k.reshape(-1, 1, d)
    paged.rope_append(kk, kk, kk, p.k, p.v, p.table, dev([s for s in p.slots for _ in range(page)]),
                      dev(list(range(page)) * 5), cos, sin, layer=0, index=idx)
    biggest = torch.finfo(torch.bfloat16).max
    for b in range(5):
        x = torch.nan_to_num(k[b, :, 0].float(), nan=0.0, posinf=biggest, neginf=-biggest)
        if b == 2:   # NaN-free: bounds over the rows with infinities as the largest values
            assert x.abs().max() == biggest
        assert torch.equal(idx[p.rows[b][0], 0, 0, :2 * d + 1], index_ref(x[None])[0]), b


# ---- bookkeeping ---------------------------------------------------------------------------------------------------

class Model:
    """The page table in Python."""

    def __init__(self, slots, cols, pages, page):
        self.t, self.n = [[] for _ in range(slots)], [0] * slots
        self.refs, self.cols, self.page = [0] * pages, cols, page

    def lowest(self, count):
        f = [p for p, r in enumerate(self.refs) if r == 0][:count]
        assert len(f) == count
        return f

    def reserve(self, slots, lens):
        for s, n in zip(slots, lens):
            more = -(-n // self.page) - len(self.t[s])
            got = self.lowest(more)
            for p in got:
                self.refs[p] = 1
            self.t[s] += got
            self.n[s] = n

    def fork(self, parents, children):
        """Returns the copies (source, destination, rows)."""
        moves = []
        for a, c in zip(parents, children):
            full, part = divmod(self.n[a], self.page)
            self.t[c] = self.t[a][:full]
            for p in self.t[c]:
                self.refs[p] += 1
            self.n[c] = self.n[a]
        for a, c in zip(parents, children):
            full, part = divmod(self.n[a], self.page)
            if part:
                d = self.lowest(1)[0]
                self.refs[d] = 1
                self.t[c].append(d)
                moves.append((self.t[a][full], d, part))
        return moves

    def free(self, slots):
        for s in slots:
            for p in self.t[s]:
                self.refs[p] -= 1
            self.t[s], self.n[s] = [], 0

    def same(self, cache):
        table = [r + [-1] * (self.cols - len(r)) for r in self.t]
        assert cache.page_table.tolist() == table
        assert cache.lengths.tolist() == self.n
        assert cache.refs.tolist() == self.refs


@pytest.mark.parametrize("page,pages,dtype,d", [(16, 300, torch.bfloat16, 64), (128, 41, torch.float16, 128)])
def test_pages_random_walk(paged, page, pages, dtype, d):
    import random
    r = random.Random(page)
    slots, cols = 13, 9
    cache = paged.PagedKVCache(pages, slots, cols, num_layers=2, num_kv_heads=2, head_dim=d, page_size=page, dtype=dtype)
    cache.k_pages.normal_()
    cache.v_pages.normal_()
    m = Model(slots, cols, pages, page)
    for step in range(60):
        empty = [s for s in range(slots) if m.n[s] == 0]
        used = [s for s in range(slots) if m.n[s]]
        free_now = m.refs.count(0)
        kind = r.choice(["reserve", "fork", "free"])
        if kind == "reserve":
            s = r.sample(range(slots), r.randint(1, 4))
            n = [min(cols * page, m.n[x] + r.choice([0, 1, page - 1, page, 2 * page + 3])) for x in s]
            if sum(-(-b // page) - len(m.t[x]) for x, b in zip(s, n)) > free_now:
                continue
            cache.reserve(s, n)
            m.reserve(s, n)
        elif kind == "fork" and used and empty:
            kids = r.sample(empty, r.randint(1, len(empty)))
            par = [r.choice(used) for _ in kids]
            if sum(1 for p in par if m.n[p] % page) > free_now:
                continue
            k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
            cache.fork(par, kids)
            for src, dst, rows in m.fork(par, kids):
                k0[dst, :, :, :rows] = k0[src, :, :, :rows]
                v0[dst, :, :, :rows] = v0[src, :, :, :rows]
            assert torch.equal(cache.k_pages, k0) and torch.equal(cache.v_pages, v0)
        elif kind == "free" and used:
            s = r.sample(used, r.randint(1, max(1, len(used) // 2)))
            cache.free(s)
            m.free(s)
        m.same(cache)
    cache.check()
    # gathered into another pool, smaller and larger
    live = [p for p, c in enumerate(m.refs) if c]
    for size in (max(1, len(live)), pages + 5):
        new = cache.compact(size)
        cache.check()
        assert new.refs.tolist() == [m.refs[p] for p in live] + [0] * (size - len(live))
        name = {p: i for i, p in enumerate(live)}
        assert new.page_table.tolist() == [[name[p] for p in row] + [-1] * (cols - len(row)) for row in m.t]
        ids = torch.tensor(live, device="cuda", dtype=torch.long)
        assert torch.equal(new.k_pages[:len(live)], cache.k_pages[ids])
        assert torch.equal(new.v_pages[:len(live)], cache.v_pages[ids])
        assert not new.k_pages[len(live):].any()


def test_copy_pages(paged):
    g = gen(3)
    k, v = normal(g, 9, 2, 3, 16, 64), normal(g, 9, 2, 3, 16, 64)
    # K and V side by side in one tensor, and an index
    both = torch.zeros(12, 2, 2, 3, 16, 64, dtype=torch.bfloat16, device="cuda")
    dk, dv = both[:, 0], both[:, 1]
    ix = torch.randint(-127, 127, (9, 2, 3, 144), dtype=torch.int8, device="cuda", generator=g)
    dx = torch.zeros(12, 2, 3, 144, dtype=torch.int8, device="cuda")
    paged.copy(k, v, dev([8, 0, 0]), dev([11, 2, 5]), dst_k_pages=dk, dst_v_pages=dv, index=ix, dst_index=dx)
    for s, d in ((8, 11), (0, 2), (0, 5)):
        assert torch.equal(dk[d], k[s]) and torch.equal(dv[d], v[s]) and torch.equal(dx[d], ix[s])
    assert not dk[[0, 1, 3, 4, 6, 7, 8, 9, 10]].any()
    k0 = k.clone()
    paged.copy(k, v, dev([1, 2]), dev([3, 4]))
    assert torch.equal(k[3], k0[1]) and torch.equal(k[4], k0[2]) and torch.equal(k[[0, 1, 2, 5, 6, 7, 8]], k0[[0, 1, 2, 5, 6, 7, 8]])
    status = dev([0])
    for src, dst in (([1, 2], [2, 3]), ([1, 2], [3, 3]), ([1, 9], [3, 4]), ([1], [-1])):
        k0 = k.clone()
        paged.copy(k, v, dev(src), dev(dst), status=status)
        assert status.item() == 9
        assert torch.equal(k, k0)
        status.zero_()


def test_host_lists_may_be_written_again(paged):
    """Lists and tensors of the host are read before the call returns, however far behind the GPU is."""
    cache = paged.PagedKVCache(10, 3, 8, num_layers=1, num_kv_heads=1, head_dim=64, page_size=16)
    for make in (torch.Tensor.clone, torch.Tensor.pin_memory):
        slots, lens = make(torch.tensor([0, 2], dtype=torch.int32)), make(torch.tensor([40, 17], dtype=torch.int32))
        torch.cuda._sleep(50_000_000)
        cache.reserve(slots, lens)
        slots[:], lens[:] = 1, 3
        cache.check()
        assert cache.lengths.tolist() == [40, 0, 17]
        cache.free([0, 2])


def test_compact_that_does_not_fit(paged):
    """Neither cache passes for sound, and the new one is empty; an error from before is the old cache's alone."""
    cache = paged.PagedKVCache(10, 3, 8, num_layers=1, num_kv_heads=1, head_dim=64, page_size=16)
    cache.reserve([0, 1], [40, 17])
    small = cache.compact(4)
    for c in (cache, small):
        with pytest.raises(RuntimeError, match="free pages"):
            c.check()
    assert not small.lengths.any() and small.free_pages() == 4
    small.reserve([2], [64])
    small.check()
    cache.reserve([1], [3])
    new = cache.compact(5)
    new.check()
    assert new.lengths.tolist() == [40, 17, 0] and new.free_pages() == 0
    with pytest.raises(RuntimeError, match="position"):
        cache.check()
    cache.check()


def test_copy_between_views(paged):
    """Pools that are views of one storage: a page that is read and written is found under both of its numbers, and
    pages past the smaller pool are no matter."""
    g = gen(4)
    k, v = normal(g, 4000, 1, 1, 16, 64), normal(g, 4000, 1, 1, 16, 64)
    ix = torch.randint(-127, 127, (4000, 1, 1, 144), dtype=torch.int8, device="cuda", generator=g)
    for lo, n, src, dst, ok in [
        (0, 4, [3999, 5, 2000], [1, 0, 3], True), (0, 4, [3, 9], [2, 3], False), (0, 40, [33], [33], False),
        (4, 3000, [4, 3999, 0], [1, 2, 2999], True), (4, 3000, [6, 7], [3, 9], False), (4, 3000, [0, 1, 2, 3], [3, 2, 1, 0], True),
        (3990, 10, [3994], [4], False), (3990, 10, [4, 3989], [4, 5], True), (3990, 10, [0], [10], False),
    ]:
        want, status = [x.clone() for x in (k, v, ix)], dev([0])
        if ok:
            for x in want:
                x[[lo + d for d in dst]] = x[src]
        cut = slice(lo, lo + n)
        paged.copy(k, v, dev(src), dev(dst), dst_k_pages=k[cut], dst_v_pages=v[cut], index=ix, dst_index=ix[cut], status=status)
        assert status.item() == (0 if ok else 9)
        assert all(torch.equal(a, b) for a, b in zip(want, (k, v, ix)))
        paged.copy(k[cut], v[cut], dev(dst), dev(src), dst_k_pages=k, dst_v_pages=v, status=status.zero_())
        assert status.item() == (0 if ok else 9)
    # pools that share memory in another way, and pages gathered into a view of their own pool
    with pytest.raises(RuntimeError, match="invalid argument"):
        paged.copy(k, v, dev([0]), dev([9]), dst_k_pages=k[1:3999], dst_v_pages=v[2:4000])
    with pytest.raises(RuntimeError, match="invalid argument"):
        paged.compact(k, v, dev([[0]]), dev([1] * 4000), k[5:9], v[5:9], dev([[0]]), dev([0] * 4))


def test_refused_tables_change_nothing(paged):
    page, d = 16, 64
    cache = paged.PagedKVCache(10, 6, 4, num_layers=1, num_kv_heads=1, head_dim=d, page_size=page)
    cache.reserve([0, 1], [40, 17])
    cache.check()
    before = [x.clone() for x in (cache.page_table, cache.lengths, cache.refs, cache.k_pages)]

    def same():
        return all(torch.equal(a, b) for a, b in zip(before, (cache.page_table, cache.lengths, cache.refs, cache.k_pages)))
    for call, what in [
        (lambda: cache.reserve([0, 0], [41, 41]), "slot"),
        (lambda: cache.reserve([6], [1]), "slot"),
        (lambda: cache.reserve([-1], [1]), "slot"),
        (lambda: cache.reserve([0], [39]), "position"),
        (lambda: cache.reserve([0], [65]), "position"),
        (lambda: cache.reserve([2, 3], [64, 64]), "free pages"),
        (lambda: cache.free([1, 1]), "slot"),
        (lambda: cache.free([9]), "slot"),
        (lambda: cache.fork([0], [1]), "slot"),
        (lambda: cache.fork([0, 1], [2, 2]), "slot"),
        (lambda: cache.fork([0, 2], [2, 3]), "slot"),
        (lambda: cache.fork([7], [2]), "slot"),
        (lambda: cache.fork([0], [-2]), "slot"),
    ]:
        call()
        with pytest.raises(RuntimeError, match=what):
            cache.check()
        assert same()
    cache.check()
    cache.reserve([2], [64])      # nine pages in use, one free
    cache.check()
    before = [x.clone() for x in (cache.page_table, cache.lengths, cache.refs, cache.k_pages)]
    cache.fork([0, 1], [3, 4])    # two part pages, one free page
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    assert same()
    small = cache.compact(4)
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    assert not small.refs.any() and (small.page_table == -1).all()
    # empty lists and empty parents
    cache.free([])
    cache.reserve([], [])
    cache.fork([], [])
    cache.fork([5], [4])
    cache.check()
    assert same()


def bad_rows(paged, run):
    """A cache whose slot 1 (40 full pages and a part) holds pages that are out of range or not in use; run(cache) may
    change nothing and leaves code 9."""
    page = 16
    for col, bad in ((0, -1), (0, 10 ** 6), (17, 80), (39, 75), (40, -5), (40, 76)):
        cache = paged.PagedKVCache(80, 6, 48, num_layers=1, num_kv_heads=1, head_dim=64, page_size=page)
        cache.reserve([0, 1], [20, 40 * page + 5])     # 2 + 41 pages; 43 and up are free
        cache.check()
        cache.page_table[1, col] = bad
        before = [x.clone() for x in (cache.page_table, cache.lengths, cache.refs, cache.k_pages)]
        run(cache)
        with pytest.raises(RuntimeError, match="page number"):
            cache.check()
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.page_table, cache.lengths, cache.refs, cache.k_pages))), (col, bad)


def test_fork_of_bad_rows_changes_nothing(paged):
    bad_rows(paged, lambda cache: cache.fork([0, 1, 1], [2, 3, 4]))


def test_free_of_bad_rows_changes_nothing(paged):
    bad_rows(paged, lambda cache: cache.free([0, 1]))


def test_free_of_many(paged):
    """Lists from one to several hundred sequences (more than one CTA), pages shared by all of them; a page held by more of
    the rows than its count says."""
    page, slots = 16, 400
    cache = paged.PagedKVCache(2000, slots, 40, num_layers=1, num_kv_heads=1, head_dim=64, page_size=page)
    for n in (1, 31, 32, 33, 64, 200, 399):
        cache.reserve([0], [30 * page + 3])
        kids = list(range(1, n + 1)) if n < slots - 1 else list(range(1, slots))
        cache.fork([0] * len(kids), kids)
        cache.reserve(kids[::2], [30 * page + 3 + 17 * (i % 5) for i in range(len(kids[::2]))])
        cache.check()
        before = [x.clone() for x in (cache.page_table, cache.lengths, cache.refs)]
        cache.refs[cache.page_table[0, 7].long()] = n      # n + 1 rows hold it
        cache.free([0] + kids)
        with pytest.raises(RuntimeError, match="page number"):
            cache.check()
        cache.refs[cache.page_table[0, 7].long()] = n + 1
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.page_table, cache.lengths, cache.refs)))
        cache.free([0] + kids)
        cache.check()
        assert (cache.page_table == -1).all() and not cache.lengths.any() and not cache.refs.any()


# ---- attention ---------------------------------------------------------------------------------------------------------

def check_attend(paged, p, hq, qlens, groups=None, prefix=None, layer=1, scale=None, q=None, std=2.0):
    """groups: sizes of the leading groups of sequences."""
    d, n = p.k.shape[4], sum(qlens)
    if q is None:
        q = normal(p.g, n, hq, d, dtype=p.dtype, std=std)
    starts = [0]
    for x in qlens:
        starts.append(starts[-1] + x)
    kw = {}
    if groups is not None:
        gs = [0]
        for x in groups:
            gs.append(gs[-1] + x)
        kw = {"group_starts": dev(gs), "prefix_pages": dev(prefix)}
    status = dev([0])
    out = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots[:len(qlens)]), layer=layer,
                       q_starts=None if all(x == 1 for x in qlens) else dev(starts), scale=scale, status=status, **kw)
    assert status.item() == 0
    sc = scale if scale is not None else 1.0 / math.sqrt(d)
    for b, x in enumerate(qlens):
        k, v = p.kv(b, layer)
        for i in range(x):
            pos = p.lens[b] - x + i
            seen = torch.arange(p.lens[b], device="cuda") <= pos
            ref = softmax_rows(q[starts[b] + i], k, v, seen, sc)
            close(out[starts[b] + i], ref, v.abs().max().item() if p.lens[b] else 0.0)
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", [(128, 16, 8, 2), (128, 64, 2, 5), (64, 32, 4, 1), (64, 128, 1, 8), (128, 128, 2, 17)])
def test_attend_single_tokens(paged, dtype, d, page, hkv, grp):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 129, 700]
    p = Pool(lens, page, hkv, d, dtype, seed=d + page)
    check_attend(paged, p, hkv * grp, [1] * len(lens))


@pytest.mark.parametrize("dtype,d,page,hkv,grp", [(torch.bfloat16, 128, 16, 2, 2), (torch.float16, 64, 64, 1, 3)])
def test_attend_several_tokens(paged, dtype, d, page, hkv, grp):
    # more query tokens than positions (rows that see nothing), none at all, a whole prompt
    p = Pool([5, 130, 40, 9, 0, 77, 33], page, hkv, d, dtype, seed=9)
    out = check_attend(paged, p, hkv * grp, [5, 3, 0, 12, 2, 77, 1])
    assert not out[8:11].any()     # the three tokens of sequence 3 that stand before its start


def test_attend_long(paged):
    p = Pool([20000], 64, 2, 128, torch.bfloat16, seed=2, layers=1)
    check_attend(paged, p, 4, [2], layer=0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", [(128, 16, 2, 2), (64, 64, 4, 3), (128, 32, 1, 8)])
@pytest.mark.parametrize("qlen", [1, 3])
@pytest.mark.parametrize("sizes,prefix", [([3], [4]), ([1, 9, 2], [2, 5, 3]), ([40], [7]), ([150], [2])])
def test_attend_shared_prefix(paged, dtype, d, page, hkv, grp, qlen, sizes, prefix):
    lens, share, b = [], {}, 0
    for n, pre in zip(sizes, prefix):
        for i in range(n):
            lens.append(pre * page + qlen + (b * 7) % 50)
            if i:
                share[b] = (b - i, pre)
            b += 1
    # two sequences that belong to no group
    lens += [33 + qlen, qlen]
    p = Pool(lens, page, hkv, d, dtype, seed=len(lens) + page, share=share)
    check_attend(paged, p, hkv * grp, [qlen] * len(lens), groups=sizes, prefix=prefix)


def test_attend_prefix_longer_than_a_member(paged):
    """A declared prefix that reaches past a member's first query token is read as far as all members see it."""
    page = 16
    lens = [5 * page + 3, 2 * page + 5, 4 * page]
    p = Pool(lens, page, 2, 128, torch.bfloat16, share={1: (0, 2), 2: (0, 3)}, seed=4)
    check_attend(paged, p, 4, [1, 1, 1], groups=[3], prefix=[2])
    check_attend(paged, p, 4, [2, 6, 1], groups=[3], prefix=[2])
    # all members share page 0 and 1; the third query token of sequence 1 stands on page 1
    check_attend(paged, p, 4, [1, 20, 1], groups=[3], prefix=[2])
    # members without query tokens, the leader among them
    check_attend(paged, p, 4, [0, 1, 1], groups=[3], prefix=[2])
    check_attend(paged, p, 4, [0, 0, 1], groups=[3], prefix=[2])


def test_attend_masked_infinities(paged):
    """What lies behind the mask does not matter: stale rows of the last page, and later tokens of the same step."""
    page = 16
    p = Pool([37, 50], page, 2, 128, torch.bfloat16, seed=8)
    q = normal(p.g, 8, 4, 128)
    clean = check_attend(paged, p, 4, [4, 4], q=q)
    for b, n in enumerate(p.lens):
        last = p.rows[b][-1]
        p.k[last, :, :, n % page:] = math.nan
        p.v[last, :, :, n % page:] = math.inf
    for bad in (math.inf, -math.inf, math.nan):
        p.v[p.rows[0][2], :, :, 4] = bad      # position 36: the last token's own row
        p.v[p.rows[1][3], :, :, 0] = bad      # position 48: seen by two of the four tokens
        kw = dict(layer=1, q_starts=dev([0, 4, 8]))
        out = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), **kw)
        assert torch.equal(out[:3], clean[:3]) and torch.equal(out[4:6], clean[4:6])
        assert not torch.isfinite(out[3]).any() and not torch.isfinite(out[6:8]).any()
    # scores of minus infinity everywhere but one position, and masked keys of minus infinity
    p = Pool([20], page, 1, 64, torch.float16, seed=8)
    p.k[p.rows[0][0], :, :, 1:] = -math.inf
    p.k[p.rows[0][1], :, :, :4] = -math.inf
    q = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    out = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=0)
    assert torch.equal(out[0, 0], p.v[p.rows[0][0], 0, 0, 0])


def test_attend_strided_and_layers(paged):
    """K and V side by side in one tensor, q a view of a wider row, more than one layer."""
    page, hkv, d = 32, 2, 64
    p = Pool([70, 33], page, hkv, d, torch.bfloat16, layers=3, seed=1)
    both = torch.stack([p.k, p.v], 1)
    wide = normal(p.g, 2, 4, 3, d)
    q = wide[:, :, 1]
    for layer in range(3):
        a = paged.attend(q, both[:, 0], both[:, 1], p.table, p.lengths, dev(p.slots), layer=layer)
        b = check_attend(paged, p, 4, [1, 1], layer=layer, q=q.contiguous())
        assert torch.equal(a, b)
    odd = torch.zeros(2, 4, d + 3, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:d + 1] = q
    assert torch.equal(paged.attend(odd[..., 1:d + 1], p.k, p.v, p.table, p.lengths, dev(p.slots), layer=2), b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.3])
@pytest.mark.parametrize("d,members", [(128, 40), (64, 2)])
def test_attend_scales(paged, dtype, scale, d, members):
    """Any sign and none: own parts alone, a shared prefix on the tensor cores (but for zero) and in the row kernel."""
    page, pages = 32, 5
    lens = [pages * page + 1 + 3 * b for b in range(members)] + [70]
    p = Pool(lens, page, 2, d, dtype, seed=members, share={b: (0, pages) for b in range(1, members)})
    q = normal(p.g, len(lens), 4, d, dtype=dtype, std=2.0)
    check_attend(paged, p, 4, [1] * len(lens), scale=scale, q=q)
    check_attend(paged, p, 4, [1] * len(lens), groups=[members], prefix=[pages], scale=scale, q=q)
    # every page selected: the same as reading everything
    idx = torch.zeros(p.k.shape[0], 2, 2, 2 * d + 16, dtype=torch.int8, device="cuda")
    want = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=1, scale=scale)
    out, _ = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(p.slots), dev([n - 1 for n in lens]), layer=1, top_k=40, scale=scale)
    # (twice check_attend's bound: both are rounded)
    tol = 2 * ROUND[dtype] * want.double().abs() + 2.0 ** -12 * p.v.abs().max().item()
    assert bool(((out.double() - want.double()).abs() <= tol).all())


@pytest.mark.parametrize("groups,members,grp", [(256, 3, 8), (257, 3, 8), (600, 3, 2), (1024, 2, 1)])
def test_attend_many_groups(paged, groups, members, grp):
    """Around the most groups of the tensor-core kernel, and the most sequences of a call (2048)."""
    page, d = 16, 64
    lens, share = [], {}
    for g in range(groups):
        for i in range(members):
            if i:
                share[len(lens)] = (len(lens) - i, 2)
            lens.append(2 * page + 1 + (7 * len(lens)) % 23)
    p = Pool(lens, page, 1, d, torch.bfloat16, layers=1, seed=groups, share=share)
    n = len(lens)
    q = normal(p.g, n, grp, d, std=2.0)
    status = dev([0])
    starts = torch.arange(0, n + 1, members, dtype=torch.int32, device="cuda")
    out = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=0, group_starts=starts, prefix_pages=dev([2] * groups),
                       status=status)
    assert status.item() == 0
    for b in list(range(0, n, 97)) + [n - 1]:
        k, v = p.kv(b, 0)
        close(out[b], softmax_rows(q[b], k, v, torch.ones(lens[b], dtype=torch.bool, device="cuda"), d ** -0.5), v.abs().max().item())
    # nothing declared shared: other sums, the same result within twice the bound
    flat = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=0)
    tol = 2 * ROUND[out.dtype] * flat.double().abs() + 2.0 ** -12 * p.v.abs().max().item()
    assert bool(((out.double() - flat.double()).abs() <= tol).all())


@pytest.mark.parametrize("d,page,hkv,grp", [(128, 64, 2, 2), (64, 16, 1, 5)])
def test_attend_prompts(paged, d, page, hkv, grp):
    """Whole prompts and a chunk behind a context, of many row tiles each, beside a single token."""
    p = Pool([1300, 1777, 513, 900], page, hkv, d, torch.bfloat16, layers=1, seed=d)
    check_attend(paged, p, hkv * grp, [1300, 700, 513, 1], layer=0)


def test_contiguous_q_at_odd_offsets(paged):
    """A contiguous q whose first element is on no 16-byte boundary, and one token whose strides are odd."""
    page, hkv, d = 16, 2, 64
    p = Pool([70, 33], page, hkv, d, torch.bfloat16, seed=1)
    idx = full_index(p, 2, hkv, d)
    q = normal(p.g, 2, 4, d)
    want = check_attend(paged, p, 4, [1, 1], q=q)
    pos, slots = dev([69, 32]), dev(p.slots)
    chosen, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, slots, pos, layer=1, top_k=3)
    flat = torch.zeros(q.numel() + 8, dtype=q.dtype, device="cuda")
    for lo in (1, 3, 4):
        x = flat[lo:lo + q.numel()].view(q.shape)
        x.copy_(q)
        assert x.is_contiguous() and x.data_ptr() % 16
        assert torch.equal(paged.attend(x, p.k, p.v, p.table, p.lengths, slots, layer=1), want)
        out = paged.sparse_attend(x, p.k, p.v, idx, p.table, slots, pos, layer=1, top_k=3)
        assert torch.equal(out[0], chosen) and torch.equal(out[1], sel)
    one = q[1:].as_strided((1, 4, d), (5 * d + 1, d, 1))
    assert torch.equal(paged.attend(one, p.k, p.v, p.table, p.lengths, slots[1:], layer=1), want[1:])


def test_attend_wrong_tables(paged):
    page = 16
    p = Pool([40, 20, 30], page, 1, 64, torch.bfloat16, seed=6)
    q = normal(p.g, 3, 1, 64)
    good = check_attend(paged, p, 1, [1, 1, 1], q=q)

    def call(**kw):
        status = dev([0])
        a = dict(page_table=p.table, lengths=p.lengths, slots=dev(p.slots), layer=1, status=status)
        a.update(kw)
        return paged.attend(q, p.k, p.v, a.pop("page_table"), a.pop("lengths"), a.pop("slots"), **a), status.item()
    out, code = call(slots=dev([p.slots[0], 99, p.slots[2]]))
    assert code == 8 and not out[1].any() and torch.equal(out[::2], good[::2])
    lengths = p.lengths.clone()
    lengths[p.slots[0]] = 10 ** 9
    out, code = call(lengths=lengths)
    assert code == 5 and not out[0].any() and torch.equal(out[1:], good[1:])
    table = p.table.clone()
    table[p.slots[2], 0] = 10 ** 6
    out, code = call(page_table=table)
    assert code == 9 and torch.equal(out[:2], good[:2])
    for starts in ([0, 2, 1, 3], [1, 1, 2, 3], [0, 1, 2, 2]):
        out, code = call(q_starts=dev(starts))
        assert code == 1 and not out.any()
    out, code = call(group_starts=dev([0, 9]), prefix_pages=dev([1]))
    assert code == 1 and not out.any()


@pytest.mark.parametrize("d,page,hkv,grp,members,pages", [(128, 16, 2, 2, 40, 21), (64, 64, 1, 4, 9, 5), (128, 128, 1, 8, 30, 3),
                                                          (64, 32, 2, 1, 3, 9)])
def test_attend_bad_shared_pages(paged, d, page, hkv, grp, members, pages):
    """A page out of range is left out: its positions count for no row, whichever kernel reads the prefix."""
    lens = [pages * page + 1 + 5 * b for b in range(members)]
    p = Pool(lens, page, hkv, d, torch.bfloat16, seed=pages, share={b: (0, pages) for b in range(1, members)})
    q = normal(p.g, members, hkv * grp, d, std=2.0)
    for bad in ([0], [pages - 1], [1, 2], list(range(pages))):
        table = p.table.clone()
        for i, col in enumerate(bad):
            table[:members + 1, col] = (-1, p.k.shape[0], 10 ** 9)[i % 3]
        for kw in ({}, dict(group_starts=dev([0, members]), prefix_pages=dev([pages]))):
            status = dev([0])
            out = paged.attend(q, p.k, p.v, table, p.lengths, dev(p.slots), layer=1, status=status, **kw)
            assert status.item() == 9
            for b in range(0, members, 4):
                k, v = p.kv(b, 1)
                seen = torch.ones(lens[b], dtype=torch.bool, device="cuda")
                for col in bad:
                    seen[col * page:(col + 1) * page] = False
                close(out[b], softmax_rows(q[b], k, v, seen, 1.0 / math.sqrt(d)), v.abs().max().item())


def test_attend_past_32_bits(paged):
    """Pages whose offsets in the pool pass 2^31 elements."""
    page, layers, hkv, d = 128, 28, 8, 128
    pages = 700            # 2.57e9 elements, 5.1 GB each
    k = torch.empty(pages, layers, hkv, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    g = gen(0)
    rows = [699, 3, 698]
    for r in rows:
        k[r].normal_(generator=g)
        v[r].normal_(generator=g)
    p = Pool([300], page, hkv, d, torch.bfloat16, seed=0)
    p.k, p.v, p.rows = k, v, [rows]
    p.table[p.slots[0], :3] = dev(rows)
    check_attend(paged, p, 16, [1], layer=27)
    p.lens = [290]
    kk = normal(g, 1, hkv, d)
    cos, sin = paged.rope_tables(400)
    paged.rope_append(normal(g, 1, 16, d), kk, kk, k, v, p.table, dev(p.slots), dev([290]), cos, sin, layer=27)
    assert torch.equal(v[698, 27, :, 290 - 256], kk[0])
    del k, v, p
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d,members,grp", [(128, 40, 2), (64, 12, 4)])
def test_steps_without_a_pause(paged, d, members, grp):
    """Reserve, append and attend (a shared prefix on the tensor cores, the own parts beside it) step after step with
    nothing between them: the same bits as with a synchronisation after every call."""
    page, hkv, layers, steps = 16, 2, 3, 50
    g = gen(d)
    cos, sin = paged.rope_tables(600, d)
    first = [normal(g, 200, (1 + i) * hkv, d) for i in (0, 0)]
    new = [[[normal(g, members, h, d) for h in (hkv * grp, hkv, hkv)] for _ in range(layers)] for _ in range(steps)]
    got = []
    for wait in (True, False):
        def pause():
            if wait:
                torch.cuda.synchronize()
        c = paged.PagedKVCache(13 + members * 6, members + 1, 20, num_layers=layers, num_kv_heads=hkv, head_dim=d, page_size=page)
        c.reserve([0], [200])
        for layer in range(layers):
            c.append(layer, first[0], first[0], first[1], dev([0] * 200), dev(list(range(200))), cos, sin)
        kids = list(range(1, members + 1))
        c.fork([0] * members, kids)
        slots, gs, pp, one = dev(kids), dev([0, members]), dev([12]), dev([1] * members)
        torch.cuda.synchronize()
        outs = []
        for step in range(steps):
            pos = c.lengths[slots]
            pause()
            c.reserve(slots, pos + one)
            pause()
            for layer in range(layers):
                q, k, v = new[step][layer]
                q = c.append(layer, q, k, v, slots, pos, cos, sin)
                pause()
                outs.append(c.attend(layer, q, slots, group_starts=gs, prefix_pages=pp))
                pause()
        c.check()
        got.append(torch.stack(outs))
    assert torch.equal(*got)


def test_other_stream_and_graph(paged):
    p = Pool([500, 300], 64, 2, 128, torch.bfloat16, seed=3)
    q = normal(p.g, 2, 4, 128)
    slots = dev(p.slots)
    want = paged.attend(q, p.k, p.v, p.table, p.lengths, slots, layer=0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged.attend(q, p.k, p.v, p.table, p.lengths, slots, layer=0)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged.attend(q, p.k, p.v, p.table, p.lengths, slots, layer=0)
    q.mul_(0.5)
    p.lengths.sub_(1)      # the lengths are read on the device: a replay follows them
    graph.replay()
    assert torch.equal(got, paged.attend(q, p.k, p.v, p.table, p.lengths, slots, layer=0))
    assert not torch.equal(got, want)


# ---- sparse attention ------------------------------------------------------------------------------------------------------

def select_ref(q, index, row, own, top_k, d):
    """q [grp, d] of one token and kv head; index records [pages, 2 d + 16]: the selected places."""
    if own <= top_k - 1:
        got = list(range(own + 1))
    else:
        best = None
        rec = index[torch.tensor(row[:own], dtype=torch.long, device=index.device)].double()
        units = torch.tensor([2.0 ** i for i in range(-60, 41)], dtype=torch.float64, device=index.device)
        for x in q.double():
            a = x.abs().max()
            e = int((torch.frexp(a).exponent - 7).clamp(-60, 40)) if a > 0 else 0
            w = torch.round(x / 2.0 ** e).clamp(-127, 127)
            s = torch.where(w > 0, w * rec[:, :d], w * rec[:, d:2 * d]).sum(1) * 2.0 ** e
            best = s if best is None else torch.maximum(best, s)
        best = best * units[rec[:, 2 * d].long() + 60]
        order = sorted(range(own), key=lambda j: (-best[j].item(), j))
        got = sorted(order[:top_k - 1]) + [own]
    return got + [-1] * (top_k - len(got))


def check_sparse(paged, p, hq, index, slots, positions, seqs, top_k, q=None, layer=1):
    d, page, hkv = p.k.shape[4], p.page, p.k.shape[2]
    n = len(positions)
    if q is None:
        q = normal(p.g, n, hq, d, dtype=p.dtype, std=1.5)
    status = dev([0])
    out, sel = paged.sparse_attend(q, p.k, p.v, index, p.table, dev(slots), dev(positions), layer=layer, top_k=top_k,
                                   status=status)
    assert status.item() == 0
    grp = hq // hkv
    for i in range(n):
        k, v = p.kv(seqs[i], layer)
        own = positions[i] // page
        seen = torch.zeros(hkv, p.lens[seqs[i]], dtype=torch.bool, device="cuda")
        for h in range(hkv):
            want = select_ref(q[i, h * grp:(h + 1) * grp], index[:, layer, h], p.rows[seqs[i]], own, top_k, d)
            assert sel[i, h].tolist() == want, (i, h)
            for j in want:
                if j >= 0:
                    seen[h, j * page:(j + 1) * page] = True
        seen[:, positions[i] + 1:] = False
        close(out[i], softmax_rows(q[i], k, v, seen, 1.0 / math.sqrt(d)), v.abs().max().item())


def full_index(p, layers, hkv, d):
    idx = torch.zeros(p.k.shape[0], layers, hkv, 2 * d + 16, dtype=torch.int8, device="cuda")
    for x in range(layers):
        for h in range(hkv):
            idx[:, x, h, :2 * d + 1] = index_ref(p.k[:, x, h])
    return idx


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp,top_k", [(128, 16, 8, 2, 4), (64, 32, 2, 5, 7), (128, 64, 1, 8, 1), (64, 128, 4, 1, 2),
                                                  (128, 16, 1, 20, 9)])
def test_sparse(paged, dtype, d, page, hkv, grp, top_k):
    lens = [1, page, page + 1, 7 * page - 1, 1500]
    p = Pool(lens, page, hkv, d, dtype, seed=d + top_k)
    p.k += normal(p.g, p.k.shape[0], 2, hkv, 1, d, dtype=dtype, std=0.5)
    idx = full_index(p, 2, hkv, d)
    # decode: the last position of each; and several tokens of one sequence
    check_sparse(paged, p, hkv * grp, idx, p.slots, [n - 1 for n in lens], list(range(5)), top_k)
    pos = [0, 15, 16, 700, 701, 1023, 1499]
    check_sparse(paged, p, hkv * grp, idx, [p.slots[4]] * 7, pos, [4] * 7, top_k)


@pytest.mark.parametrize("dtype,d,grp", [(torch.bfloat16, 64, 2), (torch.float16, 128, 1), (torch.bfloat16, 64, 9)])
def test_sparse_many_tokens(paged, dtype, d, grp):
    """Enough tokens for eight to a CTA: runs of one sequence, sequences taking turns, a count that is no multiple of
    eight, tokens with nothing to choose among them."""
    page, hkv, top_k = 16, 8, 4
    lens = [900, 300, 40]
    p = Pool(lens, page, hkv, d, dtype, seed=grp)
    idx = full_index(p, 2, hkv, d)
    seqs = [0] * 90 + [i % 3 for i in range(40)] + [1] * 25
    pos = [(i * 131) % lens[s] for i, s in enumerate(seqs)]
    check_sparse(paged, p, hkv * grp, idx, [p.slots[s] for s in seqs], pos, seqs, top_k)


def test_sparse_long_table(paged):
    """More pages than one CTA scores: a cluster per item, and keys all in one bin (pages in few kinds)."""
    page, d = 16, 64
    p = Pool([16 * 3000 - 5], page, 1, d, torch.bfloat16, seed=7)
    idx = full_index(p, 2, 1, d)
    check_sparse(paged, p, 2, idx, p.slots, [16 * 3000 - 6], [0], 40)
    p.k[:] = p.k[:7].repeat(p.k.shape[0] // 7 + 1, 1, 1, 1, 1)[:p.k.shape[0]]
    idx = full_index(p, 2, 1, d)
    check_sparse(paged, p, 2, idx, p.slots, [16 * 3000 - 6], [0], 500)


def test_sparse_ties(paged):
    """Equal scores: the lowest pages win; zero queries make every score equal."""
    page, d = 16, 64
    p = Pool([40 * page], page, 1, d, torch.bfloat16, seed=1)
    p.k[:] = p.k[:1]       # all pages alike
    idx = full_index(p, 2, 1, d)
    check_sparse(paged, p, 2, idx, p.slots, [40 * page - 1], [0], 6)
    p.k.normal_()
    idx = full_index(p, 2, 1, d)
    check_sparse(paged, p, 2, idx, p.slots, [40 * page - 3], [0], 6,
                 q=torch.zeros(1, 2, d, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("pages,n,hkv", [(40, 140, 8), (3, 140, 8), (600, 70, 8), (3000, 2, 4)])
def test_sparse_ties_everywhere(paged, pages, n, hkv):
    """All keys of every item equal (queries of zeros), many items to a call and many calls: most warps of an item have
    no pages, and none may go ahead of another's reads.  One CTA to an item, and clusters (3000 pages)."""
    page, d, top_k = 16, 64, min(6, pages - 1)
    p = Pool([pages * page], page, hkv, d, torch.bfloat16, seed=1)
    idx = torch.randint(-127, 128, (p.k.shape[0], 2, hkv, 2 * d + 16), dtype=torch.int8, device="cuda", generator=p.g)
    idx[..., 2 * d] = 0
    q = torch.zeros(n, hkv, d, dtype=torch.bfloat16, device="cuda")
    kw = dict(layer=1, top_k=top_k)
    args = (q, p.k, p.v, idx, p.table, dev(p.slots * n), dev([pages * page - 1] * n))
    want = dev(list(range(top_k - 1)) + [pages - 1]).expand(n, hkv, top_k)
    for _ in range(100):
        assert torch.equal(paged.sparse_attend(*args, **kw)[1], want)


@pytest.mark.parametrize("dtype,d,page,grp,top_k", [(torch.bfloat16, 128, 32, 2, 5), (torch.float16, 64, 64, 3, 3), (torch.bfloat16, 64, 128, 8, 2),
                                                    (torch.float16, 128, 16, 1, 1)])
def test_sparse_by_page(paged, dtype, d, page, grp, top_k):
    """More tokens than slots, pages that are large beside their parts: a page is read once for all tokens that chose
    it.  Pages chosen by one token and by scores of them, tokens with fewer pages than top_k, q with strides."""
    hkv = 8
    lens = [12 * page + 3, 5 * page, page - 3]
    p = Pool(lens, page, hkv, d, dtype, seed=grp)
    idx = full_index(p, 2, hkv, d)
    seqs = [0] * 100 + [i % 3 for i in range(30)] + [1] * 25
    pos = [(i * 37) % lens[s] for i, s in enumerate(seqs)]
    q = normal(p.g, len(seqs), hkv * grp + 2, d + 8, dtype=dtype, std=1.5)[:, 1:-1, :d]
    check_sparse(paged, p, hkv * grp, idx, [p.slots[s] for s in seqs], pos, seqs, top_k, q=q)


def test_sparse_by_page_bad_values(paged):
    """Infinities and NaN where no token of the call looks, and beside tokens that do not see them; wrong places; pages
    out of range.  Rows must not depend on which others share their page, so two calls agree in every bit."""
    page, hkv, grp, d, n = 64, 8, 2, 128, 160
    p = Pool([640, 200], page, hkv, d, torch.bfloat16, seed=3)
    idx = full_index(p, 2, hkv, d)
    slots = [p.slots[0]] * (n - 20) + [p.slots[1]] * 20
    seqs = [0] * (n - 20) + [1] * 20
    pos = [(i * 7) % 600 for i in range(n - 20)] + [180 + i % 20 for i in range(20)]
    q = normal(p.g, n, hkv * grp, d, std=1.5)
    kw = dict(layer=1, top_k=4)
    ref, want = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(slots), dev(pos), **kw)
    # positions 600 .. 639 of sequence 0 and 200 .. 255 of sequence 1 are seen by no token
    for row, at in ((p.rows[0][9], 24), (p.rows[1][3], 8)):
        p.k[row, :, :, at:] = math.nan
        p.v[row, :, :, at:] = math.inf
    out, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(slots), dev(pos), **kw)
    assert torch.equal(sel, want)
    close(out, ref.double(), p.v[:, 1].float().nan_to_num(posinf=0).abs().max().item())
    # an infinity in the middle of a page reaches the tokens behind it alone
    p.v[p.rows[0][9], 1, :, 10, 5] = math.inf
    out, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(slots), dev(pos), **kw)
    sees = dev([s == 0 and x >= 9 * page + 10 for s, x in zip(seqs, pos)]).bool()
    assert sees.any() and not torch.isfinite(out[sees][:, :, 5]).any()
    rest = out.clone()
    rest[sees, :, 5] = 0
    assert torch.isfinite(rest).all()
    same = ref.clone()
    same[sees, :, 5] = 0
    close(rest, same.double(), p.v[:, 1].float().nan_to_num(posinf=0).abs().max().item())
    bits = out.view(torch.int16)   # (a NaN is not equal to itself)
    for _ in range(5):
        assert torch.equal(paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(slots), dev(pos), **kw)[0].view(torch.int16), bits)
    # wrong places: zeros there, the others as before
    for i, slot, x, code in ((3, 99, 5, 8), (70, p.slots[0], -1, 5), (159, p.slots[1], 10 ** 9, 5)):
        s2, p2, status = list(slots), list(pos), dev([0])
        s2[i], p2[i] = slot, x
        got, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(s2), dev(p2), status=status, **kw)
        assert status.item() == code and not got[i].any() and (sel[i] == -1).all()
        keep = torch.arange(n, device="cuda") != i
        assert torch.equal(got[keep].view(torch.int16), bits[keep])
    table, status = p.table.clone(), dev([0])
    table[p.slots[1], 3] = p.k.shape[0]
    got, _ = paged.sparse_attend(q, p.k, p.v, idx, table, dev(slots), dev(pos), status=status, **kw)
    assert status.item() == 9 and torch.isfinite(got[n - 20:]).all() and torch.equal(got[:n - 20].view(torch.int16), bits[:n - 20])


def test_sparse_by_page_rounds(paged):
    """So many choices to a token that its parts do not all fit at once: the same as a few tokens at a time."""
    page, hkv, d, top_k, n = 16, 8, 64, 300, 470
    p = Pool([340 * page, 40 * page], page, hkv, d, torch.bfloat16, seed=9)
    idx = torch.zeros(p.k.shape[0], 2, hkv, 2 * d + 16, dtype=torch.int8, device="cuda")
    idx[:, 1, :, :2 * d + 1] = torch.stack([index_ref(p.k[:, 1, h]) for h in range(hkv)], 1)
    slots = dev([p.slots[i % 7 == 0] for i in range(n)])
    pos = dev([40 * page - 1 - i % 50 if i % 7 == 0 else 340 * page - 1 - i for i in range(n)])
    q = normal(p.g, n, hkv, d, std=1.5)
    out, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, slots, pos, layer=1, top_k=top_k)
    for i in range(0, n, 47):
        ref, want = paged.sparse_attend(q[i:i + 47], p.k, p.v, idx, p.table, slots[i:i + 47], pos[i:i + 47], layer=1, top_k=top_k)
        assert torch.equal(sel[i:i + 47], want)
        close(out[i:i + 47], ref.double(), p.v.abs().max().item())


def test_sparse_all_pages_is_full_attention(paged):
    p = Pool([333], 32, 2, 128, torch.float16, seed=5)
    idx = torch.zeros(p.k.shape[0], 2, 2, 272, dtype=torch.int8, device="cuda")
    q = normal(p.g, 1, 6, 128, dtype=torch.float16)
    out, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(p.slots), dev([332]), layer=1, top_k=40)
    ref = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=1)
    assert sel[0, 0].tolist() == list(range(11)) + [-1] * 29
    close(out, ref.double(), p.v.abs().max().item())


def test_sparse_wrong_places(paged):
    p = Pool([100, 50], 16, 1, 64, torch.bfloat16, seed=5)
    idx = full_index(p, 2, 1, 64)
    q = normal(p.g, 3, 1, 64)
    for slots, pos, code in (([p.slots[0], 77, p.slots[1]], [99, 3, 49], 8), ([p.slots[0], p.slots[0], p.slots[1]], [99, -1, 49], 5),
                             ([p.slots[0], p.slots[0], p.slots[1]], [99, 10 ** 9, 49], 5)):
        status = dev([0])
        out, sel = paged.sparse_attend(q, p.k, p.v, idx, p.table, dev(slots), dev(pos), layer=1, top_k=3, status=status)
        assert status.item() == code and not out[1].any() and (sel[1] == -1).all()
        assert out[0].any() and out[2].any()


# ---- arguments that are wrong on the host -----------------------------------------------------------------------------------

def test_refusals(paged):
    p = Pool([40, 20], 16, 2, 64, torch.bfloat16)
    q = normal(p.g, 2, 4, 64)
    idx = full_index(p, 2, 2, 64)
    slots, pos = dev(p.slots), dev([39, 19])
    cos, sin = paged.rope_tables(64, 64)

    def attend(q=q, k=p.k, v=p.v, table=p.table, lengths=p.lengths, slots=slots, layer=0, **kw):
        return paged.attend(q, k, v, table, lengths, slots, layer=layer, **kw)

    def sparse(q=q, index=idx, pos=pos, layer=0, top_k=2):
        return paged.sparse_attend(q, p.k, p.v, index, p.table, slots, pos, layer=layer, top_k=top_k)

    def append(q=q, k=q[:, :2], v=q[:, 2:], cos=cos, sin=sin, layer=0, positions=pos, **kw):
        return paged.rope_append(q, k, v, p.k, p.v, p.table, slots, positions, cos, sin, layer=layer, **kw)
    attend(), sparse(), append()
    bad = [
        lambda: attend(q=q.float()), lambda: attend(q=q.half()), lambda: attend(q=q[:, :3]), lambda: attend(q=q[0]),
        lambda: attend(q=q[:1]), lambda: attend(layer=2), lambda: attend(layer=-1), lambda: attend(k=p.k.float()),
        lambda: attend(v=p.v[:, :1]), lambda: attend(k=p.k.transpose(3, 4)), lambda: attend(table=p.table.long()),
        lambda: attend(table=p.table.cpu()), lambda: attend(lengths=p.lengths[:1]), lambda: attend(slots=slots.long()),
        lambda: attend(q=q.cpu()), lambda: attend(k=p.k.cpu(), v=p.v.cpu()), lambda: attend(q_starts=dev([0, 1])),
        lambda: attend(group_starts=dev([0, 2])), lambda: attend(group_starts=dev([0, 2]), prefix_pages=dev([1, 1])),
        lambda: attend(k=p.k[:, :, :, :8].contiguous(), v=p.v[:, :, :, :8].contiguous()),
        lambda: sparse(top_k=0), lambda: sparse(index=idx[..., :64]), lambda: sparse(index=idx.int()),
        lambda: sparse(pos=pos[:1]), lambda: sparse(layer=5), lambda: sparse(q=q[:, :1]),
        lambda: append(k=q[:, :3]), lambda: append(cos=cos.half(), sin=sin.half()), lambda: append(cos=cos[:, :3]),
        lambda: append(positions=pos[:1]), lambda: append(layer=9), lambda: append(q=q[..., :32]),
        lambda: append(index=idx[:1]), lambda: paged.rope(q[..., :48], pos, cos, sin),
        lambda: paged.rope(q, pos, *paged.rope_tables(64, 128)), lambda: paged.rope(q.cpu(), pos, cos, sin),
        lambda: paged.fork(p.k, p.v, p.table, p.lengths, dev([0]), dev([0]), dev([1])),
        lambda: paged.free(p.table, p.lengths, dev([0] * 9), dev([0] * 99), 16),
        lambda: paged.free(p.table, p.lengths, dev([0] * 9), dev([0]), 17),
        lambda: paged.compact(p.k, p.v, p.table, dev([0] * p.k.shape[0]), p.k, p.v, p.table.clone(), dev([0] * p.k.shape[0])),
        lambda: paged.copy(p.k, p.v, dev([0]), dev([1, 2])),
        lambda: paged.copy(p.k, p.v, dev([0]), dev([1]), dst_k_pages=p.k),
        lambda: paged.copy(p.k, p.v, dev([0]), dev([1]), dst_k_pages=p.k[:, :1], dst_v_pages=p.v[:, :1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"case {i} was accepted")
    # nothing to do is not an error
    assert attend(q=q[:0], slots=slots[:0]).shape == (0, 4, 64)
    assert paged.rope(q[:0], pos[:0], cos, sin).shape == (0, 4, 64)


def test_append_wrong_places(paged):
    p = Pool([40, 20], 16, 2, 64, torch.bfloat16)
    q = normal(p.g, 3, 4, 64)
    cos, sin = paged.rope_tables(64, 64)
    for slots, pos, code in (([p.slots[0], 99, p.slots[1]], [39, 3, 19], 8), ([p.slots[0], p.slots[1], p.slots[1]], [39, 64, 19], 5),
                             ([p.slots[0], p.slots[1], p.slots[1]], [39, -1, 19], 5),
                             ([p.slots[0], p.slots[1], p.slots[1]], [39, 40, 19], 9)):
        k0 = p.k.clone()
        status = dev([0])
        out = paged.rope_append(q, q[:, :2], q[:, 2:], p.k, p.v, p.table, dev(slots), dev(pos), cos, sin, layer=0, status=status)
        assert status.item() == code
        assert out[0].any() and out[2].any()
        touched = {(p.rows[0][2], 7), (p.rows[1][1], 3)}
        diff = (p.k != k0).any(dim=(1, 2, 4)).nonzero().tolist()
        assert {tuple(x) for x in diff} <= touched
