"""accept: the walk, the rows that move, lengths, pages and index against a Python model of it, exactly."""
from __future__ import annotations

import pytest
import torch

from test_paged_gpu import dev, gen, normal
from test_paged_span_gpu import random_tree, starts_of

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


def walk(parents, tokens, chosen):
    path = [0] if parents else []
    while path:
        kids = [i for i, up in enumerate(parents) if up == path[-1] and tokens[i] == chosen[path[-1]]]
        if not kids:
            break
        path.append(kids[0])
    return path


class Model:
    """A cache with sequences that end in drafted trees, and what is expected of it."""

    def __init__(self, paged, lens, trees, page, dtype=torch.bfloat16, layers=3, hkv=2, d=64, seed=0, index=False, right=0.7):
        g, self.gc = gen(seed), torch.Generator().manual_seed(seed)
        pages = sum(-(-(n + len(t)) // page) for n, t in zip(lens, trees)) + 5
        self.cache = c = paged.PagedKVCache(pages, len(lens) + 2, max(-(-(n + len(t)) // page) for n, t in zip(lens, trees)) + 1,
                                            num_layers=layers, num_kv_heads=hkv, head_dim=d, page_size=page, dtype=dtype, index=index)
        self.slots = torch.randperm(len(lens) + 2, generator=self.gc)[:len(lens)].tolist()
        # interleaved growth, so that pages lie mixed
        c.reserve(self.slots, [n // 2 for n in lens])
        c.reserve(self.slots, [n + len(t) for n, t in zip(lens, trees)])
        c.k_pages.copy_(normal(g, *c.k_pages.shape, dtype=dtype))
        c.v_pages.copy_(normal(g, *c.v_pages.shape, dtype=dtype))
        self.lens, self.trees = lens, trees
        # chosen tokens that follow the drafted ones some of the way; the same token among several children
        self.tokens, self.chosen = [], []
        for t in trees:
            tok = torch.randint(0, 4, (len(t),), generator=self.gc).tolist()
            ch = torch.randint(0, 4, (len(t),), generator=self.gc).tolist()
            for i in range(len(t)):
                kids = [j for j, up in enumerate(t) if up == i]
                if kids and torch.rand(1, generator=self.gc).item() < right:
                    ch[i] = tok[kids[int(torch.randint(0, len(kids), (1,), generator=self.gc))]]
            self.tokens.append(tok)
            self.chosen.append(ch)
        self.starts = starts_of([len(t) for t in trees])

    def args(self):
        return (self.slots, sum(self.trees, []), sum(self.tokens, []), sum(self.chosen, []), self.starts)

    def state(self):
        c = self.cache
        out = [c.k_pages, c.v_pages, c.page_table, c.lengths, c.refs]
        return [x.clone() for x in out + ([c.index] if c.index is not None else [])]

    def expect(self):
        """(path, emitted, count), and the state after the call."""
        c, page = self.cache, self.cache.page_size
        k, v, table, lengths, refs = self.state()[:5]
        path, emitted, count = [], [], []
        for s, n, t, tok, ch in zip(self.slots, self.lens, self.trees, self.tokens, self.chosen):
            p = walk(t, tok, ch)
            path += p + [-1] * (len(t) - len(p))
            emitted += [ch[i] for i in p] + [-1] * (len(t) - len(p))
            count.append(len(p))
            row = table[s].tolist()
            for x in (k, v):
                rows = [x[row[(n + i) // page], :, :, (n + i) % page].clone() for i in p]
                for i, r in enumerate(rows):
                    x[row[(n + i) // page], :, :, (n + i) % page] = r
            for col in range(-(-(n + len(p)) // page), -(-(n + len(t)) // page)):
                refs[row[col]] -= 1
                table[s, col] = -1
            lengths[s] = n + len(p)
        return (path, emitted, count), [k, v, table, lengths, refs]


def check(m):
    (path, emitted, count), state = m.expect()
    got = m.cache.accept(*m.args())
    m.cache.check()
    assert all(x.dtype == torch.int32 for x in got)
    assert got[0].tolist() == path and got[1].tolist() == emitted and got[2].tolist() == count
    for a, b in zip(m.state(), state):
        assert torch.equal(a, b)
    return count


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("layers,hkv", [(1, 1), (6, 3)])
def test_accept(paged, dtype, d, page, layers, hkv):
    sizes = [1, 7, 16, 40, 64, 0, 256, 33]
    lens = [0, 5, 15, 100, 64, 30, 17, 127]
    for seed in range(3):
        trees = [random_tree(seed * 10 + i, n, back=4, roots=0.05) for i, n in enumerate(sizes)]
        count = check(Model(paged, lens, trees, page, dtype, layers, hkv, d, seed))
        assert max(count) > 2


@pytest.mark.parametrize("page", [16, 32])
def test_accept_long_paths(paged, page):
    """Chains that are right all the way, in place and every second node: batches of rows that overlap."""
    n = 200
    chain = [i - 1 for i in range(n)]
    second = [-1] + [i - 1 if i % 2 else i - 2 for i in range(1, n)]   # even nodes a chain, an odd leaf on each
    deep = [-1] + [max(0, i - 3) for i in range(1, n)]
    m = Model(paged, [3, 50, 16], [chain, second, deep], page, layers=5)
    for t, tok, ch in zip(m.trees, m.tokens, m.chosen):
        for i in range(n):
            tok[i] = i
            kids = [j for j in range(n) if t[j] == i]
            ch[i] = kids[-1] if kids else -5
    assert check(m)[0] == n


def test_accept_many_sequences(paged):
    lens = [(i * 13) % 50 for i in range(300)]
    trees = [random_tree(i, i % 20, back=3) for i in range(300)]
    check(Model(paged, lens, trees, 16, layers=2, hkv=1, seed=5))


def test_accept_one_node_each(paged):
    m = Model(paged, [5, 16, 0], [[-1]] * 3, 16)
    slots, parents, tokens, chosen, _ = m.args()
    path, emitted, count = m.cache.accept(slots, parents, tokens, chosen)
    m.cache.check()
    assert path.tolist() == [0, 0, 0] and emitted.tolist() == chosen and count.tolist() == [1, 1, 1]
    assert [m.cache.lengths[s].item() for s in slots] == [6, 17, 1]


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_accept_keeps_the_index(paged, dtype, d):
    """The records of full pages are those of the keys that are there then."""
    from test_paged_gpu import index_ref
    m = Model(paged, [10, 40, 31], [random_tree(i, 60, back=3) for i in range(3)], 16, dtype, d=d, index=True, right=0.95, seed=2)
    count = check_index_free(m)
    full = 0
    for s, n, k in zip(m.slots, m.lens, count):
        row = m.cache.page_table[s].tolist()
        for c in range(n // 16, (n + k) // 16):
            ref = torch.stack([index_ref(x) for x in m.cache.k_pages[row[c]]])   # of [layers, heads, page, d]
            assert torch.equal(m.cache.index[row[c], :, :, :2 * d + 1], ref)
            full += 1
    assert full


def check_index_free(m):
    (path, _, count), state = m.expect()
    got = m.cache.accept(*m.args())
    m.cache.check()
    assert got[0].tolist() == path
    for a, b in zip(m.state()[:5], state):
        assert torch.equal(a, b)
    return count


def refused(m, code, change, args=None):
    """A call that changes nothing but its outputs."""
    c = m.cache
    change(c)
    before = m.state()
    path, emitted, count = c.accept(*(args or m.args()))
    assert bool((path == -1).all()) and bool((emitted == -1).all()) and not bool(count.any())
    assert c.status.item() == code
    for a, b in zip(before, m.state()):
        assert torch.equal(a, b)


def test_wrong_calls_change_nothing(paged):
    def model():
        m = Model(paged, [20, 40, 7], [random_tree(i, 40, back=3) for i in range(3)], 16, seed=4)
        m.chosen[0] = [99] * 40   # only the root: its pages are given back
        return m

    def setter(name, *at):
        def change(c):
            getattr(c, name)[at[:-1]] = at[-1]
        return change

    m = model()
    slots, parents, tokens, chosen, starts = m.args()
    none = lambda c: None   # noqa: E731
    for bad in ([slots[0], slots[1], slots[0]], [slots[0], -1, slots[2]], [slots[0], slots[1], 5]):
        refused(model(), 8, none, (bad, parents, tokens, chosen, starts))
    for bad in ([0, 40, 30, 120], [1, 40, 80, 120], [0, 40, 80, 119]):
        refused(model(), 1, none, (slots, parents, tokens, chosen, bad))
    for at, up in ((0, 0), (45, 5), (85, 200), (100, -2)):
        wrong = list(parents)
        wrong[at] = up
        refused(model(), 1, none, (slots, wrong, tokens, chosen, starts))
    refused(model(), 5, setter("lengths", slots[1], 39))
    refused(model(), 5, setter("lengths", slots[1], -1))
    refused(model(), 5, setter("lengths", slots[1], 10 ** 9))
    for page in (-1, 10 ** 6):
        refused(model(), 9, setter("page_table", slots[0], 3, page))    # given back
    # a page that a row moves to: out of range, or with another holder
    for seed in range(20):
        m = Model(paged, [20, 40, 7], [random_tree(i, 40, back=3) for i in range(3)], 16, seed=seed, right=0.95)
        p = walk(m.trees[1], m.tokens[1], m.chosen[1])
        if any(i != k for k, i in enumerate(p)):
            break
    k = next(k for k, i in enumerate(p) if i != k)
    col = (40 + k) // 16
    page = m.cache.page_table[m.slots[1], col].item()
    refused(m, 9, lambda c: c.refs.__setitem__(page, 2))
    m.cache.refs[page] = 1
    m.cache.status.zero_()
    refused(m, 9, setter("page_table", m.slots[1], col, -3))
    # a count that is not there to take
    m = model()
    page = m.cache.page_table[m.slots[0], 3].item()
    refused(m, 9, lambda c: c.refs.__setitem__(page, 0))


def test_refused_calls_leave_the_index(paged):
    """What a call finds in its workspace (places of full pages, here) must not reach the index when it is refused."""
    trees = [random_tree(i, 20, back=3) for i in range(18)]
    m = Model(paged, [40] * 18, trees, 16, layers=2, index=True, seed=5)
    m.cache.index.fill_(99)
    slots, parents, tokens, chosen, starts = m.args()
    wrong = list(parents)
    wrong[7] = 9
    for args, code in (((slots, wrong, tokens, chosen, starts), 1), (([*slots[:-1], slots[0]], parents, tokens, chosen, starts), 8)):
        left = [torch.full((len(parents) * 6 + 64,), 15, dtype=torch.int32, device="cuda") for _ in range(4)]
        del left   # 15: a slot, and the last row of a page
        refused(m, code, lambda c: None, args)
        m.cache.status.zero_()


def test_a_written_page_given_back_by_another(paged):
    """Two sequences that share the pages of their trees: neither may write there, whatever the other gives back."""
    page, n = 16, 48
    for chosen_of_other in (5, 99):
        c = paged.PagedKVCache(12, 3, 6, num_layers=1, num_kv_heads=1, head_dim=64, page_size=page)
        c.reserve([0], [page + n])
        c.k_pages.normal_()
        c.fork([0], [1])
        before = [x.clone() for x in (c.k_pages, c.v_pages, c.page_table, c.lengths, c.refs)]
        # the first takes its second branch, of 40 nodes behind 7 others; the other one all or only its root
        parents = [-1, 0, 1, 2, 3, 4, 5, 6] + [0] + list(range(8, 47))
        tokens = [0] + [1] * 7 + [2] + [3] * 39
        chosen = [2] + [9] * 7 + [3] * 39 + [4]
        other = [chosen_of_other] * n
        path, emitted, count = c.accept([0, 1], parents * 2, tokens * 2, chosen + other, [0, n, 2 * n])
        assert c.status.item() == 9 and not bool(count.any()) and bool((path == -1).all())
        for a, b in zip(before, (c.k_pages, c.v_pages, c.page_table, c.lengths, c.refs)):
            assert torch.equal(a, b)


def test_too_many_nodes(paged):
    m = Model(paged, [3, 4], [[-1] * 257, [-1, 0]], 16)
    refused(m, 1, lambda c: None)


def test_other_stream_and_graph(paged):
    """A step's reserve and accept, captured and replayed, against the eager ones."""
    def one():
        m = Model(paged, [20, 33], [random_tree(i, 30, back=3) for i in range(2)], 16, seed=6, right=0.9)
        grown = dev([n + 30 for n in m.lens])
        args = [dev(x) for x in m.args()]

        def step():
            m.cache.reserve(args[0], grown)
            return m.cache.accept(*args)
        return m, step

    (a, step_a), (b, step_b) = one(), one()
    for _ in range(4):
        want = [x.tolist() for x in step_a()]
    warm, step_w = one()
    step_w()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_b()
    for _ in range(4):
        graph.replay()
    assert [x.tolist() for x in out] == want
    for x, y in zip(a.state(), b.state()):
        assert torch.equal(x, y)
    a.cache.check()
    b.cache.check()
    c, step_c = one()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            got = step_c()
    side.synchronize()
    assert [x.tolist() for x in got] == want


def test_refusals(paged):
    c = paged.PagedKVCache(8, 3, 4, num_layers=1, num_kv_heads=1, head_dim=64, page_size=16)
    c.reserve([0, 1], [5, 6])
    one = dev([0, 1])

    def call(k=c.k_pages, v=c.v_pages, table=c.page_table, lengths=c.lengths, refs=c.refs, slots=one, parents=dev([-1, -1]),
             tokens=one, chosen=one, **kw):
        return paged.accept(k, v, table, lengths, refs, slots, parents, tokens, chosen, **kw)

    for kw in (dict(k=c.k_pages.cpu()), dict(v=c.v_pages.half()), dict(table=c.page_table.cpu()), dict(lengths=c.lengths[:2]),
               dict(refs=c.refs[:4]), dict(refs=c.refs.long()), dict(slots=one.long()), dict(slots=one.cpu()), dict(slots=one[:1]),
               dict(parents=one[:1]), dict(tokens=one[:1]), dict(chosen=one.float()), dict(q_starts=one), dict(q_starts=dev([0, 1, 2]).cpu()),
               dict(slots=dev([0, 1, 2, 0]), q_starts=dev([0, 1, 2, 2, 2])), dict(status=one), dict(slots=one[:0], q_starts=dev([0]))):
        with pytest.raises(RuntimeError):
            call(**kw)
    path, emitted, count = call(slots=one[:0], parents=one[:0], tokens=one[:0], chosen=one[:0])
    assert path.numel() == emitted.numel() == count.numel() == 0
    path, emitted, count = call(parents=one[:0], tokens=one[:0], chosen=one[:0], q_starts=dev([0, 0, 0]))
    assert count.tolist() == [0, 0] and c.lengths.tolist() == [5, 6, 0]
