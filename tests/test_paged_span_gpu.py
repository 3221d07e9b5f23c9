"""Windowed attention and drafted trees on the paged cache against a plain implementation in 64 bits.

Tolerances.  As for the other attention of the cache (test_paged_gpu.py): the output's one rounding, half a step h of its
type, and 2^-13 of the largest value for scores in fp32 and weights in two 16-bit pieces.  Calls of more than 16 rows to a
sequence run on a kernel that rounds each weight once to 16 bits: sum_j p_j (1 + d_j) v_j with |d_j| <= h, which is off by
at most h sum_j p_j |v_j|, in the result (and rounded with it: h^2 of that, within the 2^-13).
"""
from __future__ import annotations

import math

import pytest
import torch

from test_paged_gpu import ROUND, Pool, close, dev, gen, normal

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
SHAPES = [(128, 64, 8, 2), (128, 16, 2, 5), (64, 32, 4, 1), (64, 128, 1, 8), (128, 128, 2, 17)]   # d, page, kv heads, group


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


def starts_of(qlens):
    out = [0]
    for n in qlens:
        out.append(out[-1] + n)
    return out


def window_mask(n, t, window, sinks):
    pos = torch.arange(t - n, t, device="cuda")[:, None]
    key = torch.arange(t, device="cuda")
    return (key <= pos) & ((pos - key < window) | (key < sinks))


def tree_mask(parents, t):
    """[n, t]: everything before the tree, then a node's ancestors and itself (positions from t - n on)."""
    n = len(parents)
    own = torch.zeros(n, n, dtype=torch.bool)
    for i, up in enumerate(parents):
        if up >= 0:
            own[i] = own[up]
        own[i, i] = True
    base = t - n
    seen = torch.zeros(n, max(t, 0), dtype=torch.bool)
    if base >= 0:
        seen[:, :base] = True
        seen[:, base:] = own
    else:   # the first nodes have no position: nothing sees them, and they see nothing
        seen[-base:] = own[-base:, -base:]
    return seen.cuda()


def once(tokens, group, seqs):
    """Whether such a call rounds its weights once."""
    return tokens * group > 16 * seqs


def near(got, ref, vmax, rounded):
    """ref: (the result, sum p |v|) in 64 bits."""
    out, mass = ref
    if not rounded:
        return close(got, out, vmax)
    tol = ROUND[got.dtype] * (out.abs() + mass) + 2.0 ** -13 * vmax + 2.0 ** -24
    bad = (got.double() - out).abs() - tol
    assert bool((bad <= 0).all()), f"over by {bad.max().item():.3e} (vmax {vmax:.3f})"


def pick(ref, *at):
    return tuple(x[at] for x in ref)


def reference(p, b, q, seen, scale, layer):
    """q [n, hq, d] of sequence b, seen [n, t]; in 64 bits, rows that see nothing are zero.  Also sum p |v|."""
    k, v = p.kv(b, layer)
    hq, hkv = q.shape[1], k.shape[1]
    grp = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(out)
    for h in range(hq):
        z = (q[:, h].double() @ k[:, h // grp].T) * scale
        w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
        w = torch.where(seen, w, 0)
        out[:, h] = w @ v[:, h // grp]
        mass[:, h] = w @ v[:, h // grp].abs()
    return out, mass


def check(p, call, qlens, masks, q, scale=None, layer=1):
    """call(q, slots, q_starts, status) against the masks, one for each sequence with query tokens."""
    status = dev([0])
    starts = starts_of(qlens)
    got = call(q, dev(p.slots), dev(starts), status)
    assert got.shape == q.shape and got.dtype == q.dtype
    s = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    for b, n in enumerate(qlens):
        if n:
            ref = reference(p, b, q[starts[b]:starts[b + 1]], masks[b], s, layer)
            near(got[starts[b]:starts[b + 1]], ref, p.v.abs().max().item(), once(starts[-1], q.shape[1] // p.k.shape[2], len(qlens)))
    assert status.item() == 0
    return got


def check_window(paged, p, hq, qlens, window, sinks, scale=None, std=2.0, layer=1):
    q = normal(p.g, sum(qlens), hq, p.k.shape[4], dtype=p.dtype, std=std)
    return check(p, lambda q, slots, starts, status: paged.window_attend(
        q, p.k, p.v, p.table, p.lengths, slots, layer=layer, window=window, sinks=sinks, q_starts=starts, scale=scale,
        status=status), qlens, [window_mask(n, t, window, sinks) for n, t in zip(qlens, p.lens)], q, scale, layer)


def random_tree(seed, n, back=9, roots=0.0):
    g = torch.Generator().manual_seed(seed)
    r = torch.rand(n, 2, generator=g).tolist()
    return [-1 if i == 0 or r[i][1] < roots else i - 1 - int(r[i][0] * min(i, back)) for i in range(n)]


def check_tree(paged, p, hq, trees, scale=None, std=2.0, layer=1):
    q = normal(p.g, sum(map(len, trees)), hq, p.k.shape[4], dtype=p.dtype, std=std)
    parents = dev(sum(trees, []))
    return check(p, lambda q, slots, starts, status: paged.tree_attend(
        q, p.k, p.v, p.table, p.lengths, slots, parents, layer=layer, q_starts=starts, scale=scale, status=status),
        [len(t) for t in trees], [tree_mask(t, n) for t, n in zip(trees, p.lens)], q, scale, layer)


# ---- sliding windows ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 4), (100, 16), (33, 129), (1000, 5), (10 ** 10, 10 ** 10)])
def test_window_single_tokens(paged, dtype, d, page, hkv, grp, window, sinks):
    p = Pool([1, 15, 16, 17, 100, 127, 513, 1400], page, hkv, d, dtype, seed=window % 97)
    check_window(paged, p, hkv * grp, [1] * 8, window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 3), (40, 0), (128, 16), (300, 200)])
def test_window_several_tokens(paged, dtype, d, page, hkv, grp, window, sinks):
    p = Pool([7, 300, 70, 33, 900, 41], page, hkv, d, dtype, seed=5)
    check_window(paged, p, hkv * grp, [7, 5, 0, 33, 3, 12], window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", SHAPES[:4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 4), (128, 0), (257, 150), (4000, 0)])
def test_window_prompts(paged, dtype, d, page, hkv, grp, window, sinks):
    p = Pool([700, 1300, 64, 1, 129], page, hkv, d, dtype, seed=window)
    check_window(paged, p, hkv * grp, [700, 413, 64, 1, 128], window, sinks)


def test_window_prompt_and_steps(paged):
    """A prompt among single tokens, and single tokens among which one sequence has many."""
    p = Pool([2000] + [300 + 7 * i for i in range(20)], 32, 2, 128, torch.bfloat16, seed=1)
    check_window(paged, p, 4, [2000] + [1] * 20, 512, 8)
    check_window(paged, p, 4, [150] + [1] * 20, 512, 8)


@pytest.mark.parametrize("window", [1, 255, 256, 257, 1025])
def test_window_long(paged, window):
    p = Pool([40000, 33], 64, 1, 128, torch.bfloat16, seed=2)
    check_window(paged, p, 2, [1, 1], window, 20)
    check_window(paged, p, 2, [300, 33], window, 20)


@pytest.mark.parametrize("qlens", [[1, 1], [90, 40]])
def test_window_of_everything_is_attend(paged, qlens):
    p = Pool([500, 90], 16, 2, 64, torch.float16, seed=3)
    q = normal(p.g, sum(qlens), 4, 64, dtype=torch.float16, std=2.0)
    starts = dev(starts_of(qlens))
    a = paged.attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=0, q_starts=starts)
    b = paged.window_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=0, window=500, q_starts=starts)
    for i, (n, t) in enumerate(zip(qlens, p.lens)):
        rows = slice(i * qlens[0], i * qlens[0] + n)
        ref = reference(p, i, q[rows], window_mask(n, t, t, 0), 1 / 8, 0)
        for x in (a, b):
            near(x[rows], ref, p.v.abs().max().item(), once(sum(qlens), 2, 2))


@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.3])
@pytest.mark.parametrize("n", [1, 200])
def test_window_scales(paged, scale, n):
    p = Pool([300, 260], 32, 2, 128, torch.bfloat16, seed=4)
    check_window(paged, p, 4, [n, n], 70, 4, scale=scale)


@pytest.mark.parametrize("n", [1, 3, 200])
def test_window_does_not_read_what_no_token_sees(paged, n):
    """Pages between the sinks and the windows: table entries out of range, and pages full of NaN."""
    p = Pool([1000, 800], 16, 2, 128, torch.bfloat16, seed=6)
    window, sinks = 100, 20
    q = normal(p.g, 2 * n, 4, 128)
    starts = dev([0, n, 2 * n])
    args = dict(layer=1, window=window, sinks=sinks, q_starts=starts)
    want = paged.window_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), **args)
    for b, t in enumerate(p.lens):
        first = -(-sinks // 16)
        last = (t - n - window + 1) // 16   # the first page that a token's window reaches
        for c in range(first, last):
            p.table[p.slots[b], c] = (-7, 10 ** 6)[c % 2]
    status = dev([0])
    got = paged.window_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), status=status, **args)
    assert status.item() == 0 and torch.equal(got, want)


@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_window_masked_infinities(paged, n, d):
    """NaN and infinities among keys and values: rows that do not see them are as without, in rows that see a value
    the channel is not finite, and in rows that see a NaN key all are NaN."""
    t, window, sinks = 700, 130, 3
    p = Pool([t], 16, 1, d, torch.bfloat16, seed=7)
    q = normal(p.g, n, 2, d)
    row = torch.tensor(p.rows[0], device="cuda")
    for bad in (math.inf, -math.inf, math.nan):
        for at, chan, key in ((t - 1, 5, False), (t - 60, 40, False), (t - window - 100, 63, False), (2, 17, False), (4, 1, False),
                              (t - window - 1, 0, False), (t - n - window, 33, False), (t - 50, 3, True), (300, 9, True)):
            k, v = p.k.clone(), p.v.clone()
            if key:
                k[row[at // 16], 1, 0, at % 16, chan] = math.nan
            else:
                v[row[at // 16], 1, 0, at % 16, chan] = bad
            # behind the sequence's end, in its last page
            v[row[-1], 1, 0, t % 16:] = bad
            k[row[-1], 1, 0, t % 16:] = bad
            got = paged.window_attend(q, k, v, p.table, p.lengths, dev(p.slots), layer=1, window=window, sinks=sinks,
                                      q_starts=dev([0, n]))
            seen = window_mask(n, t, window, sinks)
            sees = seen[:, at]
            ref = reference(p, 0, q, seen, 1 / math.sqrt(d), 1)
            vmax, rounded = p.v.abs().max().item(), once(n, 2, 1)
            near(got[~sees], pick(ref, ~sees), vmax, rounded)
            if key:
                assert bool(got[sees].isnan().all())
            else:
                assert not bool(got[sees][..., chan].isfinite().any())
                other = [c for c in range(d) if c != chan]
                near(got[sees][..., other], tuple(x[sees][..., other] for x in ref), vmax, rounded)


# ---- trees -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", SHAPES)
@pytest.mark.parametrize("nodes", [[1, 1, 1, 1], [4, 1, 7, 2], [16, 17, 3, 31], [64, 63, 0, 33], [256, 100, 129, 5]])
def test_trees(paged, dtype, d, page, hkv, grp, nodes):
    p = Pool([n + b for n, b in zip(nodes, (0, 500, 17, 1000))], page, hkv, d, dtype, seed=sum(nodes))
    check_tree(paged, p, hkv * grp, [random_tree(7 * i, n, roots=0.1 * (i % 2)) for i, n in enumerate(nodes)])


@pytest.mark.parametrize("kind", ["chain", "star", "roots", "binary"])
@pytest.mark.parametrize("n", [13, 200])
def test_tree_shapes(paged, kind, n):
    p = Pool([n + 100, n], 32, 2, 128, torch.bfloat16, seed=n)
    tree = {"chain": [i - 1 for i in range(n)], "star": [-1] + [0] * (n - 1), "roots": [-1] * n,
            "binary": [-1] + [(i - 1) // 2 for i in range(1, n)]}[kind]
    check_tree(paged, p, 4, [tree, tree])


@pytest.mark.parametrize("dtype", TYPES)
def test_trees_on_long_contexts(paged, dtype):
    p = Pool([30016, 5001, 12345], 64, 2, 128, dtype, seed=9)
    check_tree(paged, p, 4, [random_tree(1, 16), random_tree(2, 60), random_tree(3, 1)])
    check_tree(paged, p, 4, [random_tree(1, 100), random_tree(2, 60), random_tree(3, 1)])


@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.3])
@pytest.mark.parametrize("n", [5, 90])
def test_tree_scales(paged, scale, n):
    p = Pool([300, n + 1], 32, 2, 128, torch.float16, seed=4)
    check_tree(paged, p, 4, [random_tree(1, n)] * 2, scale=scale)


@pytest.mark.parametrize("n", [6, 120])
def test_tree_masked_infinities(paged, n):
    """Values of nodes that a row does not descend from change nothing there."""
    t = n + 75
    p = Pool([t], 32, 1, 64, torch.bfloat16, seed=7)
    tree = random_tree(5, n)
    seen = tree_mask(tree, t)
    q = normal(p.g, n, 2, 64)
    row = torch.tensor(p.rows[0], device="cuda")
    ref, vmax = reference(p, 0, q, seen, 1 / 8, 1), p.v.abs().max().item()
    for bad in (math.inf, math.nan):
        for at in (t - n, t - n + 2, t - 3, t - 1, 10):
            v = p.v.clone()
            v[row[at // 32], 1, 0, at % 32, 11] = bad
            v[row[-1], 1, 0, (t - 1) % 32 + 1:] = bad
            got = paged.tree_attend(q, p.k, v, p.table, p.lengths, dev(p.slots), dev(tree), layer=1, q_starts=dev([0, n]))
            sees = seen[:, at]
            near(got[~sees], pick(ref, ~sees), vmax, once(n, 2, 1))
            assert not bool(got[sees][..., 11].isfinite().any())
            near(got[sees][..., 12:], tuple(x[sees][..., 12:] for x in ref), vmax, once(n, 2, 1))


@pytest.mark.parametrize("n,other", [(5, 1), (100, 40)])
def test_tree_wrong_parents(paged, n, other):
    """A parent that does not come before its node counts as none, and is reported; so is a tree of too many nodes."""
    p = Pool([n + 50, other + 9], 16, 2, 64, torch.bfloat16, seed=8)
    good = random_tree(3, n)
    for at, up in ((0, 0), (n - 1, n - 1), (2, 4), (1, 10 ** 9), (3, -2), (n - 1, -10 ** 9)):
        tree, as_read = list(good), list(good)
        tree[at], as_read[at] = up, -1
        q = normal(p.g, n + other, 4, 64)
        status = dev([0])
        rest = random_tree(4, other)
        got = paged.tree_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), dev(tree + rest), layer=1,
                                q_starts=dev([0, n, n + other]), status=status)
        assert status.item() == 1
        vmax = p.v.abs().max().item()
        rounded = once(n + other, 2, 2)
        near(got[:n], reference(p, 0, q[:n], tree_mask(as_read, n + 50), 1 / 8, 1), vmax, rounded)
        near(got[n:], reference(p, 1, q[n:], tree_mask(rest, other + 9), 1 / 8, 1), vmax, rounded)
    p = Pool([400, 40], 16, 2, 64, torch.bfloat16, seed=8)
    q = normal(p.g, 257 + 7, 4, 64)
    rest, status = random_tree(4, 7), dev([0])
    got = paged.tree_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), dev([-1] * 257 + rest), layer=1,
                            q_starts=dev([0, 257, 264]), status=status)
    assert status.item() == 1 and not bool(got[:257].any())
    near(got[257:], reference(p, 1, q[257:], tree_mask(rest, 40), 1 / 8, 1), p.v.abs().max().item(), True)


# ---- both ----------------------------------------------------------------------------------------------------------

def calls(paged, p, n, seed=0):
    """The two operators as call(q, slots, starts, status), their masks for sequences of n query tokens."""
    tree = random_tree(seed, n)
    up = dev(tree * len(p.lens))

    def window(q, slots, starts, status, **kw):
        return paged.window_attend(q, kw.get("k", p.k), kw.get("v", p.v), kw.get("table", p.table), kw.get("lengths", p.lengths),
                                   slots, layer=kw.get("layer", 1), window=50, sinks=5, q_starts=starts, status=status)

    def drafted(q, slots, starts, status, **kw):
        return paged.tree_attend(q, kw.get("k", p.k), kw.get("v", p.v), kw.get("table", p.table), kw.get("lengths", p.lengths),
                                 slots, up, layer=kw.get("layer", 1), q_starts=starts, status=status)

    return ((window, [window_mask(n, t, 50, 5) for t in p.lens]), (drafted, [tree_mask(tree, t) for t in p.lens]))


@pytest.mark.parametrize("n", [2, 150])
def test_more_tokens_than_positions(paged, n):
    """Tokens at positions before the first see nothing; lengths of zero leave rows of zeros."""
    p = Pool([n - 1, 0, 30 + n], 16, 2, 64, torch.bfloat16, seed=3)
    q = normal(p.g, 3 * n, 4, 64)
    for call, masks in calls(paged, p, n):
        got = call(q, dev(p.slots), dev([0, n, 2 * n, 3 * n]), None)
        assert not bool(got[0].any()) and not bool(got[n:2 * n].any())
        vmax = p.v.abs().max().item()
        if n > 1:
            ref = reference(p, 0, q[1:n], masks[0][1:], 1 / 8, 1)
            near(got[1:n], ref, vmax, once(3 * n, 2, 3))
        near(got[2 * n:], reference(p, 2, q[2 * n:], masks[2], 1 / 8, 1), vmax, once(3 * n, 2, 3))


@pytest.mark.parametrize("n", [2, 150])
def test_wrong_tables(paged, n):
    """Wrong slots, lengths, starts and pages: rows of zeros, a reported code, the other sequences as they were."""
    p = Pool([200, 160, 180], 16, 2, 64, torch.float16, seed=11)
    q = normal(p.g, 3 * n, 4, 64, dtype=torch.float16)
    starts = dev([0, n, 2 * n, 3 * n])
    vmax, rounded = p.v.abs().max().item(), once(3 * n, 2, 3)
    for call, masks in calls(paged, p, n):
        want = [reference(p, b, q[b * n:b * n + n], masks[b], 1 / 8, 1) for b in range(3)]

        def others(got, *bad):
            for b in range(3):
                if b in bad:
                    assert not bool(got[b * n:b * n + n].any())
                else:
                    near(got[b * n:b * n + n], want[b], vmax, rounded)

        others(call(q, dev(p.slots), starts, None))
        for bad, code in ((-1, 8), (4, 8), (10 ** 9, 8)):
            status, slots = dev([0]), list(p.slots)
            slots[1] = bad
            others(call(q, dev(slots), starts, status), 1)
            assert status.item() == code
        for length in (-3, 16 * p.table.shape[1] + 1):
            status, lengths = dev([0]), p.lengths.clone()
            lengths[p.slots[1]] = length
            others(call(q, dev(p.slots), starts, status, lengths=lengths), 1)
            assert status.item() == 5
        for wrong in ([0, 2 * n, n, 3 * n], [1, n, 2 * n, 3 * n], [0, n, 2 * n, 3 * n - 1], [-n, 0, n, 3 * n]):
            status = dev([0])
            others(call(q, dev(p.slots), dev(wrong), status), 0, 1, 2)
            assert status.item() == 1
        # a page out of range: its positions are left out
        for page in (-1, p.k.shape[0], 2 ** 31 - 1):
            for back in (20, 100):
                status, table = dev([0]), p.table.clone()
                c = (p.lens[2] - back) // 16
                table[p.slots[2], c] = page
                got = call(q, dev(p.slots), starts, status, table=table)
                seen = masks[2].clone()
                assert status.item() == (9 if bool(seen[:, c * 16:c * 16 + 16].any()) else 0)
                seen[:, c * 16:c * 16 + 16] = False
                near(got[2 * n:], reference(p, 2, q[2 * n:], seen, 1 / 8, 1), vmax, rounded)
                for b in range(2):
                    near(got[b * n:b * n + n], want[b], vmax, rounded)


@pytest.mark.parametrize("n", [1, 40, 150])
def test_strides_layers_and_offsets(paged, n):
    """q with gaps, K and V side by side in one tensor, a q that starts at an odd place: the same bits."""
    p = Pool([300, 210], 32, 2, 64, torch.bfloat16, layers=3, seed=12)
    q = normal(p.g, 2 * n, 4, 64)
    starts = dev([0, n, 2 * n])
    both = torch.stack([p.k, p.v], 3).contiguous()     # [pages, layers, heads, 2, page, d]
    wide = torch.zeros(2 * n, 5, 80, dtype=q.dtype, device="cuda")
    wide[:, :4, 8:72] = q
    odd = torch.zeros(q.numel() + 3, dtype=q.dtype, device="cuda")[3:].view_as(q)
    odd.copy_(q)
    for call, masks in calls(paged, p, n):
        want = call(q, dev(p.slots), starts, None, layer=2)
        for b in range(2):
            near(want[b * n:b * n + n], reference(p, b, q[b * n:b * n + n], masks[b], 1 / 8, 2), p.v.abs().max().item(), once(2 * n, 2, 2))
        for other in (wide[:, :4, 8:72], odd):
            assert torch.equal(call(other, dev(p.slots), starts, None, layer=2), want)
        assert torch.equal(call(q, dev(p.slots), starts, None, layer=2, k=both[:, :, :, 0], v=both[:, :, :, 1]), want)


@pytest.mark.parametrize("n", [1, 40, 150])
def test_other_stream_graph_and_twice(paged, n):
    """The same bits on another stream, twice in a row, and from a replayed graph that follows the lengths."""
    p = Pool([300, 210], 32, 2, 64, torch.bfloat16, seed=13)
    q = normal(p.g, 2 * n, 4, 64)
    starts, slots = dev([0, n, 2 * n]), dev(p.slots)
    for call, _ in calls(paged, p, n):
        lengths = p.lengths.clone()
        want = call(q, slots, starts, None)
        assert torch.equal(call(q, slots, starts, None), want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call(q, slots, starts, None)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = call(q, slots, starts, None, lengths=lengths)
            b = call(a, slots, starts, None, lengths=lengths)
        for less in (0, 7, 100):
            lengths.copy_(torch.clamp(p.lengths - less, min=0))
            graph.replay()
            first = call(q, slots, starts, None, lengths=lengths)
            assert torch.equal(a, first) and torch.equal(b, call(first, slots, starts, None, lengths=lengths))


def test_past_32_bits(paged):
    """A pool of more than 2^32 bytes a side, pages at its ends."""
    page, d, pages = 128, 128, 140000
    k = torch.zeros(pages, 1, 1, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(1)
    at = [pages - 1, 0, 131072, pages - 2, 65537]
    for x in at:
        k[x], v[x] = normal(g, 1, 1, page, d), normal(g, 1, 1, page, d)
    table = torch.full((1, 5), -1, dtype=torch.int32, device="cuda")
    table[0] = dev(at)
    t = 5 * page - 3
    kk, vv = (torch.cat([x[i, 0, 0] for i in at])[:t, None].double() for x in (k, v))
    whole = type("", (), {"kv": lambda self, b, layer: (kk, vv)})()
    for n in (1, 100):
        q = normal(g, n, 2, d)
        tree = random_tree(n, n)
        for got, seen in (
            (paged.window_attend(q, k, v, table, dev([t]), dev([0]), layer=0, window=300, sinks=9, q_starts=dev([0, n])),
             window_mask(n, t, 300, 9)),
            (paged.tree_attend(q, k, v, table, dev([t]), dev([0]), dev(tree), layer=0, q_starts=dev([0, n])), tree_mask(tree, t)),
        ):
            near(got, reference(whole, 0, q, seen, 1 / math.sqrt(d), 0), vv.abs().max().item(), once(n, 2, 1))


def test_refusals(paged):
    p = Pool([20, 30], 16, 2, 64, torch.bfloat16)
    q, slots, up = normal(p.g, 2, 4, 64), dev(p.slots), dev([-1, -1])

    def window(q=q, k=p.k, v=p.v, table=p.table, lengths=p.lengths, slots=slots, layer=0, window=4, **kw):
        return paged.window_attend(q, k, v, table, lengths, slots, layer=layer, window=window, **kw)

    def tree(q=q, k=p.k, v=p.v, table=p.table, lengths=p.lengths, slots=slots, parents=up, layer=0, **kw):
        return paged.tree_attend(q, k, v, table, lengths, slots, parents, layer=layer, **kw)

    for call in (window, tree):
        for kw in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[:1]), dict(q=q.cpu()),
                   dict(layer=2), dict(layer=-1), dict(slots=slots.long()), dict(slots=slots[:1]), dict(lengths=p.lengths[:1]),
                   dict(lengths=p.lengths.cpu()), dict(table=p.table[0]), dict(table=p.table.long()), dict(v=p.v[:, :1]),
                   dict(k=p.k.transpose(3, 4)), dict(q_starts=dev([0, 2])), dict(q_starts=torch.tensor([0, 1, 2])),
                   dict(status=dev([0, 0]))):
            with pytest.raises(RuntimeError):
                call(**kw)
        with pytest.raises(RuntimeError, match="2048"):
            call(slots=slots.repeat(1025), q=q.repeat(1025, 1, 1), **({"parents": up.repeat(1025)} if call is tree else {}))
        assert call(q=q[:0], slots=slots[:0], **({"parents": up[:0]} if call is tree else {})).shape == (0, 4, 64)
        with pytest.raises(RuntimeError):
            call(slots=slots[:0], q_starts=dev([0]))
    for kw in (dict(window=0), dict(window=-1), dict(sinks=-1)):
        with pytest.raises(RuntimeError):
            window(**kw)
    for kw in (dict(parents=up[:1]), dict(parents=up.long()), dict(parents=up.cpu()), dict(parents=up.float())):
        with pytest.raises(RuntimeError):
            tree(**kw)
