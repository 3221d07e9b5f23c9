"""accept where a sequence would end inside a page that another one holds."""
from __future__ import annotations

import pytest
import torch

from test_paged_gpu import dev, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


def forked(paged, page=16, nodes=40, start=5):
    c = paged.PagedKVCache(16, 3, 6, num_layers=2, num_kv_heads=1, head_dim=64, page_size=page)
    c.reserve([0], [start + nodes])
    c.k_pages.normal_()
    c.v_pages.normal_()
    c.fork([0], [1])
    return c


def state(c):
    return [x.clone() for x in (c.k_pages, c.v_pages, c.page_table, c.lengths, c.refs)]


@pytest.mark.parametrize("keep", [1, 7, 20, 26])
def test_no_sequence_ends_inside_a_page_of_another(paged, keep):
    """A chain whose first `keep` nodes are right: nothing moves, but the page that the sequence would end in is the fork's,
    too, and the next token would be written there."""
    c, n = forked(paged), 40
    before = state(c)
    chosen = [1] * (keep - 1) + [9] * (n - keep + 1)
    path, emitted, count = c.accept([0], [i - 1 for i in range(n)], [1] * n, chosen, [0, n])
    assert c.status.item() == 9 and count.tolist() == [0] and bool((path == -1).all()) and bool((emitted == -1).all())
    for a, b in zip(before, state(c)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("keep", [11, 27, 36, 40])
def test_a_whole_number_of_shared_pages_stays(paged, keep):
    """Where the cut falls between pages, in a page that the sequence has to itself, or nowhere, it is accepted; tokens
    appended then leave the other sequence as it was."""
    c, n, start = forked(paged), 40, 5
    other = c.page_table[1].clone()
    held = [x[other[:3].long()].clone() for x in (c.k_pages, c.v_pages)]
    chosen = [1] * (keep - 1) + [9] * (n - keep + 1)
    path, emitted, count = c.accept([0], [i - 1 for i in range(n)], [1] * n, chosen, [0, n])
    c.check()
    assert count.tolist() == [keep] and path.tolist() == list(range(keep)) + [-1] * (n - keep)
    assert c.lengths.tolist() == [start + keep, start + n, 0]
    length = start + keep
    c.reserve([0], [length + 3])
    g = torch.Generator(device="cuda").manual_seed(0)
    cos, sin = paged.rope_tables(128, 64)
    for layer in range(2):
        c.append(layer, normal(g, 3, 2, 64), normal(g, 3, 1, 64), normal(g, 3, 1, 64), dev([0] * 3),
                 dev([length, length + 1, length + 2]), cos, sin)
    c.check()
    assert torch.equal(c.page_table[1], other)
    for x, y in zip((c.k_pages, c.v_pages), held):
        assert torch.equal(x[other[:2].long()], y[:2])
        assert torch.equal(x[other[2].long()][..., :start + n - 32, :], y[2][..., :start + n - 32, :])
