"""Windowed attention and drafted trees hold their weights as the cache's other attention does, whatever the rows of a call.

Tolerance: that of test_paged_gpu.py, the output's one rounding (half a step) and 2^-13 of the largest value: scores are fp32
sums of 16-bit products, weights enter the second product in two 16-bit pieces (2^-16 of each).
"""
from __future__ import annotations

import math

import pytest
import torch

from test_paged_gpu import Pool, close, dev, normal
from test_paged_span_gpu import TYPES, random_tree, reference, starts_of, tree_mask, window_mask

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,hkv,grp", [(128, 64, 2, 2), (64, 16, 1, 5), (128, 128, 1, 17)])
@pytest.mark.parametrize("n", [1, 3, 60, 200])
def test_weights_in_two_pieces(paged, dtype, d, page, hkv, grp, n):
    """Few keys of about equal weight, where one 16-bit piece is more than that off."""
    lens = [n + 5, n + 40, n + 300]
    p = Pool(lens, page, hkv, d, dtype, seed=n)
    q = normal(p.g, 3 * n, hkv * grp, d, dtype=dtype, std=2.0)
    starts, tree = dev(starts_of([n] * 3)), random_tree(n, n)
    vmax = p.v.abs().max().item()
    for got, masks in (
        (paged.window_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=1, window=90, sinks=7, q_starts=starts),
         [window_mask(n, t, 90, 7) for t in lens]),
        (paged.tree_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), dev(tree * 3), layer=1, q_starts=starts),
         [tree_mask(tree, t) for t in lens]),
    ):
        for b in range(3):
            rows = slice(b * n, b * n + n)
            close(got[rows], reference(p, b, q[rows], masks[b], 1 / math.sqrt(d), 1)[0], vmax)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("above", [3.1, 6.9, 9.6, 20.0])   # nats
def test_one_key_far_above_the_sinks(paged, dtype, above):
    """A row that is one key's value: the weight it is multiplied by is the one it is divided by, wherever the reference of
    the weights stood before."""
    t, d, n = 640, 128, 100
    p = Pool([t], 64, 1, d, dtype, seed=2)
    q = torch.zeros(n, 2, d, dtype=dtype, device="cuda")
    q[..., 0] = above
    q[..., 1:] = normal(p.g, n, 2, d - 1, dtype=dtype, std=0.02)
    p.k[..., 0] = 0
    at = t - n - 20
    page = p.rows[0][at // 64]
    p.k[page, 1, 0, at % 64, 0] = 1.0
    starts = dev([0, n])
    vmax = p.v.abs().max().item()
    for got, seen in (
        (paged.window_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), layer=1, window=300, sinks=4, q_starts=starts, scale=1.0),
         window_mask(n, t, 300, 4)),
        (paged.tree_attend(q, p.k, p.v, p.table, p.lengths, dev(p.slots), dev([-1] * n), layer=1, q_starts=starts, scale=1.0),
         tree_mask([-1] * n, t)),
    ):
        close(got, reference(p, 0, q, seen, 1.0, 1)[0], vmax)


class Flat:
    """Sequences of one length on the same pages: the first key `above` nats above all others, its value -1, theirs 1."""

    def __init__(self, seqs, length, hkv, d, dtype, above, page=128):
        pages = -(-length // page)
        self.k = torch.zeros(pages, 1, hkv, page, d, dtype=dtype, device="cuda")
        self.v = torch.ones_like(self.k)
        self.k[0, 0, :, 0, 3] = above / 4
        self.v[0, 0, :, 0] = -1
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(seqs, 1)
        self.lengths = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
        self.slots = torch.arange(seqs, dtype=torch.int32, device="cuda")

    def q(self, tokens, heads):
        q = torch.zeros(tokens, heads, self.k.shape[4], dtype=self.k.dtype, device="cuda")
        q[..., 3] = 4
        return q


def flat_result(above, keys):
    """Of the first key and `keys - 1` others; `above` as the type has it."""
    w = (keys - 1) * math.exp(-above)
    return (w - 1) / (w + 1)


ABOVE = [8.0, 16.5, 17.0, 17.25, 18.5, 20.0]   # times 1/4 they are 16-bit numbers; near 2^-24 and below


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("above", ABOVE)
@pytest.mark.parametrize("length,n", [(30000, 9), (100000, 9), (30000, 70)])
def test_many_small_weights_behind_a_sink(paged, dtype, above, length, n):
    """Weights of 2^-25 of a row's largest count when there are enough of them (many rows to a sequence, and sequences enough
    for one to be a CTA's work from its first position to its last)."""
    seqs = 300
    p = Flat(seqs, length, 1, 64, dtype, above)
    q = p.q(seqs * n, 2)
    starts = torch.arange(0, seqs * n + 1, n, dtype=torch.int32, device="cuda")
    got = paged.window_attend(q, p.k, p.v, p.table, p.lengths, p.slots, layer=0, window=length, q_starts=starts, scale=1.0)
    ref = torch.tensor([flat_result(above, length - n + 1 + i) for i in range(n)], dtype=torch.float64, device="cuda")
    close(got, ref.repeat(seqs)[:, None, None].expand_as(got), 1.0)
    got = paged.window_attend(q, p.k, p.v, p.table, p.lengths, p.slots, layer=0, window=length // 2, sinks=1, q_starts=starts, scale=1.0)
    ref = torch.full_like(got, flat_result(above, length // 2 + 1), dtype=torch.float64)
    close(got, ref, 1.0)
    tree = [-1] * n
    got = paged.tree_attend(q, p.k, p.v, p.table, p.lengths, p.slots, dev(tree * seqs), layer=0, q_starts=starts, scale=1.0)
    ref = torch.full_like(got, flat_result(above, length - n + 1), dtype=torch.float64)
    close(got, ref, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("above", ABOVE)
@pytest.mark.parametrize("n", [1, 2])
def test_many_small_weights_single_tokens(paged, dtype, above, n):
    """The same for few rows to a sequence, where a warp has thousands of positions."""
    length, seqs = 40000, 2000
    p = Flat(seqs, length, 2, 64, dtype, above)
    q = p.q(seqs * n, 4)
    starts = torch.arange(0, seqs * n + 1, n, dtype=torch.int32, device="cuda")
    got = paged.window_attend(q, p.k, p.v, p.table, p.lengths, p.slots, layer=0, window=30000, sinks=1, q_starts=starts, scale=1.0)
    close(got, torch.full_like(got, flat_result(above, 30001), dtype=torch.float64), 1.0)
    got = paged.tree_attend(q, p.k, p.v, p.table, p.lengths, p.slots, dev([-1] * (seqs * n)), layer=0, q_starts=starts, scale=1.0)
    close(got, torch.full_like(got, flat_result(above, length - n + 1), dtype=torch.float64), 1.0)
