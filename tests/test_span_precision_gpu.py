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
