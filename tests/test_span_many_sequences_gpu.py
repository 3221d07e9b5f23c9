"""Windows and trees of several hundred sequences in one call: both sides of what the tensor-core kernel's schedule holds, and
of the threads that sum it."""
from __future__ import annotations

import math

import pytest
import torch

from test_paged_gpu import Pool, close, dev, normal
from test_paged_span_gpu import random_tree, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


@pytest.mark.parametrize("seqs", [383, 384, 385, 447, 448, 449, 700])
@pytest.mark.parametrize("d", [128, 64])
def test_many_sequences(paged, seqs, d):
    """About 20 rows to a sequence, empty ones and sequences without query tokens among them."""
    lens = [0 if i % 29 == 7 else 30 + i * 37 % 170 for i in range(seqs)]
    qlens = [0 if i % 23 == 5 else 10 if i % 31 else 28 for i in range(seqs)]
    p = Pool(lens, 16, 1, d, torch.bfloat16, layers=1, seed=seqs)
    q = normal(p.g, sum(qlens), 2, d, std=2.0)
    starts = starts_of(qlens)
    trees = [random_tree(i, n) for i, n in enumerate(qlens)]
    status = dev([0])
    args = (q, p.k, p.v, p.table, p.lengths, dev(p.slots))
    window = paged.window_attend(*args, layer=0, window=50, sinks=3, q_starts=dev(starts), status=status)
    tree = paged.tree_attend(*args, dev(sum(trees, [])), layer=0, q_starts=dev(starts), status=status)
    assert status.item() == 0
    # every token's row over the longest sequence, in 64 bits
    most = max(lens)
    keys, values = torch.zeros(2, seqs, most, d, dtype=torch.float64, device="cuda")
    seen = torch.zeros(2, len(q), most, dtype=torch.bool)
    seq = torch.zeros(len(q), dtype=torch.long)
    for b, (n, t) in enumerate(zip(qlens, lens)):
        if t:
            k, v = p.kv(b, 0)
            keys[b, :t], values[b, :t] = k[:, 0], v[:, 0]
        base, key = t - n, torch.arange(most)
        bits = [0] * n   # of the nodes' ancestors
        for i, up in enumerate(trees[b]):
            bits[i] = (bits[up] if up >= 0 else 0) | 1 << i
            row, pos = starts[b] + i, base + i
            seq[row] = b
            if pos < 0:
                continue
            seen[0, row] = (key <= pos) & ((pos - key < 50) | (key < 3))
            seen[1, row] = key < base
            for j in range(i + 1):
                if bits[i] >> j & 1 and base + j >= 0:
                    seen[1, row, base + j] = True
    seq = seq.cuda()
    for got, mask in ((window, seen[0].cuda()), (tree, seen[1].cuda())):
        s = torch.einsum("nhd,nkd->nhk", q.double(), keys[seq]) / math.sqrt(d)
        w = torch.softmax(s.masked_fill(~mask[:, None], -math.inf), -1).nan_to_num(0.0)
        close(got, torch.einsum("nhk,nkd->nhd", w, values[seq]), p.v.abs().max().item())
