"""Windows, drafted trees and sampling on a host without a GPU: argument checks that come before any CUDA call."""
from __future__ import annotations

import ctypes

import pytest
import torch

from megaqwen_b200.build import LIB


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    from megaqwen_b200 import paged, sampling
    k = torch.zeros(4, 1, 2, 16, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(2, 2, dtype=torch.int32), ints(1, 0)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for call in (
        lambda: paged.window_attend(q, k, k, table, n, ints(0), layer=0, window=4),
        lambda: paged.tree_attend(q, k, k, table, n, ints(0), ints(-1), layer=0),
        lambda: paged.accept(k, k, table, n, ints(0, 0, 0, 0), ints(0), ints(-1), ints(0), ints(0)),
        lambda: sampling.sample(torch.zeros(1, 8), torch.zeros(1)),
    ):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_c_entries_refuse_null():
    lib = ctypes.CDLL(str(LIB))
    for name, args in (("mq_paged_window", 2), ("mq_paged_tree", 2), ("mq_sample", 2)):
        assert getattr(lib, name)(*[None] * args) == 1, name
    assert lib.mq_paged_accept(*[None] * 7, 0, 0, *[None] * 4) == 1
    lib.mq_paged_span_workspace_bytes.restype = lib.mq_paged_accept_workspace_bytes.restype = ctypes.c_size_t
    assert lib.mq_paged_span_workspace_bytes(None) == 0
    assert lib.mq_paged_accept_workspace_bytes(-1) == 0


def test_decoder_options():
    from megaqwen_b200.paged_decoder import PagedDecoder
    for bad in (dict(window=4, sparse_pages=2), dict(window=0), dict(window=4, sinks=-1), dict(sinks=1)):
        with pytest.raises(ValueError, match="window"):
            PagedDecoder(None, num_pages=1, max_seqs=1, **bad)
