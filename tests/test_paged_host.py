"""Paged cache on a host without a GPU: argument checks that come before any CUDA call, sizes of the C ABI."""
from __future__ import annotations

import ctypes

import pytest
import torch

from megaqwen_b200.build import LIB


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_cpu_tensors_are_refused(paged):
    k = torch.zeros(4, 1, 2, 16, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(2, 2, dtype=torch.int32), ints(1, 0)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    cos, sin = paged.rope_tables(8, 64, device="cpu")
    for call in (
        lambda: paged.attend(q, k, k, table, n, ints(0), layer=0),
        lambda: paged.sparse_attend(q, k, k, torch.zeros(4, 1, 2, 144, dtype=torch.int8), table, ints(0), ints(0), layer=0, top_k=1),
        lambda: paged.rope(q, ints(0), cos, sin),
        lambda: paged.rope_append(q, q[:, :2], q[:, :2], k, k, table, ints(0), ints(0), cos, sin, layer=0),
        lambda: paged.free(table, n, ints(0, 0, 0, 0), ints(0), 16),
        lambda: paged.reserve(table, n, ints(0, 0, 0, 0), ints(0), ints(3), 16),
        lambda: paged.fork(k, k, table, n, ints(0, 0, 0, 0), ints(0), ints(1)),
        lambda: paged.copy(k, k, ints(0), ints(1)),
        lambda: paged.compact(k, k, table, ints(0, 0, 0, 0), k, k, table, ints(0, 0, 0, 0)),
    ):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_cache_sizes_are_checked(paged):
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            paged.PagedKVCache(*bad, device="cpu")
    c = paged.PagedKVCache(4, 2, 3, num_layers=1, num_kv_heads=1, head_dim=64, page_size=16, device="cpu")
    assert c.index is None and c.free_pages() == 4
    c.check()
    with pytest.raises(ValueError, match="index=True"):
        c.sparse_attend(0, None, None, None, 1)
    c.status.fill_(10)
    with pytest.raises(RuntimeError, match="not enough free pages"):
        c.check()
    c.check()


def test_c_entries_refuse_null():
    lib = ctypes.CDLL(str(LIB))
    lib.mq_paged_workspace_bytes.restype = ctypes.c_size_t
    assert lib.mq_paged_workspace_bytes(100, 10) >= 4 * (3 * 100 + 2 * 100 + 10)
    assert lib.mq_paged_workspace_bytes(-1, 0) == 0
    for name, args in (("mq_paged_free", 4), ("mq_paged_reserve", 5), ("mq_paged_fork", 6), ("mq_rope", 2),
                       ("mq_paged_attend", 2), ("mq_paged_sparse", 2)):
        assert getattr(lib, name)(*[None] * args) == 1, name
    for name in ("mq_paged_attend_workspace_bytes", "mq_paged_sparse_workspace_bytes"):
        assert getattr(lib, name)(None) == 0
    lib.mq_error_string.restype = ctypes.c_char_p
    assert lib.mq_error_string(10) == b"not enough free pages"
