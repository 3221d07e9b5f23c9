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


class CPool(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "index")]
                + [(n, ctypes.c_int) for n in ("dtype", "num_pages", "num_layers", "num_kv_heads", "page_size", "head_dim")]
                + [(n, ctypes.c_longlong) for t in "kvi" for n in (f"{t}_page", f"{t}_layer", f"{t}_head")])


BLOCK = 16 * 64          # elements of a [page_size, head_dim] block


def c_pool(k, v, pages, layers=2, heads=3, page=None, layer=None, head=BLOCK):
    """A pool of bf16 pages of 16 x 64; addresses in elements, nothing is ever read there."""
    layer = layer or heads * head
    page = page or layers * layer
    base = 1 << 40
    return CPool(base + 2 * k, base + 2 * v, None, 0, pages, layers, heads, 16, 64, page, layer, head, page, layer, head, 0, 0, 0)


def test_pools_that_share_memory():
    """copy and compact tell pools that share pages from those that only lie in one storage.  Without a workspace nothing
    is launched: a call whose pools are accepted answers 7, others 1."""
    lib = ctypes.CDLL(str(LIB))
    page, far = 6 * BLOCK, 10 ** 9
    some = ctypes.c_void_p(4096)
    table = (ctypes.c_char * 256)()

    def copy(a, b):
        return lib.mq_paged_copy(ctypes.byref(a), ctypes.byref(b), some, some, 2, None, None, ctypes.c_size_t(0), None)

    class CTable(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in ("table", "lengths", "refs")]
                    + [(n, ctypes.c_int) for n in ("num_slots", "cols", "num_pages", "page_size")]
                    + [("row_stride", ctypes.c_longlong), ("status", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                       ("workspace_bytes", ctypes.c_size_t)])

    def compact(a, b):
        t = CTable(ctypes.addressof(table), None, ctypes.addressof(table) + 64, 1, 1, a.num_pages, 16, 1, None, None, 0)
        return lib.mq_paged_compact(ctypes.byref(a), ctypes.byref(b), ctypes.byref(t), ctypes.c_void_p(ctypes.addressof(table) + 128),
                                    ctypes.c_longlong(1), ctypes.c_void_p(ctypes.addressof(table) + 192), None)
    whole = c_pool(0, far, 40)
    # another storage; the same pool; its first pages; its last ones
    assert copy(whole, c_pool(far * 2, far * 3, 40)) == 7 and compact(whole, c_pool(far * 2, far * 3, 40)) == 7
    for view in (whole, c_pool(0, far, 4), c_pool(36 * page, far + 36 * page, 4)):
        assert copy(whole, view) == 7 and copy(view, whole) == 7
        assert compact(whole, view) == 1 and compact(view, whole) == 1
    # two halves of one storage
    assert copy(c_pool(0, far, 20), c_pool(20 * page, far + 20 * page, 20)) == 7
    assert compact(c_pool(0, far, 20), c_pool(20 * page, far + 20 * page, 20)) == 7
    # layers of one storage, layers that overlap
    four = dict(pages=40, page=2 * page)
    assert copy(c_pool(0, far, **four), c_pool(page, far + page, **four)) == 7
    assert compact(c_pool(0, far, **four), c_pool(page, far + page, **four)) == 7
    assert compact(c_pool(0, far, **four), c_pool(page // 2, far + page // 2, **four)) == 1
    # K and V in one storage: the pool itself, its halves, keys of one on the values of the other
    both = dict(page=2 * page)
    assert copy(c_pool(0, page, 40, **both), c_pool(0, page, 40, **both)) == 7
    assert compact(c_pool(0, page, 20, **both), c_pool(40 * page, 41 * page, 20, **both)) == 7
    assert compact(c_pool(0, page, 20, **both), c_pool(page, far, 20, **both)) == 1
    # pages the innermost dimension
    inner = dict(pages=40, page=BLOCK, head=40 * BLOCK, layer=120 * BLOCK)
    assert copy(c_pool(0, far, **inner), c_pool(0, far, **inner)) == 7
    # a layer on (page p lies on p and p + 1), rows on, keys and values shifted by different pages, other strides
    assert copy(whole, c_pool(page // 2, far + page // 2, 30)) == 1
    assert copy(whole, c_pool(512, far + 512, 30)) == 1
    assert copy(whole, c_pool(page, far + 2 * page, 30)) == 1
    assert copy(whole, c_pool(0, far, 20, page=2 * page)) == 1
