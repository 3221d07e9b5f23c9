"""The C entries from other host threads (ctypes lets go of the interpreter's lock during a call), in a process of its
own, so that the first use of a kernel is theirs."""
from __future__ import annotations

import ctypes
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


class CPool(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "index")]
                + [(n, ctypes.c_int) for n in ("dtype", "num_pages", "num_layers", "num_kv_heads", "page_size", "head_dim")]
                + [(n, ctypes.c_longlong) for t in "kvi" for n in (f"{t}_page", f"{t}_layer", f"{t}_head")])


class CAttend(ctypes.Structure):
    _fields_ = ([("pool", ctypes.POINTER(CPool)), ("q", ctypes.c_void_p), ("q_token", ctypes.c_longlong), ("q_head", ctypes.c_longlong),
                 ("out", ctypes.c_void_p), ("table", ctypes.c_void_p), ("table_row", ctypes.c_longlong), ("num_slots", ctypes.c_int),
                 ("table_cols", ctypes.c_int)]
                + [(n, ctypes.c_void_p) for n in ("lengths", "slots", "q_starts", "group_starts", "prefix_pages")]
                + [(n, ctypes.c_int) for n in ("num_seqs", "num_groups", "total_q", "num_q_heads", "layer")]
                + [("scale", ctypes.c_float), ("status", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                   ("workspace_bytes", ctypes.c_size_t)])


def main(threads):
    sys.path.insert(0, str(ROOT))
    from megaqwen_b200.build import LIB
    lib = ctypes.CDLL(str(LIB))
    lib.mq_paged_attend_workspace_bytes.restype = ctypes.c_size_t
    lib.mq_last_error_detail.restype = ctypes.c_char_p
    hkv, hq, d, page = 2, 4, 64, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    k = torch.randn(40, 1, hkv, page, d, device="cuda", generator=g).bfloat16()
    v = torch.randn(k.shape, device="cuda", generator=g).bfloat16()
    pool = CPool(k.data_ptr(), v.data_ptr(), None, 0, 40, 1, hkv, page, d, *([hkv * page * d, hkv * page * d, page * d] * 2), 0, 0, 0)
    jobs = []
    for i in range(threads):
        n = (1, 2048, 3, 1500, 20, 900, 100, 2000)[i]     # sequences of one table, their sizes as far apart as they may be
        table = torch.randint(0, 40, (n, 3), device="cuda", generator=g).int()
        lengths = torch.randint(1, 48, (n,), device="cuda", generator=g).int()
        slots = torch.arange(n, device="cuda").int()
        q = torch.randn(n, hq, d, device="cuda", generator=g).bfloat16()
        out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
        p = CAttend(ctypes.pointer(pool), q.data_ptr(), hq * d, d, out.data_ptr(), table.data_ptr(), 3, n, 3, lengths.data_ptr(),
                    slots.data_ptr(), None, None, None, n, 0, n, hq, 0, d ** -0.5, status.data_ptr(), None, 0)
        p.workspace_bytes = lib.mq_paged_attend_workspace_bytes(ctypes.byref(p))
        ws = torch.empty(p.workspace_bytes, dtype=torch.uint8, device="cuda")
        p.workspace = ws.data_ptr()
        jobs.append((p, torch.cuda.Stream(), out, status, (table, lengths, slots, q, ws)))
    torch.cuda.synchronize()
    gate, codes, detail = threading.Barrier(threads), [[] for _ in range(threads)], [b""] * threads

    def work(i):
        p, stream = jobs[i][:2]
        gate.wait()
        for _ in range(30):
            codes[i].append(lib.mq_paged_attend(ctypes.byref(p), ctypes.c_void_p(stream.cuda_stream)))
        detail[i] = lib.mq_last_error_detail()
    ts = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not any(any(c) for c in codes), (codes, detail)
    from megaqwen_b200 import paged
    for p, _, out, status, (table, lengths, slots, q, _) in jobs:
        assert status.item() == 0
        assert torch.equal(out, paged.attend(q, k, v, table, lengths, slots, layer=0))


def run(threads):
    r = subprocess.run([sys.executable, __file__, str(threads)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_a_thread_without_a_context():
    """The entry is the first CUDA call that its thread makes."""
    run(1)


def test_sizes_that_differ_at_once():
    """What is set up on a kernel's first use must not depend on which of several sizes is first."""
    for _ in range(3):
        run(8)


if __name__ == "__main__":
    main(int(sys.argv[1]))
