"""Paged KV cache: pages shared between sequences, and the attention that reads them.

The decoders of this package keep one contiguous cache per sequence.  Here K
and V live in pages of ``page_size`` positions of every layer and kv head,
``k_pages`` / ``v_pages`` ``[pages, layers, kv_heads, page_size, head_dim]``
(bf16 or fp16, head_dim 64 or 128, page_size 16, 32, 64 or 128), and a sequence
is a row ("slot") of ``page_table`` (int32 ``[slots, pages per slot]``) with a
length.  ``refs[p]`` counts the slots that hold page ``p``; 0 means free.  Only
full pages are shared: a fork copies a part page at once, so a page that is
written has one owner.  The reference has no counterpart.

Functions on plain tensors (all int32 arguments live on the GPU; nothing
synchronises, and outputs come from the current stream's allocator):

``rope_tables``    cos / sin tables, optionally scaled for long contexts
``rope``           rotary positions (half or interleaved pairs, part of the head)
``rope_append``    the same for q, fused with the write of rotated k and of v
``reserve`` ``fork`` ``free`` ``copy`` ``compact``   pages and their bookkeeping
``attend``         attention, shared prefixes read once per group
``sparse_attend``  attention over the pages that a cheap score selects

Arguments that live on the GPU are checked there: a wrong slot, page or
position writes its code to ``status`` (int32 ``[1]``, if given) and changes no
table; attention reads a wrong slot or position as an empty sequence and leaves
out the positions of a page that is out of range.  :class:`PagedKVCache` holds the tensors
and raises from :meth:`PagedKVCache.check`.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _C
from .weights import HEAD_DIM, NUM_KV_HEADS, NUM_LAYERS, ROPE_THETA

rope = _C.paged_rope
rope_append = _C.paged_rope_append
reserve = _C.paged_reserve
fork = _C.paged_fork
free = _C.paged_free
copy = _C.paged_copy
compact = _C.paged_compact
attend = _C.paged_attend
sparse_attend = _C.paged_sparse_attend

INDEX_PAD = 16   # bytes of an index record after the two bounds: the exponent and padding

BAD_TOKEN = 4
STATUS = {
    1: "starts out of order",
    3: "a wait of a kernel ran out",
    BAD_TOKEN: "token id out of range",
    5: "position out of range",
    8: "slot out of range, named twice or not empty",
    9: "page number out of range or in the wrong state",
    10: "not enough free pages",
}


def to_device(x, dtype: torch.dtype, device) -> torch.Tensor:
    """x (a list, or a tensor) as a tensor there, without waiting for the GPU: host data goes through pinned memory of its
    own, so the caller may write to x again at once."""
    x = torch.as_tensor(x, dtype=dtype)
    if x.device.type == "cpu" and torch.device(device).type == "cuda":
        return (x.clone() if x.is_pinned() else x).pin_memory().to(device, non_blocking=True)
    return x.to(device)


def rope_tables(max_pos: int, rotary_dim: int = HEAD_DIM, theta: float = ROPE_THETA, scaling: Optional[dict] = None,
                device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 cos and sin ``[max_pos, rotary_dim / 2]`` for :func:`rope_append`.

    Channel pair i turns by ``pos * theta^(-2 i / rotary_dim)``, computed in 64
    bits and rounded once.  ``scaling`` stretches this for contexts longer than
    the trained one:

    * ``{"type": "linear", "factor": f}``: all frequencies divided by f;
    * ``{"type": "ntk", "factor": f}``: theta raised so that the slowest pair is divided by f;
    * ``{"type": "yarn", "factor": f, "trained": n}``: pairs that turn less than ``beta_slow`` (1) times over
      the trained length divided by f, more than ``beta_fast`` (32) times kept, a ramp between them; the tables
      times ``0.1 ln f + 1`` (or ``mscale``);
    * ``{"type": "llama3", "factor": f, "trained": n, "low": 1, "high": 4}``: wavelengths above n / low divided by f,
      below n / high kept, a smooth blend between them.
    """
    if max_pos < 1:
        raise ValueError("max_pos must be positive")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    mult = 1.0
    s = dict(scaling or {})
    kind = s.pop("type", None)
    factor = float(s.pop("factor", 1.0))
    if factor < 1.0:
        raise ValueError("the scaling factor must be at least 1")
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of at least 4")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** (-2.0 * i / rotary_dim)
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        trained, fast, slow = s.pop("trained"), s.pop("beta_fast", 32.0), s.pop("beta_slow", 1.0)

        def pair_of(turns):   # the pair that turns so many times over the trained length
            return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(0.0, math.floor(pair_of(fast))), min(rotary_dim - 1.0, math.ceil(pair_of(slow)))
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
        mult = s.pop("mscale", 0.1 * math.log(factor) + 1.0)
    elif kind == "llama3":
        trained, low, high = s.pop("trained"), s.pop("low", 1.0), s.pop("high", 4.0)
        if high <= low:
            raise ValueError("llama3 scaling needs high > low")
        turns = trained * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
    elif kind not in (None, "ntk"):
        raise ValueError(f"unknown scaling type {kind!r}")
    if s:
        raise ValueError(f"unknown scaling entries {sorted(s)}")
    a = torch.outer(torch.arange(max_pos, dtype=torch.float64), inv)
    return (a.cos() * mult).float().to(device), (a.sin() * mult).float().to(device)


class PagedKVCache:
    """A pool of pages with its tables, on one GPU.

    ``index=True`` keeps the page scores that :meth:`sparse_attend` needs.
    Device-side errors collect in ``status``; :meth:`check` raises the first.
    """

    def __init__(self, num_pages: int, max_seqs: int, max_pages_per_seq: int, num_layers: int = NUM_LAYERS,
                 num_kv_heads: int = NUM_KV_HEADS, head_dim: int = HEAD_DIM, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", index: bool = False):
        if min(num_pages, max_seqs, max_pages_per_seq, num_layers, num_kv_heads) < 1:
            raise ValueError("sizes must be positive")
        shape = (num_pages, num_layers, num_kv_heads, page_size, head_dim)
        self.page_size = page_size
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.index = (torch.zeros(num_pages, num_layers, num_kv_heads, 2 * head_dim + INDEX_PAD, dtype=torch.int8,
                                  device=device) if index else None)
        self.page_table = torch.full((max_seqs, max_pages_per_seq), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def _ints(self, x) -> torch.Tensor:
        return to_device(x, torch.int32, self.k_pages.device).reshape(-1)

    def check(self) -> None:
        """Raises the first device-side error since the last check (synchronises)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError(f"paged cache: {STATUS.get(code, 'error')} (code {code})")

    def free_pages(self) -> int:
        """Pages that no sequence holds (synchronises)."""
        return int((self.refs == 0).sum().item())

    def reserve(self, slots, lengths) -> None:
        reserve(self.page_table, self.lengths, self.refs, self._ints(slots), self._ints(lengths), self.page_size,
                status=self.status)

    def fork(self, parents, children) -> None:
        fork(self.k_pages, self.v_pages, self.page_table, self.lengths, self.refs, self._ints(parents),
             self._ints(children), status=self.status)

    def free(self, slots) -> None:
        free(self.page_table, self.lengths, self.refs, self._ints(slots), self.page_size, status=self.status)

    def compact(self, num_pages: int) -> "PagedKVCache":
        """This cache with its pages in use gathered into a pool of num_pages.  Where they do not fit, both caches'
        :meth:`check` raises and the new one is empty."""
        if num_pages < 1:
            raise ValueError("num_pages must be positive")
        new = object.__new__(PagedKVCache)
        new.page_size = self.page_size
        new.k_pages = self.k_pages.new_zeros((num_pages,) + tuple(self.k_pages.shape[1:]))
        new.v_pages = torch.zeros_like(new.k_pages)
        new.index = None if self.index is None else self.index.new_zeros((num_pages,) + tuple(self.index.shape[1:]))
        new.page_table = torch.full_like(self.page_table, -1)
        new.refs = self.refs.new_zeros(num_pages)
        new.status = torch.zeros_like(self.status)
        compact(self.k_pages, self.v_pages, self.page_table, self.refs, new.k_pages, new.v_pages, new.page_table,
                new.refs, index=self.index, out_index=new.index, status=new.status)
        new.lengths = torch.where(new.status == 0, self.lengths, 0)
        self.status.copy_(torch.where(self.status == 0, new.status, self.status))
        return new

    def append(self, layer: int, q, k, v, slots, positions, cos, sin, interleaved: bool = False) -> torch.Tensor:
        return rope_append(q, k, v, self.k_pages, self.v_pages, self.page_table, slots, positions, cos, sin, layer=layer,
                           interleaved=interleaved, index=self.index, status=self.status)

    def attend(self, layer: int, q, slots, q_starts=None, group_starts=None, prefix_pages=None, scale=None) -> torch.Tensor:
        return attend(q, self.k_pages, self.v_pages, self.page_table, self.lengths, slots, layer=layer, q_starts=q_starts,
                      group_starts=group_starts, prefix_pages=prefix_pages, scale=scale, status=self.status)

    def sparse_attend(self, layer: int, q, slots, positions, top_k: int, scale=None):
        if self.index is None:
            raise ValueError("sparse attention needs a cache with index=True")
        return sparse_attend(q, self.k_pages, self.v_pages, self.index, self.page_table, slots, positions, layer=layer,
                             top_k=top_k, scale=scale, status=self.status)
