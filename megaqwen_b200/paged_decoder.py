"""Qwen3 decoding on the paged KV cache: prompts shared between samples.

:class:`PagedDecoder` runs the model of this package with its projections as
plain matrix products and everything around the cache on the operators of
:mod:`megaqwen_b200.paged`: rotary positions and the write of K and V in one
pass, pages reserved, forked and freed on the device, attention that reads a
shared prompt once for all its samples, or a chosen part of a long context.
The batched decoder of the native library (``MegakernelBatchDecoder``) is the
faster one for sequences that share nothing.

The reference decodes one sequence from one contiguous cache; there is no
counterpart.  Numerics follow it: activations, residual stream, norms and
softmax in fp32, K/V and RoPE tables in bf16; q is rounded to bf16 too, the
cache operators' type.
"""
from __future__ import annotations

from collections import Counter
from itertools import count
from typing import List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

from .paged import BAD_TOKEN, PagedKVCache, to_device
from .weights import (HEAD_DIM, NUM_KV_HEADS, NUM_Q_HEADS, Q_SIZE, KV_SIZE, RMS_NORM_EPS, Qwen3Weights, rope_tables)


def _rms_norm(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + RMS_NORM_EPS) * w


def _product(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """fp32 activations by bf16 weights ``[out, in]``, fp32 result: the activations as two bf16 pieces, side by side in
    one product, so that the weights are read once and the activations are not rounded."""
    x = x.float()
    hi = x.to(w.dtype)
    y = torch.mm(torch.cat([hi, (x - hi.float()).to(w.dtype)]), w.T, out_dtype=torch.float32)
    return y[:x.shape[0]] + y[x.shape[0]:]


class PagedDecoder:
    """``max_seqs`` sequences on a pool of ``num_pages`` pages.

    ``sparse_pages``: decode steps read at most this many pages per query and
    kv head (chosen by score); ``None`` reads everything.

    The host keeps account of lengths and pages, so a call that the cache would
    refuse raises before anything is changed on either side.  :meth:`check`
    raises what the device found all the same (the cache used directly, say) and
    takes lengths and pages over from there.
    """

    def __init__(self, weights: Qwen3Weights, num_pages: int, max_seqs: int, max_seq_len: int = 4096, page_size: int = 64,
                 sparse_pages: Optional[int] = None):
        dev = weights.embed.device
        self.embed, self.final_norm, self.sparse_pages = weights.embed, weights.final_norm.float(), sparse_pages
        self.layers = []
        for layer in weights.layers:
            self.layers.append({
                "qkv": torch.cat([layer["q_proj"], layer["k_proj"], layer["v_proj"]]),
                "gate_up": torch.cat([layer["gate_proj"], layer["up_proj"]]),
                **{k: layer[k] for k in ("o_proj", "down_proj")},
                **{k: layer[k].float() for k in ("input_layernorm", "post_attention_layernorm", "q_norm", "k_norm")},
            })
        cos, sin = rope_tables(max_seq_len, device=dev)   # the reference's bf16 values, one half of the duplicated columns
        self.cos, self.sin = (x[:, :HEAD_DIM // 2].float().contiguous() for x in (cos, sin))
        self.cache = PagedKVCache(num_pages, max_seqs, -(-max_seq_len // page_size), num_layers=len(self.layers),
                                  page_size=page_size, device=dev, index=sparse_pages is not None)
        self.max_seq_len = max_seq_len
        self._families = 0
        self._take_over()

    def _take_over(self) -> None:
        """Lengths and pages as the device has them (synchronises)."""
        c = self.cache
        self.lengths: List[int] = c.lengths.tolist()
        table = c.page_table.tolist()
        # each sequence's pages, and how many sequences hold a page; pages handed out from here on get names of their own
        self._pages = [row[:-(-n // c.page_size)] for row, n in zip(table, self.lengths)]
        self._held = Counter(p for row in self._pages for p in row)
        self._free_pages = c.free_pages()
        self._names = count(c.refs.numel())
        self._family: List[Optional[Tuple[int, int]]] = [None] * len(self.lengths)   # (family, pages it shares)
        self._plan = None

    def _grow(self, slots: Sequence[int], lengths: Sequence[int]) -> None:
        """Accounts for sequences that grow; raises without a change where the pages do not suffice."""
        need = [-(-n // self.cache.page_size) - len(self._pages[s]) for s, n in zip(slots, lengths)]
        if sum(need) > self._free_pages:
            raise RuntimeError("paged cache: not enough free pages")
        self._free_pages -= sum(need)
        for s, n, k in zip(slots, lengths, need):
            new = [next(self._names) for _ in range(k)]
            self._pages[s] += new
            self._held.update(new)
            self.lengths[s] = n

    def _known(self, slots: Sequence[int]) -> None:
        if len(set(slots)) != len(slots) or any(not 0 <= s < len(self.lengths) for s in slots):
            raise ValueError("a sequence is named twice or out of range")

    def _ints(self, x, dtype: torch.dtype = torch.int32) -> torch.Tensor:
        return to_device(x, dtype, self.embed.device)

    def _tokens(self, ids, n: int) -> torch.Tensor:
        """n token ids on the device.  One out of range raises if it is known on the host; on the device it is read as
        the nearest one and :meth:`check` raises."""
        ids = torch.as_tensor(ids)
        if ids.numel() != n or (n and ids.is_floating_point()):   # (an empty list becomes a float tensor)
            raise ValueError("there must be one token id for each sequence")
        ids, top = ids.reshape(-1), self.embed.shape[0] - 1
        if ids.device.type == "cpu":
            if n and not 0 <= int(ids.min()) <= int(ids.max()) <= top:
                raise ValueError("token id out of range")
            return self._ints(ids, torch.int64)
        ids = ids.to(self.embed.device).long()
        safe = ids.clamp(0, top)
        status = self.cache.status
        status.copy_(torch.where((safe != ids).any() & (status == 0), BAD_TOKEN, status))
        return safe

    def _forward(self, ids, slots, positions, attend) -> torch.Tensor:
        """Hidden states of the tokens after the final norm; ``attend(layer, q)`` reads the cache."""
        h = self.embed[ids].float()
        n = h.shape[0]
        for li, w in enumerate(self.layers):
            x = _rms_norm(h, w["input_layernorm"])
            q, k, v = _product(x, w["qkv"]).split([Q_SIZE, KV_SIZE, KV_SIZE], -1)
            q = _rms_norm(q.view(n, NUM_Q_HEADS, HEAD_DIM), w["q_norm"]).to(self.embed.dtype)
            k = _rms_norm(k.view(n, NUM_KV_HEADS, HEAD_DIM), w["k_norm"]).to(self.embed.dtype)
            v = v.view(n, NUM_KV_HEADS, HEAD_DIM).to(self.embed.dtype)
            q = self.cache.append(li, q, k, v, slots, positions, self.cos, self.sin)
            h = h + _product(attend(li, q).view(n, Q_SIZE), w["o_proj"])
            x = _rms_norm(h, w["post_attention_layernorm"])
            gate, up = _product(x, w["gate_up"]).chunk(2, -1)
            h = h + _product(F.silu(gate) * up, w["down_proj"])
        return _rms_norm(h, self.final_norm)

    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        return _product(h, self.embed)

    @torch.no_grad()
    def prefill(self, slot: int, ids: Sequence[int]) -> torch.Tensor:
        """Appends a prompt (or a further piece of one) to a sequence; fp32 logits of its last token."""
        self._known([slot])
        n, start = len(ids), self.lengths[slot]
        if n < 1 or start + n > self.max_seq_len:
            raise ValueError("prompt is empty or exceeds max_seq_len")
        ids = self._tokens(ids, n)
        self._grow([slot], [start + n])
        self.cache.reserve([slot], [start + n])
        one = self._ints([slot])
        starts = self._ints([0, n])
        h = self._forward(ids, one.expand(n).contiguous(),
                          torch.arange(start, start + n, dtype=torch.int32, device=self.embed.device),
                          lambda li, q: self.cache.attend(li, q, one, q_starts=starts))
        return self._logits(h[-1:])[0]

    def fork(self, parent: int, children: Sequence[int]) -> None:
        """Empty slots become copies of a sequence; decode steps read what they share once for all of them."""
        children = list(children)
        self._known([parent, *children])
        if any(self.lengths[s] for s in children):
            raise ValueError("a child must be an empty slot")
        full, part = divmod(self.lengths[parent], self.cache.page_size)
        if part and len(children) > self._free_pages:
            raise RuntimeError("paged cache: not enough free pages")
        if not children:
            return
        self.cache.fork([parent] * len(children), children)
        shared = self._pages[parent][:full]
        for s in children:
            self._pages[s] = list(shared)
            self._held.update(shared)
        self._grow(children, [self.lengths[parent]] * len(children))
        for s in [parent, *children]:
            self._family[s] = (self._families, full)
        self._families += 1
        self._plan = None

    def free(self, slots: Sequence[int]) -> None:
        slots = list(slots)
        self._known(slots)
        self.cache.free(slots)
        for s in slots:
            for p in self._pages[s]:
                self._held[p] -= 1
                if not self._held[p]:
                    del self._held[p]
                    self._free_pages += 1
            self._pages[s], self.lengths[s], self._family[s] = [], 0, None
        self._plan = None

    def _groups(self, slots):
        """Order of the batch that puts families side by side, and their starts and pages; kept while the batch stays."""
        key = tuple(slots)
        if self._plan is None or self._plan[0] != key:
            order = sorted(range(len(slots)), key=lambda i: (self._family[slots[i]] is None, self._family[slots[i]] or (0, 0)))
            starts, pages = [], []
            last = object()
            for at, i in enumerate(order):
                f = self._family[slots[i]]
                if f is None:
                    break
                if f != last:
                    starts.append(at)
                    pages.append(f[1])
                    last = f
            else:
                at = len(order)
            groups = (self._ints(starts + [at]), self._ints(pages)) if starts else (None, None)
            back = self._ints(order, torch.int64)
            self._plan = (key, order, back, self._ints([slots[i] for i in order]), *groups)
        return self._plan[1:]

    @torch.no_grad()
    def step(self, slots: Sequence[int], tokens: torch.Tensor) -> torch.Tensor:
        """One token for each of the named sequences: fp32 logits ``[len(slots), vocab]``.  No host synchronisation."""
        slots = list(slots)
        self._known(slots)
        if any(self.lengths[s] >= self.max_seq_len for s in slots):
            raise ValueError("a sequence is full")
        tokens = self._tokens(tokens, len(slots))
        if not slots:
            return self.embed.new_empty((0, self.embed.shape[0]), dtype=torch.float32)
        self._grow(slots, [self.lengths[s] + 1 for s in slots])
        _, back, dev_slots, starts, pages = self._groups(slots)
        positions = self.cache.lengths[dev_slots]
        self.cache.reserve(dev_slots, positions + 1)
        if self.sparse_pages is None:
            def attend(li, q):
                return self.cache.attend(li, q, dev_slots, group_starts=starts, prefix_pages=pages)
        else:
            def attend(li, q):
                return self.cache.sparse_attend(li, q, dev_slots, positions, self.sparse_pages)[0]
        h = self._forward(tokens[back], dev_slots, positions, attend)
        out = torch.empty_like(h)
        out[back] = h
        return self._logits(out)

    def check(self) -> None:
        """Raises if a device-side check failed, with lengths and pages then as the device has them (synchronises)."""
        try:
            self.cache.check()
        except RuntimeError:
            self._take_over()
            raise
