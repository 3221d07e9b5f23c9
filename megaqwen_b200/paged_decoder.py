"""Qwen3 decoding on the paged KV cache: prompts shared between samples.

:class:`PagedDecoder` runs the model of this package with its projections as
plain matrix products and everything around the cache on the operators of
:mod:`megaqwen_b200.paged`: rotary positions and the write of K and V in one
pass, pages reserved, forked and freed on the device, attention that reads a
shared prompt once for all its samples, a chosen part of a long context, or a
window of it; and trees of drafted tokens checked in one pass.  Tokens are drawn
from the logits by :mod:`megaqwen_b200.sampling`.
The batched decoder of the native library (``MegakernelBatchDecoder``) is the
faster one for sequences that share nothing.

The reference decodes one sequence from one contiguous cache; there is no
counterpart.  Numerics follow it: activations, residual stream, norms and
softmax in fp32, K/V and RoPE tables in bf16; q is rounded to bf16 too, the
cache operators' type.
"""
from __future__ import annotations

from collections import Counter
from itertools import accumulate, count
from typing import Callable, List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

from .paged import BAD_TOKEN, PagedKVCache, to_device
from .sampling import sample
from .weights import (HEAD_DIM, NUM_KV_HEADS, NUM_Q_HEADS, Q_SIZE, KV_SIZE, RMS_NORM_EPS, Qwen3Weights, rope_tables)

MAX_NODES = 256   # of a drafted tree


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
    kv head (chosen by score); ``None`` reads everything.  ``window``: a token
    sees the last ``window`` positions, itself among them, and the first
    ``sinks``, in prompts and in steps; not together with ``sparse_pages``.

    The host keeps account of lengths and pages, so a call that the cache would
    refuse raises before anything is changed on either side.  :meth:`check`
    raises what the device found all the same (the cache used directly, say) and
    takes lengths and pages over from there.
    """

    def __init__(self, weights: Qwen3Weights, num_pages: int, max_seqs: int, max_seq_len: int = 4096, page_size: int = 64,
                 sparse_pages: Optional[int] = None, window: Optional[int] = None, sinks: int = 0):
        if window is not None and sparse_pages is not None:
            raise ValueError("window and sparse_pages exclude each other")
        if sinks < 0 or (window is None and sinks) or (window is not None and window < 1):
            raise ValueError("window must be positive, and sinks go with a window")
        self.window, self.sinks = window, sinks
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

    def _forward(self, ids, slots, positions, attend, places=None) -> torch.Tensor:
        """Hidden states of the tokens after the final norm; ``attend(layer, q)`` reads the cache.  Keys lie at ``places``,
        or at the positions."""
        h = self.embed[ids].float()
        n = h.shape[0]
        for li, w in enumerate(self.layers):
            x = _rms_norm(h, w["input_layernorm"])
            q, k, v = _product(x, w["qkv"]).split([Q_SIZE, KV_SIZE, KV_SIZE], -1)
            q = _rms_norm(q.view(n, NUM_Q_HEADS, HEAD_DIM), w["q_norm"]).to(self.embed.dtype)
            k = _rms_norm(k.view(n, NUM_KV_HEADS, HEAD_DIM), w["k_norm"]).to(self.embed.dtype)
            v = v.view(n, NUM_KV_HEADS, HEAD_DIM).to(self.embed.dtype)
            q = self.cache.append(li, q, k, v, slots, positions, self.cos, self.sin, places=places)
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
        if self.window is None:
            def attend(li, q):
                return self.cache.attend(li, q, one, q_starts=starts)
        else:
            def attend(li, q):
                return self.cache.window_attend(li, q, one, self.window, self.sinks, q_starts=starts)
        h = self._forward(ids, one.expand(n).contiguous(),
                          torch.arange(start, start + n, dtype=torch.int32, device=self.embed.device), attend)
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
        if self.window is not None:
            def attend(li, q):
                return self.cache.window_attend(li, q, dev_slots, self.window, self.sinks)
        elif self.sparse_pages is None:
            def attend(li, q):
                return self.cache.attend(li, q, dev_slots, group_starts=starts, prefix_pages=pages)
        else:
            def attend(li, q):
                return self.cache.sparse_attend(li, q, dev_slots, positions, self.sparse_pages)[0]
        h = self._forward(tokens[back], dev_slots, positions, attend)
        out = torch.empty_like(h)
        out[back] = h
        return self._logits(out)

    @staticmethod
    def draw(logits: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             generator: Optional[torch.Generator] = None) -> torch.Tensor:
        """A token for each row of logits (int32), drawn with ``generator``'s random numbers by the rules of
        :func:`megaqwen_b200.sampling.sample`.  No host synchronisation."""
        logits = logits.reshape(-1, logits.shape[-1])
        u = torch.rand(logits.shape[0], generator=generator, device=logits.device)
        return sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)

    @torch.no_grad()
    def verify(self, slots: Sequence[int], tokens: Sequence[Sequence[int]], parents: Sequence[Sequence[int]],
               choose: Optional[Callable[[torch.Tensor], torch.Tensor]] = None) -> List[List[int]]:
        """Drafted trees checked in one pass: the tokens that each sequence goes on with.

        ``tokens[i]`` are the nodes of sequence ``slots[i]``, at most 256, the first one the token that a step would take
        next; ``parents[i]`` their parents' numbers, -1 for the first and smaller than the node's own for the others.
        ``choose(logits)`` picks a token at each node, all sequences' nodes one after another (the largest logit, or
        :meth:`draw` with its arguments).  A sequence keeps the first node and those drafted ones that were chosen at
        the node before them, and the list returned holds the tokens chosen at the kept nodes: its last one is not in the
        cache yet.  The other nodes' room is given back.  Where ``choose`` raises, each sequence keeps its first node, as
        after a step.  Reads the whole context, whatever ``sparse_pages``; synchronises, for the counts.
        """
        slots, tokens, parents = list(slots), [list(t) for t in tokens], [list(p) for p in parents]
        self._known(slots)
        if self.window is not None:
            raise ValueError("drafted trees are not checked through a window")
        if len(tokens) != len(slots) or [len(t) for t in tokens] != [len(p) for p in parents]:
            raise ValueError("there must be a tree for each sequence and a parent for each node")
        depths: List[int] = []
        for t in parents:
            if not 1 <= len(t) <= MAX_NODES or t[0] != -1 or any(not 0 <= up < i for i, up in enumerate(t) if i):
                raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, each behind its parent, and one root")
            first = len(depths)
            for up in t:
                depths.append(depths[first + up] + 1 if up >= 0 else 0)
        sizes = [len(t) for t in tokens]
        old = [self.lengths[s] for s in slots]
        ends = [n + k for n, k in zip(old, sizes)]
        if any(n > self.max_seq_len for n in ends):
            raise ValueError("a sequence would exceed max_seq_len")
        ids = self._tokens([x for t in tokens for x in t], sum(sizes))
        if not slots:
            return []
        self._grow(slots, ends)
        dev_slots, nodes = self._ints(slots), self._ints([x for t in tokens for x in t])
        self.cache.reserve(dev_slots, ends)
        up = self._ints([x for t in parents for x in t])
        starts = self._ints([0, *accumulate(sizes)])
        base = [n for n, k in zip(old, sizes) for _ in range(k)]
        positions = self._ints([n + d for n, d in zip(base, depths)])
        places = self._ints([n + i for n, k in zip(old, sizes) for i in range(k)])
        h = self._forward(ids, self._ints([s for s, k in zip(slots, sizes) for _ in range(k)]), positions,
                          lambda li, q: self.cache.tree_attend(li, q, dev_slots, up, q_starts=starts), places)
        logits = self._logits(h)
        failed = None
        try:
            chosen = self.draw(logits, temperature=0.0) if choose is None else choose(logits)
            if chosen.numel() != nodes.numel():
                raise ValueError("there must be a chosen token for each node")
            chosen = self._ints(chosen.reshape(-1))
        except BaseException as e:   # (a step has no such callback: the trees must not stay in the cache)
            failed, chosen = e, torch.full_like(nodes, -1)
        _, emitted, count = self.cache.accept(dev_slots, up, nodes, chosen, q_starts=starts)
        emitted, kept = emitted.tolist(), count.tolist()
        if not all(kept):   # refused on the device, where nothing was cut
            self._take_over()
            self.check()
            raise RuntimeError("paged cache: the trees were refused")
        out, at = [], 0
        for s, n, size, k in zip(slots, old, sizes, kept):
            out.append(emitted[at:at + k])
            at += size
            self.lengths[s] = n + k
            full = -(-(n + k) // self.cache.page_size)
            for p in self._pages[s][full:]:   # no one else's: they were reserved for the tree
                del self._held[p]
                self._free_pages += 1
            del self._pages[s][full:]
        if failed is not None:
            raise failed
        return out

    def check(self) -> None:
        """Raises if a device-side check failed, with lengths and pages then as the device has them (synchronises)."""
        try:
            self.cache.check()
        except RuntimeError:
            self._take_over()
            raise
