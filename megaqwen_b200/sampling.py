"""Tokens drawn from logits.

``sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)``: int32
``[rows]``, a token for each row of ``logits`` ``[rows, vocab]`` (fp32, bf16 or
fp16 on the GPU, vocab at most 2^20) by the random number ``u[i]`` in [0, 1)
(fp32 ``[rows]``).  Each parameter is a number for all rows or a tensor with one
for each (``top_k`` int32, the others fp32).  With ``w = exp((logit - largest) /
temperature)`` there stay, in this order,

* the ``top_k`` largest logits (0: all; equal ones in the order of their numbers),
* of those, in descending order, the tokens before which less than ``top_p`` of
  their sum of ``w`` lies,
* of those, the tokens with ``w >= min_p`` (the largest has 1),

and the token is the first, in ascending order of the number, up to which the
sum of ``w`` over what stays exceeds ``u`` times its total.  Weights are held in
64 bits and summed exactly: the same inputs give the same token on every run, and
in any batch.  A temperature of 0 takes the largest logit.  Minus infinity (or
NaN) is never drawn, and a row of nothing else gives -1.  Nothing synchronises;
the call can be captured into a CUDA graph.

The reference decodes greedily only (its argmax is part of the decode kernel);
there is no counterpart.
"""
from __future__ import annotations

from . import _C

sample = _C.sample
