"""A `choose` that is interrupted leaves the decoder as after a step, like one that raises."""
from __future__ import annotations

import pytest
import torch

from test_serving_gpu import decoder, prompt_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [KeyboardInterrupt, SystemExit, ZeroDivisionError])
def test_interrupted_choice(kind):
    prompt = prompt_of(20, 3)
    dec, other = decoder(), decoder()
    for d in (dec, other):
        d.prefill(1, prompt)

    def choose(logits):
        raise kind

    with pytest.raises(kind):
        dec.verify([1], [[5, 6, 7]], [[-1, 0, 1]], choose)
    other.step([1], torch.tensor([5], device="cuda"))
    for d in (dec, other):
        d.check()
        assert d.lengths[1] == 21 and d.cache.lengths[1].item() == 21
    assert dec.cache.free_pages() == other.cache.free_pages()
    a, b = (d.step([1], torch.tensor([9], device="cuda")) for d in (dec, other))
    assert (a - b).abs().max().item() < 3e-2
