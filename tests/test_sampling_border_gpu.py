"""The border of a nucleus where logits lie closer together than the histogram's bins can be told apart."""
from __future__ import annotations

import pytest
import torch

from test_sampling_gpu import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sample():
    from megaqwen_b200.sampling import sample
    return sample


@pytest.mark.parametrize("step,temperature", [(5e-38, 1e-37), (2e-38, 1e-37), (5e-38, 4e-37), (3e-39, 1e-38), (1e-44, 1e-44)])
@pytest.mark.parametrize("top_p", [0.05, 0.2, 0.35, 0.5, 0.8, 0.99])
def test_a_spread_below_the_bins(sample, step, temperature, top_p):
    """A row whose largest and smallest logits are so near one another that 2048 bins between them have no width in fp32."""
    for counts in ((1, 100, 100), (1, 1000, 6000), (5, 3, 2), (1, 1, 1), (300, 20000, 40000)):
        x = torch.cat([torch.full((n,), -i * step) for i, n in enumerate(counts)])
        g = torch.Generator().manual_seed(len(x))
        x = torch.stack([x, x[torch.randperm(len(x), generator=g)]]).cuda()
        for u in (0.0, 0.4, 0.999):
            check(sample, x, torch.full((2,), u, device="cuda"), temperature=temperature, top_p=top_p)
