"""The border of a nucleus where it is a matter of the last unit (weights are held in units of 2^-43 of the largest, sums of them
are exact), and where logits lie closer together than the histogram's bins can be told apart."""
from __future__ import annotations

import math

import pytest
import torch

from test_sampling_gpu import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sample():
    from megaqwen_b200.sampling import sample
    return sample


# exp(-APART / HEAT) = 2^-10 (1 + 2^-37): 2^33 units and a sixteenth
HEAT, APART = 1.7486757040023804, 12.120896339416504


@pytest.mark.parametrize("ones,many", [(3, 1024), (36, 65536), (1, 7168), (100, 102400)])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_border_of_exact_sums(sample, ones, many, offset):
    """`ones` tokens of weight 1 and `many` of 2^33 units: half of the sum is a whole number of tokens, and the next does not
    stay.  The same from a row that lies anywhere in memory, alone and beside others, and with a top_k that leaves out only a
    token that is never drawn."""
    ones += many // 1024 % 2 != ones % 2   # an even sum
    vocab = ones + many + 1
    x = torch.full((vocab,), -APART)
    x[:ones] = 0.0
    x[-1] = -math.inf
    total = ones * 2 ** 43 + many * 2 ** 33
    half = total // 2
    kept = [2 ** 43] * ones + [2 ** 33] * many
    lies = 0
    for last, v in enumerate(kept):   # in descending order, which is that of the numbers
        if lies >= half:
            break
        lies += v
    assert lies == half and last < ones + many
    room = torch.zeros(3, vocab + 8, device="cuda")
    room[:, offset:offset + vocab] = x.cuda()
    rows = room[:, offset:offset + vocab]
    u = torch.full((3,), 1 - 2.0 ** -24, device="cuda")
    for kw in (dict(), dict(top_k=vocab - 1)):
        assert sample(rows, u, temperature=HEAT, top_p=0.5, **kw).tolist() == [last - 1] * 3
        assert sample(rows[1:2], u[:1], temperature=HEAT, top_p=0.5, **kw).tolist() == [last - 1]


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
