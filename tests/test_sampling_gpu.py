"""Sampling against the definition in 64 bits (numpy), exactly: a token is a whole number, and the kernel's sums are exact, so
that only a draw within 2^-40 of a border between two tokens could differ."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def sample():
    from megaqwen_b200.sampling import sample
    return sample


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def row_token(x, u, t, k, p, lowest):
    """One row, 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    best = int(np.argmax(x))
    if x[best] == -np.inf:
        return -1
    if not t > 0:
        return best
    with np.errstate(invalid="ignore"):
        w = np.where(x == x[best], 1.0, np.exp((x - x[best]) / t))
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:int(k)]
    if p < 1:
        acc = np.cumsum(w[order])
        before = acc - w[order]
        order = order[:max(1, int((before < p * acc[-1]).sum()))]
    keep = np.sort(order[w[order] >= min(lowest, 1.0)]) if lowest > 0 else np.sort(order)
    acc = np.cumsum(w[keep])
    aim = max(u, 0.0) * acc[-1] if u == u else 0.0
    at = int((acc <= aim).sum())
    if at >= len(keep):   # the last one that can be drawn
        at = int(np.flatnonzero(w[keep] > 2.0 ** -44)[-1])
    return int(keep[at])


def expect(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    n = logits.shape[0]

    def each(x):
        return x.tolist() if torch.is_tensor(x) else [float(np.float32(x))] * n

    x = logits.double().cpu().numpy()
    args = [each(v) for v in (u, temperature, top_k, top_p, min_p)]
    return [row_token(x[i], *(a[i] for a in args)) for i in range(n)]


def check(sample, logits, u, **kw):
    got = sample(logits, u, **kw)
    assert got.dtype == torch.int32 and got.shape == (logits.shape[0],)
    assert got.tolist() == expect(logits, u, **kw)


def rows(g, n, vocab, dtype, std=2.5):
    x = torch.randn(n, vocab, device="cuda", generator=g) * std
    if vocab > 50:   # a few candidates that stand out
        at = torch.randint(0, vocab, (n, 30), device="cuda", generator=g)
        x.scatter_add_(1, at, torch.rand(n, 30, device="cuda", generator=g) * 9)
    return x.to(dtype)


RULES = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=5.0), dict(top_k=1), dict(top_k=40), dict(top_k=5000),
         dict(top_p=0.9), dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0),
         dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.02), dict(temperature=1.5, top_k=3000, top_p=0.7),
         dict(top_p=0.99999, min_p=1e-4)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 100, 1000, 4096, 4097, 50257, 151936])
@pytest.mark.parametrize("rule", RULES, ids=lambda r: "-".join(f"{k}{v}" for k, v in r.items()) or "plain")
def test_rules(sample, dtype, vocab, rule):
    g = gen(vocab)
    n = 5 if vocab > 5000 else 17
    check(sample, rows(g, n, vocab, dtype), torch.rand(n, device="cuda", generator=g), **rule)


@pytest.mark.parametrize("dtype", TYPES)
def test_largest_vocabulary(sample, dtype):
    """A row that shared memory holds, and one that it does not."""
    for vocab in (300001, 1 << 20):
        g = gen(3)
        x, u = rows(g, 2, vocab, dtype), torch.rand(2, device="cuda", generator=g)
        for rule in (dict(), dict(top_p=0.9), dict(top_k=100, top_p=0.9), dict(top_k=20000)):
            check(sample, x, u, **rule)


@pytest.mark.parametrize("dtype", TYPES)
def test_parameters_per_row(sample, dtype):
    g, gc, n, vocab = gen(5), torch.Generator().manual_seed(5), 96, 32003

    def among(values, t):
        return torch.tensor(values, dtype=t)[torch.randint(0, len(values), (n,), generator=gc)].cuda()

    x = rows(g, n, vocab, dtype)
    x[::7, 10:] = -math.inf
    kw = dict(temperature=among([0.0, 0.5, 1.0, 2.0, -1.0, math.nan], torch.float32),
              top_k=among([0, -1, 1, 7, 50, 1025, 40000], torch.int32),
              top_p=among([0.0, 0.3, 0.95, 1.0, 1.5, math.nan], torch.float32),
              min_p=among([0.0, 0.01, 0.3, 1.0, 2.0, -1.0], torch.float32))
    u = torch.rand(n, device="cuda", generator=g)
    check(sample, x, u, **kw)
    # a row's token does not depend on the rows beside it
    got = sample(x, u, **kw)
    for i in (0, 13, 95):
        assert sample(x[i:i + 1], u[i:i + 1], **{k: v[i:i + 1] for k, v in kw.items()}).item() == got[i].item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rule", [dict(), dict(top_k=700), dict(top_k=70000), dict(top_p=0.5), dict(top_k=90000, top_p=0.9),
                                  dict(min_p=0.5)])
def test_flat_and_equal_rows(sample, dtype, rule):
    """Borders among thousands of equal logits: the lowest numbers stay."""
    g, vocab = gen(6), 100003
    x = torch.zeros(6, vocab, device="cuda", dtype=dtype)
    x[1, ::2] = 1.0
    x[2] = (torch.arange(vocab, device="cuda") % 3).to(dtype)
    x[3] = -0.0
    x[3, ::5] = 0.0
    x[4] = (torch.randn(vocab, device="cuda", generator=g) * 1e-3).to(dtype)
    x[5] = (torch.randn(vocab, device="cuda", generator=g) * 0.3).to(torch.bfloat16).to(dtype)
    for u in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
        check(sample, x, torch.full((6,), u, device="cuda"), **rule)


@pytest.mark.parametrize("rule", [dict(), dict(top_k=3), dict(top_k=2000), dict(top_p=0.9), dict(top_k=10, top_p=0.5, min_p=0.1),
                                  dict(temperature=1e-30), dict(temperature=1e30), dict(temperature=0.0)])
def test_odd_logits(sample, rule):
    """Masks of the lowest value, infinities, NaN, huge and tiny logits."""
    vocab = 20011
    x = rows(gen(7), 12, vocab, torch.float32)
    x[0, 5:] = torch.finfo(torch.float32).min
    x[1, :-3] = -math.inf
    x[2] = -math.inf
    x[3] = math.nan
    x[4, ::3] = math.nan
    x[5, 77] = math.inf
    x[6, 1234:1240] = math.inf
    x[7] *= 1e30
    x[8] *= 1e-30
    x[9, :] = -3e38
    x[9, 400] = 3e38
    x[10, 20:] = -1e9
    x[11, 100:] = -65504.0
    if rule.get("temperature", 1) > 1e29:
        x = x[[0, 4, 7, 8, 10, 11]]   # where a difference over the temperature is a number
    check(sample, x, torch.linspace(0, 0.99, len(x), device="cuda"), **rule)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rule", [dict(top_k=2), dict(top_k=30), dict(top_k=5000), dict(top_p=0.4), dict(top_p=0.95), dict(min_p=0.999),
                                  dict(top_p=0.4, temperature=1e-37), dict(top_p=0.9, temperature=1e-42),
                                  dict(top_k=7000, top_p=0.9, temperature=1e-42), dict(top_p=0.4, temperature=1e-7)])
def test_next_to_the_largest(sample, dtype, rule):
    """The next logits are one step of the type below the largest, or subnormal steps."""
    g, vocab = gen(13), 20011
    x = rows(g, 5, vocab, dtype)
    up = 1024 if dtype == torch.float16 else 2.0 ** 20
    step = torch.finfo(dtype).eps / 2   # below a power of two
    at = torch.randint(0, vocab, (5, 40), device="cuda", generator=g)
    x.scatter_(1, at, (up * (1 - step * (torch.arange(40, device="cuda") % 4))).to(dtype).expand(5, -1))
    x[1] = (torch.arange(vocab, device="cuda") % 5 == 0).to(dtype) * torch.finfo(dtype).tiny
    x[2] = torch.where(torch.arange(vocab, device="cuda") % 7 == 0, 1.0, 1.0 - step).to(dtype)
    x[3, 100:] = -math.inf
    check(sample, x, torch.rand(5, device="cuda", generator=g), **rule)


@pytest.mark.parametrize("rule", [dict(), dict(top_p=0.3), dict(top_p=0.95), dict(top_k=700, top_p=0.6), dict(top_k=9000, top_p=0.6)])
def test_differences_past_the_largest_number(sample, rule):
    """Logits further apart than fp32 goes, at temperatures that bring them together."""
    g, vocab = gen(14), 20011
    x = (torch.rand(4, vocab, device="cuda", generator=g) * 2 - 1) * 3.3e38
    x[2, 9:] = -3e38
    t = torch.tensor([3e38, 1e38, 2e38, 3e37], device="cuda")
    check(sample, x, torch.rand(4, device="cuda", generator=g), temperature=t, **rule)
    flat = torch.full((4,), math.inf, device="cuda")    # all weights alike
    check(sample, x, torch.rand(4, device="cuda", generator=g), temperature=flat, **rule)


def test_numbers_at_the_ends(sample):
    x = rows(gen(8), 6, 5003, torch.float32)
    u = torch.tensor([0.0, -1.0, 1.0, 2.0, math.nan, 1 - 2.0 ** -24], device="cuda")
    for rule in (dict(), dict(top_k=9), dict(top_p=0.5)):
        check(sample, x, u, **rule)


def test_many_draws_of_one_row(sample):
    """Every draw of 1000 from one row: also where sums in 32 bits would end one token off."""
    g = gen(9)
    x = (torch.randn(1, 151936, device="cuda", generator=g) * 0.5).expand(1000, -1)
    check(sample, x, torch.rand(1000, device="cuda", generator=g))


@pytest.mark.parametrize("rule", [dict(top_p=0.5), dict(top_p=0.9), dict(top_p=0.3, min_p=0.01), dict(top_k=40, top_p=0.9), dict(top_k=700),
                                  dict()])
def test_many_rows_many_times(sample, rule):
    """More clusters than fit the GPU at once, again and again: always the same tokens."""
    g = gen(12)
    x, u = rows(g, 64, 151936, torch.float32, 2.0), torch.rand(64, device="cuda", generator=g)
    x[::9, 7000:] = -math.inf
    want = sample(x, u, **rule)
    assert want.tolist() == expect(x, u, **rule)
    for _ in range(30):
        assert torch.equal(sample(x, u, **rule), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_offsets(sample, dtype):
    g = gen(10)
    x = rows(g, 7, 3001, dtype)
    u = torch.rand(7, device="cuda", generator=g)
    want = sample(x, u, top_p=0.9).tolist()
    for pad, lo in ((1, 0), (3, 2), (16, 5)):
        wide = torch.full((7, 3001 + pad + lo), 50.0, dtype=dtype, device="cuda")
        wide[:, lo:lo + 3001] = x
        assert sample(wide[:, lo:lo + 3001], u, top_p=0.9).tolist() == want
    assert sample(x.T.contiguous().T, u, top_p=0.9).tolist() == want
    assert sample(x.flip(0), u.flip(0), top_p=0.9).tolist() == want[::-1]


def test_other_stream_and_graph(sample):
    g = gen(11)
    x, u = rows(g, 30, 40000, torch.float32), torch.rand(30, device="cuda", generator=g)
    k = torch.full((30,), 20, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample(x, u, top_k=k, top_p=0.9)
    side.synchronize()
    assert got.tolist() == expect(x, u, top_k=k, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample(x, u, top_k=k, top_p=0.9)
        again = sample(x, u, top_k=k)
    for i in range(3):
        u.copy_(torch.rand(30, device="cuda", generator=g))
        k.fill_(3 + 4 * i)
        graph.replay()
        assert out.tolist() == expect(x, u, top_k=k, top_p=0.9) and again.tolist() == expect(x, u, top_k=k)


def test_refusals(sample):
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    for args in ((x[0], u), (x[None], u), (x.double(), u), (x.int(), u), (x, u[:2]), (x, u.double()), (x, u.cpu()), (x.cpu(), u),
                 (x[:, :0], u), (x, torch.zeros(6, device="cuda")[::2]), (torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1])):
        with pytest.raises(RuntimeError):
            sample(*args)
    for kw in (dict(temperature=-0.1), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_p=1.1), dict(top_p=-0.1),
               dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=math.nan), dict(top_k=1.5), dict(top_k=2 ** 40), dict(temperature="1"),
               dict(temperature=u.double()), dict(temperature=u[:2]), dict(top_k=u), dict(top_k=u.long()), dict(top_p=u.half()),
               dict(min_p=u.cpu()), dict(top_p=None)):
        with pytest.raises(RuntimeError):
            sample(x, u, **kw)
    assert sample(x[:0], u[:0]).shape == (0,)
