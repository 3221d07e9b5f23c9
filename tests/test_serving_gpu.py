"""Windows, drafted trees and drawn tokens in use: the paged decoder against the CPU oracle and plain attention."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from megaqwen_b200.weights import make_weights, seeded_prompt
from test_paged_accept_gpu import walk
from test_paged_gpu import Pool, dev, index_ref, normal

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
LAYERS = 2
# q, k and the attention output in bf16: the bound of the paged decoder's own tests
LOGIT_TOL = 3e-2
VOCAB = 151936


@pytest.fixture(scope="module")
def paged():
    from megaqwen_b200 import paged
    return paged


def decoder(**kw):
    from megaqwen_b200.paged_decoder import PagedDecoder
    return PagedDecoder(make_weights(LAYERS).to("cuda"), **{**dict(num_pages=40, max_seqs=5, max_seq_len=400, page_size=16), **kw})


def oracle_logits(tokens):
    from oracle.qwen3_cpu import Qwen3CpuOracle
    return Qwen3CpuOracle(make_weights(LAYERS), max_seq_len=400).prefill(tokens)


def close(got, ref):
    err = (got.cpu() - ref.cpu()).abs().max().item()
    assert err < LOGIT_TOL, err


def prompt_of(n, seed):
    return seeded_prompt(n, seed=seed).tolist()


# ---- keys at places of their own ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,d,page,rot,inter", [
    (torch.bfloat16, 128, 16, 128, False), (torch.float16, 64, 32, 64, True), (torch.bfloat16, 128, 64, 18, False)])
@pytest.mark.parametrize("news", [[1], [40, 0, 7]])
def test_append_at_places(paged, dtype, d, page, rot, inter, news):
    """The rows are those of an append at the positions, bit for bit, and lie at the places."""
    hkv, hq, n = 3, 6, sum(news)
    p = Pool([70 + c for c in news], page, hkv, d, dtype, seed=page + n)
    cos, sin = paged.rope_tables(200, rot)
    q, k, v = normal(p.g, n, hq, d, dtype=dtype), normal(p.g, n, hkv, d, dtype=dtype), normal(p.g, n, hkv, d, dtype=dtype)
    slots = dev([p.slots[b] for b, c in enumerate(news) for _ in range(c)])
    places = [70 + i for c in news for i in range(c)]
    gc = torch.Generator().manual_seed(n)
    pos = dev(torch.randint(0, 200, (n,), generator=gc).tolist())
    idx = torch.full((p.k.shape[0], 2, hkv, 2 * d + 16), 99, dtype=torch.int8, device="cuda")
    k0, v0, status = p.k.clone(), p.v.clone(), dev([0])
    out = paged.rope_append(q, k, v, p.k, p.v, p.table, slots, pos, cos, sin, layer=1, interleaved=inter, index=idx,
                            status=status, places=dev(places))
    assert status.item() == 0
    assert torch.equal(out, paged.rope(q, pos, cos, sin, interleaved=inter))
    turned = paged.rope(k, pos, cos, sin, interleaved=inter)
    want_index, at = torch.full_like(idx, 99), 0
    for b, c in enumerate(news):
        for i in range(c):
            pg, row = p.rows[b][(70 + i) // page], (70 + i) % page
            k0[pg, 1, :, row], v0[pg, 1, :, row] = turned[at], v[at]
            at += 1
    for b, c in enumerate(news):
        for i in range(c):
            if (70 + i) % page == page - 1:
                pg = p.rows[b][(70 + i) // page]
                for h in range(hkv):
                    want_index[pg, 1, h] = 0
                    want_index[pg, 1, h, :2 * d + 1] = index_ref(k0[pg:pg + 1, 1, h])[0]
    assert torch.equal(p.k, k0) and torch.equal(p.v, v0) and torch.equal(idx, want_index)


def test_append_at_wrong_places(paged):
    p = Pool([40, 20], 16, 2, 64, torch.bfloat16)
    q = normal(p.g, 3, 4, 64)
    cos, sin = paged.rope_tables(64, 64)
    slots = dev([p.slots[0], p.slots[1], p.slots[1]])
    for pos, places, code in (([1, 2, 3], [39, -1, 19], 5), ([1, 2, 3], [39, 1 << 30, 19], 5), ([1, 2, 3], [39, 40, 19], 9),
                              ([1, 64, 3], [39, 18, 19], 5), ([1, -1, 3], [39, 18, 19], 5)):
        k0, status = p.k.clone(), dev([0])
        paged.rope_append(q, q[:, :2], q[:, 2:], p.k, p.v, p.table, slots, dev(pos), cos, sin, layer=0, status=status,
                          places=dev(places))
        assert status.item() == code
        diff = {tuple(x) for x in (p.k != k0).any(dim=(1, 2, 4)).nonzero().tolist()}
        assert diff <= {(p.rows[0][2], 7), (p.rows[1][1], 3)}
    with pytest.raises(RuntimeError, match="places"):
        paged.rope_append(q, q[:, :2], q[:, 2:], p.k, p.v, p.table, slots, dev([1, 2, 3]), cos, sin, layer=0, places=dev([1]))


# ---- windows -----------------------------------------------------------------------------------------------------

def plain_window(dec):
    """Puts attention in 64 bits over the cache's rows in the place of the decoder's."""
    c = dec.cache

    def attend(layer, q, slots, window, sinks=0, q_starts=None, scale=None):
        slots = slots.tolist()
        starts = q_starts.tolist() if q_starts is not None else list(range(len(slots) + 1))
        out = torch.empty_like(q)
        for b, s in enumerate(slots):
            n = int(c.lengths[s])
            at = torch.arange(n, device=q.device)
            pages = c.page_table[s].long()[at // c.page_size]
            k, v = (x[pages, layer, :, at % c.page_size].double() for x in (c.k_pages, c.v_pages))
            x = q[starts[b]:starts[b + 1]].double()
            pos = torch.arange(n - x.shape[0], n, device=q.device)[:, None]
            see = (at <= pos) & ((pos - at < window) | (at < sinks))
            k, v = (y.repeat_interleave(x.shape[1] // y.shape[1], 1) for y in (k, v))
            w = torch.einsum("qhd,khd->hqk", x, k) * x.shape[2] ** -0.5
            w = torch.softmax(w.masked_fill(~see, -torch.inf), -1)
            out[starts[b]:starts[b + 1]] = torch.einsum("hqk,khd->qhd", w, v).to(q.dtype)
        return out
    c.window_attend = attend
    return dec


@pytest.mark.parametrize("window,sinks", [(20, 0), (33, 4), (1, 1), (1000, 0)])
def test_windowed_decoder(window, sinks):
    """A prompt in two pieces, forks, a stranger, steps; and with a window past everything, the oracle."""
    a, b = prompt_of(90, 7), prompt_of(11, 8)
    got = []
    for dec in (decoder(window=window, sinks=sinks), plain_window(decoder(window=window, sinks=sinks))):
        rows = [dec.prefill(2, a[:50]), dec.prefill(2, a[50:]), dec.prefill(0, b)]
        dec.fork(2, [1, 4])
        for i in range(6):
            rows += list(dec.step([4, 0, 2], torch.tensor([5 + i, 9, 70000])))
        dec.check()
        got.append(torch.stack(rows))
    close(got[0], got[1])
    if window == 1000:
        close(got[0][1], oracle_logits(a)[-1])
        close(got[0][3 + 3 * 5], oracle_logits(a + [5, 6, 7, 8, 9, 10])[-1])


# ---- drafted trees -----------------------------------------------------------------------------------------------

def paths_of(parents):
    out = []
    for i, up in enumerate(parents):
        out.append((out[up] if up >= 0 else []) + [i])
    return out


def script(trees, parents, right):
    """A token for each node that is one of its children's where `right` says so."""
    out = []
    for t, p in zip(trees, parents):
        for i in range(len(t)):
            kids = [j for j, up in enumerate(p) if up == i]
            out.append(t[kids[-1]] if kids and right(i) else 1000 + i)
    return out


@pytest.mark.parametrize("page_size,sparse", [(16, None), (64, None), (16, 64)])
def test_verify_against_the_oracle(page_size, sparse):
    """Each node's logits are those of its path's tokens; what is kept goes on as if it had been prefilled."""
    dec = decoder(page_size=page_size, num_pages=640 // page_size, sparse_pages=sparse)
    texts = {0: prompt_of(61, 4), 3: prompt_of(30, 5)}
    for s, t in texts.items():
        dec.prefill(s, t)
    dec.fork(0, [2])
    texts[2] = list(texts[0])
    slots = [3, 0, 2]
    parents = [[-1, 0, 0, 1, 3, 2], [-1], [-1, 0, 1, 2, 3, 4, 5, 6, 7, 0]]
    for turn in range(3):
        trees = [[100 * s + 10 * turn + i for i in range(len(p))] for s, p in zip(slots, parents)]
        chosen = script(trees, parents, lambda i: (i + turn) % 4 != 3)
        seen = []

        def choose(logits):
            seen.append(logits)
            return torch.tensor(chosen)
        got = dec.verify(slots, trees, parents, choose)
        dec.check()
        at = 0
        for s, t, p, g in zip(slots, trees, parents, got):
            for i, path in enumerate(paths_of(p)):
                if turn < 2:
                    close(seen[0][at + i], oracle_logits(texts[s] + [t[j] for j in path])[-1])
            kept = walk(p, t, chosen[at:at + len(t)])
            assert g == [chosen[at + i] for i in kept]
            texts[s] += [t[i] for i in kept]
            at += len(t)
        assert dec.lengths == dec.cache.lengths.tolist() and all(dec.lengths[s] == len(texts[s]) for s in slots)
        assert dec._free_pages == dec.cache.free_pages()
        logits = dec.step(slots, torch.tensor([7, 8, 9]))
        for s, x, row in zip(slots, (7, 8, 9), logits):
            texts[s].append(x)
            close(row, oracle_logits(texts[s])[-1])
    # the largest logit, of a chain
    got = dec.verify([3], [[11, 12]], [[-1, 0]])[0]
    ref = oracle_logits(texts[3] + [11])[-1]
    assert ref[got[0]] > ref.max() - 2 * LOGIT_TOL and len(got) == (2 if got[0] == 12 else 1)
    dec.free(slots)
    dec.check()
    assert dec.cache.free_pages() == 640 // page_size


def test_verify_refusals():
    a = prompt_of(20, 6)
    dec = decoder(num_pages=4, max_seq_len=60)
    dec.prefill(0, a)
    for slots, tokens, parents in (([0], [[1, 2]], [[-1]]), ([0], [[]], [[]]), ([0], [[1]], [[0]]), ([0], [[1, 2]], [[-1, -1]]),
                                   ([0], [[1, 2]], [[-1, 1]]), ([0], [], []), ([0, 0], [[1], [1]], [[-1], [-1]]),
                                   ([9], [[1]], [[-1]]), ([0], [[VOCAB]], [[-1]]), ([0], [[-1]], [[-1]]),
                                   ([0], [[1] * 41], [list(range(-1, 40))]), ([0], [[1] * 257], [list(range(-1, 256))])):
        with pytest.raises(ValueError):
            dec.verify(slots, tokens, parents)
    with pytest.raises(RuntimeError, match="free pages"):
        dec.verify([0, 1, 2], [[1] * 30, [1], [1]], [list(range(-1, 29)), [-1], [-1]])
    assert dec.verify([], [], []) == []
    dec.check()
    assert dec.lengths == dec.cache.lengths.tolist() == [20, 0, 0, 0, 0]
    # a choice that fails leaves the first node
    with pytest.raises(ZeroDivisionError):
        dec.verify([0], [[1, 2, 3]], [[-1, 0, 1]], lambda x: 1 // 0)
    with pytest.raises(ValueError, match="chosen"):
        dec.verify([0], [[2, 2, 3]], [[-1, 0, 1]], lambda x: torch.tensor([1]))
    assert dec.lengths == dec.cache.lengths.tolist() == [22, 0, 0, 0, 0]
    close(dec.step([0], [5])[0], oracle_logits(a + [1, 2, 5])[-1])
    # an empty sequence's first tokens can be a tree as well
    dec.verify([1], [[a[0], 5, a[1]]], [[-1, 0, 0]], lambda x: torch.tensor([a[1], 0, 0]))
    assert dec.lengths[1] == 2
    close(dec.step([1], [a[2]])[0], oracle_logits(a[:3])[-1])
    dec.check()
    with pytest.raises(ValueError, match="window"):
        decoder(window=8).verify([0], [[1]], [[-1]])


# ---- drawn tokens ------------------------------------------------------------------------------------------------

def test_draw():
    from megaqwen_b200.sampling import sample
    dec = decoder()
    dec.prefill(0, prompt_of(40, 5))
    dec.fork(0, [1, 2])
    g, h = (torch.Generator(device="cuda").manual_seed(1) for _ in range(2))
    tokens = torch.tensor([1, 2, 3], device="cuda")
    for rules in (dict(temperature=0.7, top_k=40, top_p=0.9), dict(min_p=0.2), dict(temperature=0.0), dict()):
        logits = dec.step([0, 1, 2], tokens)
        tokens = dec.draw(logits, generator=g, **rules)
        u = torch.rand(3, generator=h, device="cuda")
        assert torch.equal(tokens, sample(logits, u, **rules))
        if rules.get("temperature") == 0:
            assert torch.equal(logits.gather(1, tokens[:, None].long())[:, 0], logits.amax(1))
    assert dec.draw(logits[0], temperature=0.0).tolist() == [int(logits[0].argmax())]
    dec.check()


def test_windowed_steps_do_not_synchronise():
    dec = decoder(window=30, sinks=2)
    dec.prefill(0, prompt_of(40, 5))
    dec.fork(0, [1, 2])
    tokens = torch.tensor([1, 2, 3], device="cuda")
    dec.step([0, 1, 2], tokens)
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(5):
            tokens = dec.draw(dec.step([0, 1, 2], tokens), temperature=0.8, top_k=50, top_p=0.95)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    dec.check()


def test_example_runs():
    spec = importlib.util.spec_from_file_location("shared_prompt", ROOT / "examples" / "shared_prompt.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.guess([1, 2, 3, 1], 2) == [2, 3] and mod.guess([1, 2], 2) == [] and mod.guess([5, 5], 3) == [5]
    args = ["--layers", "2", "--prompt", "200", "--samples", "3", "--steps", "20"]
    a = mod.main(args + ["--window", "50", "--temperature", "0.8", "--top-k", "40", "--top-p", "0.9", "--min-p", "0.01"])
    assert len(a["tokens"]) == 3 and all(len(t) == 21 for t in a["tokens"])
    b = mod.main(args + ["--draft", "4", "--temperature", "0"])
    c = mod.main(args + ["--draft", "1", "--temperature", "0"])
    assert all(21 <= len(t) <= 101 for t in b["tokens"]) and all(21 <= len(t) <= 41 for t in c["tokens"])
