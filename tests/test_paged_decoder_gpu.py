"""The paged cache in use: a prompt prefilled once, forked into samples, decoded against the CPU oracle."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from megaqwen_b200.weights import make_weights, seeded_prompt

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
LAYERS = 2
# q, k and the attention output in bf16: the bound of the batched decoder's tests
LOGIT_TOL = 3e-2


def oracle_with(prompt):
    from oracle.qwen3_cpu import Qwen3CpuOracle
    o = Qwen3CpuOracle(make_weights(LAYERS), max_seq_len=256)
    return o, o.prefill(prompt)[-1]


def close(got, ref):
    err = (got.cpu() - ref).abs().max().item()
    assert err < LOGIT_TOL, err


@pytest.mark.parametrize("page_size,length", [(16, 75), (64, 64), (32, 5)])
def test_samples_match_oracle(page_size, length):
    from megaqwen_b200.paged_decoder import PagedDecoder
    prompt = seeded_prompt(length, seed=length).tolist()
    dec = PagedDecoder(make_weights(LAYERS).to("cuda"), num_pages=40, max_seqs=6, max_seq_len=256, page_size=page_size)
    # in two pieces; a stranger beside it
    cut = max(1, length // 3)
    dec.prefill(2, prompt[:cut])
    close(dec.prefill(2, prompt[cut:]), oracle_with(prompt)[1])
    stranger = seeded_prompt(9, seed=1).tolist()
    dec.prefill(0, stranger)
    dec.fork(2, [5, 1])
    slots = [5, 0, 2, 1]
    oracles = [oracle_with(stranger if s == 0 else prompt)[0] for s in slots]
    at = [len(stranger) if s == 0 else length for s in slots]
    g = torch.Generator().manual_seed(3)
    for step in range(20):
        tokens = torch.randint(0, 151936, (len(slots),), generator=g)
        logits = dec.step(slots, tokens)
        for i, o in enumerate(oracles):
            close(logits[i], o.decode_step(int(tokens[i]), at[i] + step))
    dec.check()
    dec.free(slots)
    assert dec.cache.free_pages() == 40


def test_sparse_steps_of_every_page_match_dense():
    from megaqwen_b200.paged_decoder import PagedDecoder
    prompt = seeded_prompt(150, seed=2).tolist()
    w = make_weights(LAYERS).to("cuda")
    got = []
    for pages in (None, 64, 4):
        dec = PagedDecoder(w, num_pages=64, max_seqs=3, max_seq_len=256, page_size=16, sparse_pages=pages)
        dec.prefill(0, prompt)
        dec.fork(0, [1, 2])
        got.append(torch.stack([dec.step([0, 1, 2], torch.tensor([5 + i, 9, 70000])) for i in range(4)]))
        dec.check()
    assert (got[0] - got[1]).abs().max().item() < LOGIT_TOL      # everything selected
    assert torch.isfinite(got[2]).all()


def decoder(**kw):
    from megaqwen_b200.paged_decoder import PagedDecoder
    return PagedDecoder(make_weights(LAYERS).to("cuda"), **{**dict(num_pages=6, max_seqs=5, max_seq_len=256, page_size=16), **kw})


def prompt_of(n, seed):
    return seeded_prompt(n, seed=seed).tolist()


def test_refused_calls_leave_the_decoder_as_it_was():
    """Not enough pages, slots that are not empty: what follows is right."""
    a, b = prompt_of(60, 4), prompt_of(40, 5)
    dec = decoder()
    dec.prefill(0, a)                       # four of six pages
    with pytest.raises(RuntimeError, match="free pages"):
        dec.prefill(1, b)
        dec.check()
    with pytest.raises((RuntimeError, ValueError), match="free pages|empty slot|not empty"):
        dec.fork(0, [1, 2, 3])              # a part page each
        dec.check()
    close(dec.prefill(1, b[:32]), oracle_with(b[:32])[1])
    with pytest.raises((RuntimeError, ValueError), match="empty"):
        dec.fork(0, [1])
        dec.check()
    with pytest.raises(RuntimeError, match="free pages"):
        dec.step([1], torch.tensor([b[32]]))    # a seventh page
        dec.check()
    oracle, _ = oracle_with(a)
    close(dec.step([0], torch.tensor([7]))[0], oracle.decode_step(7, len(a)))
    assert dec.lengths == dec.cache.lengths.tolist() == [61, 32, 0, 0, 0]
    dec.free([0])
    close(dec.prefill(1, b[32:]), oracle_with(b)[1])
    dec.free([1])
    dec.check()
    assert dec.cache.free_pages() == 6


def test_errors_found_on_the_device():
    """Pages taken behind the decoder's back: its calls are refused there, and after check() it knows how things stand."""
    b = prompt_of(40, 5)
    dec = decoder()
    dec.cache.reserve([3], [70])
    dec.prefill(1, b)
    with pytest.raises(RuntimeError, match="free pages"):
        dec.check()
    assert dec.lengths == [0, 0, 0, 70, 0]
    dec.free([3])
    close(dec.prefill(1, b), oracle_with(b)[1])
    dec.fork(1, [0, 2])
    oracle, _ = oracle_with(b)
    close(dec.step([2, 0], torch.tensor([9, 9]))[1], oracle.decode_step(9, 40))
    dec.check()


def test_tokens_and_slots_that_are_wrong():
    b = prompt_of(20, 6)
    dec = decoder()
    vocab = dec.embed.shape[0]
    for bad in ([-1], [vocab], []):
        with pytest.raises(ValueError):
            dec.prefill(0, bad)
    for slot in (-1, 5):
        with pytest.raises(ValueError):
            dec.prefill(slot, b)
    dec.prefill(0, b)
    for slots, tokens in (([0], []), ([0], [1, 2]), ([0, 0], [1, 2]), ([-1], [1]), ([9], [1]), ([0], [vocab]), ([0], [0.5])):
        with pytest.raises(ValueError):
            dec.step(slots, torch.tensor(tokens))
    for call in (lambda: dec.free([0, 0]), lambda: dec.free([7]), lambda: dec.fork(9, [1]), lambda: dec.fork(0, [1, 1]), lambda: dec.fork(0, [0])):
        with pytest.raises(ValueError):
            call()
    assert dec.step([], torch.tensor([], dtype=torch.long)).shape == dec.step([], []).shape == (0, vocab)
    oracle, _ = oracle_with(b)
    close(dec.step([0], torch.tensor([3]))[0], oracle.decode_step(3, 20))
    dec.check()
    dec.step([0], torch.tensor([vocab], device="cuda"))      # known on the device alone
    with pytest.raises(RuntimeError, match="token"):
        dec.check()
    dec.check()


def test_steps_do_not_synchronise():
    dec = decoder(num_pages=40)
    dec.prefill(0, prompt_of(40, 5))
    dec.fork(0, [1, 2])
    tokens = torch.tensor([1, 2, 3], device="cuda")
    dec.step([0, 1, 2], tokens)
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(20):
            tokens = dec.step([0, 1, 2], tokens).argmax(-1)
        dec.step([2, 0], tokens[:2])
        dec.free([1])
        dec.fork(0, [1])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    dec.check()


def test_example_runs(capsys):
    spec = importlib.util.spec_from_file_location("shared_prompt", ROOT / "examples" / "shared_prompt.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    args = ["--layers", "2", "--prompt", "200", "--samples", "3", "--steps", "70"]
    a = mod.main(args)
    assert a["used"] == 4 + 3 and len(a["tokens"]) == 3 and len(a["tokens"][0]) == 71
    b = mod.main(args + ["--sparse-pages", "2"])
    assert b["used"] == a["used"]
    assert "samples of a 200-token prompt" in capsys.readouterr().out
