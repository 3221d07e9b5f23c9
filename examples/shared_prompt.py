"""Several samples of one prompt on the paged cache.

    python examples/shared_prompt.py [--layers 28] [--prompt 1000] [--samples 8] [--steps 32] [--sparse-pages 0]
                                      [--window 0 --sinks 4] [--temperature 1 --top-k 0 --top-p 1 --min-p 0] [--draft 0]

The prompt is prefilled once, its pages forked into the samples, and every
decode step reads the shared pages once for all of them (or, with
--sparse-pages N, N pages per query and kv head; with --window N, the last N
positions and the first ones).  With a rule for sampling the tokens are drawn by
it.  With --draft N each step checks N tokens, guessed to follow as they did
where the last token stood before, and goes on behind those that are drawn.
Then the samples are freed and what is left is gathered into a smaller pool.
Weights are the package's seeded synthetic ones.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from megaqwen_b200.paged_decoder import PagedDecoder  # noqa: E402
from megaqwen_b200.weights import make_weights, seeded_prompt  # noqa: E402


def guess(text: list, n: int) -> list:
    """The up to n tokens that followed where the last token stood before (nearest the end), or none."""
    at = next((i for i in range(len(text) - 2, -1, -1) if text[i] == text[-1]), len(text))
    return text[at + 1:at + 1 + n]


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=28)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--sparse-pages", type=int, default=0)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=1.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--draft", type=int, default=0)
    a = ap.parse_args(argv)
    rules = dict(temperature=a.temperature, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p)
    ruled = bool(a.draft) or rules != dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    length = a.prompt + a.steps * (a.draft + 1) + a.draft
    own = (length - a.prompt) // 64 + 2
    dec = PagedDecoder(make_weights(a.layers).to("cuda"), num_pages=-(-a.prompt // 64) + a.samples * own, max_seqs=a.samples + 1,
                       max_seq_len=length, sparse_pages=a.sparse_pages or None, window=a.window or None,
                       sinks=a.sinks if a.window else 0)
    prompt = seeded_prompt(a.prompt).tolist()
    logits = dec.prefill(0, prompt)
    samples = list(range(1, a.samples + 1))
    dec.fork(0, samples)
    used = dec.cache.k_pages.shape[0] - dec.cache.free_pages()
    g = torch.Generator(device="cuda").manual_seed(0)

    def draw(logits):
        if ruled:
            return dec.draw(logits, generator=g, **rules)
        return torch.multinomial(torch.softmax(logits, -1), 1, generator=g)[:, 0]

    if ruled:
        tokens = draw(logits.expand(a.samples, -1))
    else:
        tokens = torch.multinomial(torch.softmax(logits, -1), a.samples, replacement=True, generator=g)
    out = [tokens]
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    if a.draft:
        texts = [prompt + [t] for t in tokens.tolist()]
        for _ in range(a.steps):
            trees = [[t[-1], *guess(t, a.draft)] for t in texts]
            parents = [list(range(-1, len(t) - 1)) for t in trees]
            for t, more in zip(texts, dec.verify(samples, trees, parents, draw)):
                t += more
    else:
        for _ in range(a.steps):
            tokens = draw(dec.step(samples, tokens))
            out.append(tokens)
    dec.check()
    took = time.perf_counter() - t0
    dec.free(samples[1:])
    kept = dec.cache.k_pages.shape[0] - dec.cache.free_pages()
    small = dec.cache.compact(kept)
    dec.cache.check()
    assert int((small.refs > 0).sum()) == kept
    print(f"{a.samples} samples of a {a.prompt}-token prompt: {used} pages after the fork "
          f"({(1 + a.samples) * -(-a.prompt // 64)} without sharing), {a.steps} steps in {took * 1e3:.1f} ms, "
          f"{kept} pages left for the prompt and one sample")
    tokens = [t[a.prompt:] for t in texts] if a.draft else torch.stack(out, 1).tolist()
    return {"tokens": tokens, "used": used, "kept": kept}


if __name__ == "__main__":
    main()
