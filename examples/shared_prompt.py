"""Several samples of one prompt on the paged cache.

    python examples/shared_prompt.py [--layers 28] [--prompt 1000] [--samples 8] [--steps 32] [--sparse-pages 0]

The prompt is prefilled once, its pages forked into the samples, and every
decode step reads the shared pages once for all of them (or, with
--sparse-pages N, N pages per query and kv head).  Then the samples are freed
and what is left is gathered into a smaller pool.  Weights are the package's
seeded synthetic ones.
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


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=28)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--sparse-pages", type=int, default=0)
    a = ap.parse_args(argv)
    length = a.prompt + a.steps
    own = a.steps // 64 + 2
    dec = PagedDecoder(make_weights(a.layers).to("cuda"), num_pages=-(-a.prompt // 64) + a.samples * own, max_seqs=a.samples + 1,
                       max_seq_len=length, sparse_pages=a.sparse_pages or None)
    logits = dec.prefill(0, seeded_prompt(a.prompt).tolist())
    samples = list(range(1, a.samples + 1))
    dec.fork(0, samples)
    used = dec.cache.k_pages.shape[0] - dec.cache.free_pages()
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens = torch.multinomial(torch.softmax(logits, -1), a.samples, replacement=True, generator=g)
    out = [tokens]
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.steps):
        tokens = torch.multinomial(torch.softmax(dec.step(samples, tokens), -1), 1, generator=g)[:, 0]
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
    return {"tokens": torch.stack(out, 1).tolist(), "used": used, "kept": kept}


if __name__ == "__main__":
    main()
