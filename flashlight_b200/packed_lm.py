"""Trains the Transformer language model on rows packed with documents, with AdamW: masked attention, the loss
without scores and the optimiser of this package as a training loop calls them.

    python -m flashlight_b200.packed_lm --steps 50 --layers 4 --state-bits 8

The documents are synthetic and can be learnt: each repeats a short pattern of its own, so that behind its first
repetition the next token is known from the context.
"""
from __future__ import annotations

import argparse
import time

import torch

from .optim import AdamWOptimizer
from .workloads import TransformerLM


def packed_batch(batch: int, length: int, vocab: int, mean: int, generator: torch.Generator):
    """(ids, targets, documents) on the host: rows of documents of about `mean` tokens; a document's last token has no
    target, what is behind a row's last document is padding."""
    ids = torch.zeros(batch, length, dtype=torch.int32)
    targets = torch.full((batch, length), -1, dtype=torch.int32)
    documents = torch.full((batch, length), -1, dtype=torch.int32)
    draw = lambda low, high: int(torch.randint(low, high + 1, (1,), generator=generator))  # noqa: E731
    for row in range(batch):
        at, number = 0, 0
        while length - at >= 2:
            n = min(length - at, draw(max(2, mean // 2), max(2, mean * 3 // 2)))
            period = draw(2, 8)
            pattern = torch.randint(vocab, (period,), generator=generator, dtype=torch.int32)
            text = pattern.repeat(n // period + 1)[:n]
            ids[row, at:at + n] = text
            targets[row, at:at + n - 1] = text[1:]
            documents[row, at:at + n] = number
            at, number = at + n, number + 1
    return ids, targets.view(-1), documents


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=512)
    ap.add_argument("--document", type=int, default=150, help="mean length of a document")
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--layers", type=int, default=12)
    ap.add_argument("--width", type=int, default=768)
    ap.add_argument("--heads", type=int, default=12)
    ap.add_argument("--kv-heads", type=int, default=None)
    ap.add_argument("--softcap", type=float, default=0.0)
    ap.add_argument("--distance-bias", action="store_true")
    ap.add_argument("--lr", type=float, default=3e-4)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    ap.add_argument("--seed", type=int, default=1)
    a = ap.parse_args(argv)
    generator = torch.Generator().manual_seed(a.seed)
    model = TransformerLM(a.vocab, a.width, a.heads, 4 * a.width, a.layers, seed=a.seed,
                          compute_dtype=torch.bfloat16, packed=True, kv_heads=a.kv_heads, softcap=a.softcap,
                          distance_bias=a.distance_bias)
    optimiser = AdamWOptimizer(model.parameters(), a.lr, 0.9, 0.95, 1e-8, 0.1, state_bits=a.state_bits)
    loss, began = float("nan"), time.perf_counter()
    for step in range(1, a.steps + 1):
        ids, targets, documents = (t.cuda() for t in packed_batch(a.batch, a.length, a.vocab, a.document, generator))
        optimiser.zeroGrad()
        out = model.loss(ids, targets, documents)
        value = out.tensor
        out.backward()
        optimiser.step()
        if step in (1, a.steps) or step % 10 == 0:
            loss = float(value)
            print(f"step {step}: loss {loss:.4f}, {1e3 * (time.perf_counter() - began) / step:.1f} ms a step", flush=True)
    return loss


if __name__ == "__main__":
    main()
