"""Perplexity of a prompt under an FP8 block-scaled head, with random weights: hidden states are
quantized per group of 128 and scored against the next tokens. ``--top-k`` also prints the most
likely alternatives of the first rows.

    python examples/score_prompt.py --rows 1024 --vocab 151936 --hidden 2560 --top-k 5
"""
from __future__ import annotations

import argparse
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main() -> None:
    p = argparse.ArgumentParser()
    p.add_argument("--rows", type=int, default=1024)
    p.add_argument("--vocab", type=int, default=151936)
    p.add_argument("--hidden", type=int, default=2560)
    p.add_argument("--top-k", type=int, default=0)
    a = p.parse_args()
    pkg = importlib.import_module("r9700-lru-expert-cache_b200")
    g = torch.Generator(device="cuda").manual_seed(0)
    weight = (torch.randn(a.vocab, a.hidden, device="cuda", generator=g) * 0.02).bfloat16()
    head = pkg.fp8_target_lmhead.Fp8TargetHead(None, weight)
    del weight
    hidden = torch.randn(a.rows, a.hidden, device="cuda", generator=g).bfloat16()
    tokens = torch.randint(a.vocab, (a.rows,), device="cuda", generator=g)
    for _ in range(3):
        head.score(hidden, tokens, top_k=a.top_k)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    r = head.score(hidden, tokens, top_k=a.top_k)
    end.record()
    torch.cuda.synchronize()
    print(f"{a.rows} rows x {a.vocab} tokens: perplexity {torch.exp(-r.logprob.mean()).item():.0f}, mean entropy "
          f"{r.entropy.mean().item():.3f}, {start.elapsed_time(end) * 1e3:.0f} us")
    for i in range(min(3, a.rows) if a.top_k else 0):
        alternatives = ", ".join(f"{t}: {lp:.2f}" for t, lp in zip(r.top_ids[i].tolist(), r.top_logprobs[i].tolist()))
        print(f"row {i}: token {tokens[i].item()} {r.logprob[i].item():.2f} (rank {r.rank[i].item()}); {alternatives}")


if __name__ == "__main__":
    main()
