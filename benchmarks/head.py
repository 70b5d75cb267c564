#!/usr/bin/env python3
"""Vocabulary-head losses and top log-probabilities at the 27B head (vocabulary 248077, width 5120): device time of a
forward call and of a forward and backward call, against the same product flops (2, 4 or 6 x tokens x vocabulary x
width), and of recording the top entries against reading the logits once. CUDA events, median of --iters after --warmup;
the weight (2.5 GB) and the logits exceed L2.

    python benchmarks/head.py [--tokens 1024] [--vocab 248077] [--width 5120] [--top 64]
"""
import argparse
import json
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from rwkv_theseus_b200.losses import linear_cross_entropy, linear_topk_kl, top_log_probs  # noqa: E402


def timed(fn, warmup, iters):
    for _ in range(warmup):
        fn()
    times = []
    for _ in range(iters):
        s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        s.record()
        fn()
        e.record()
        torch.cuda.synchronize()
        times.append(s.elapsed_time(e))
    return sorted(times)[len(times) // 2]


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--tokens", type=int, default=1024)
    p.add_argument("--vocab", type=int, default=248077)
    p.add_argument("--width", type=int, default=5120)
    p.add_argument("--top", type=int, default=64)
    p.add_argument("--warmup", type=int, default=3)
    p.add_argument("--iters", type=int, default=10)
    a = p.parse_args()
    g = torch.Generator(device="cuda").manual_seed(0)
    hidden = torch.randn(a.tokens, a.width, device="cuda", generator=g).to(torch.bfloat16)
    weight = (torch.randn(a.vocab, a.width, device="cuda", generator=g) / math.sqrt(a.width)).to(torch.bfloat16)
    targets = torch.randint(0, a.vocab, (a.tokens,), device="cuda", generator=g)
    logits = (torch.randn(a.tokens, a.vocab, device="cuda", generator=g) * 2).to(torch.bfloat16)
    log_probs, indices = top_log_probs(logits, a.top)
    ms = timed(lambda: top_log_probs(logits, a.top), a.warmup, a.iters)
    print(json.dumps({"bench": "top_log_probs", "tokens": a.tokens, "vocab": a.vocab, "top": a.top, "ms": ms,
                      "gbs": logits.numel() * 2 / ms / 1e6}), flush=True)
    del logits
    losses = {"linear_cross_entropy": lambda h, w: linear_cross_entropy(h, w, targets),
              "linear_topk_kl": lambda h, w: linear_topk_kl(h, w, indices, log_probs)}
    for name, loss in losses.items():
        for grads in ((), ("hidden",), ("hidden", "weight")):
            h = hidden.clone().requires_grad_("hidden" in grads)
            w = weight.detach().requires_grad_("weight" in grads)
            wanted = [t for t in (h, w) if t.requires_grad]

            def call():
                out = loss(h, w)
                return torch.autograd.grad(out, wanted) if wanted else out
            ms = timed(call, a.warmup, a.iters)
            flops = 2 * (1 + len(grads)) * a.tokens * a.vocab * a.width
            print(json.dumps({"bench": name, "grads": grads, "tokens": a.tokens, "vocab": a.vocab, "width": a.width,
                              "ms": ms, "tflops": flops / ms / 1e9, "weight_gbs": weight.numel() * 2 / ms / 1e6}),
                  flush=True)


if __name__ == "__main__":
    main()
