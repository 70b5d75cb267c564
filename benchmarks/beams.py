#!/usr/bin/env python3
"""Beam search of the 27B hybrid (random init, bf16, one GPU): time per decode step and of its parts that greedy decoding
does not have. ``--original`` keeps the full-attention blocks, whose keys and values then lie in pages that the beams of a
prompt share; otherwise each is replaced by its TimeMix student, as after a migration.

    python benchmarks/beams.py [--prompts 1] [--beams 4] [--prompt 4096] [--new 64] [--model 27b|small] [--original]
                               [--graph]

Reports the p50 / p90 step (CUDA events around every step), the same for greedy decoding of prompts x beams rows, and the
device time of one selection and one reordering of the states at these sizes.
"""
import argparse
import json
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from bench import MODEL_27B, MODEL_SMALL, layer_types  # noqa: E402
from rwkv_theseus_b200.beams import beam_search, beam_select, reorder_states_  # noqa: E402
from rwkv_theseus_b200.inference import generate  # noqa: E402
from rwkv_theseus_b200.models.hf_io import random_model  # noqa: E402
from rwkv_theseus_b200.models.qwen35 import HybridConfig  # noqa: E402
from rwkv_theseus_b200.models.runner import Runner, install, migration_order  # noqa: E402


def between(events):
    times = sorted(a.elapsed_time(b) for a, b in zip(events[2:], events[3:]))  # without the graph's capture
    return {"p50_ms": times[len(times) // 2], "p90_ms": times[int(len(times) * 0.9)]}


def median_us(fn, iters=20):
    fn()
    times = []
    for _ in range(iters):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        fn()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[iters // 2]


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--prompts", type=int, default=1)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--prompt", type=int, default=4096)
    p.add_argument("--new", type=int, default=64)
    p.add_argument("--model", choices=("27b", "small"), default="27b")
    p.add_argument("--original", action="store_true", help="keep the full-attention blocks")
    p.add_argument("--graph", action="store_true", help="replay the steps as a CUDA graph")
    a = p.parse_args()
    spec = MODEL_27B if a.model == "27b" else MODEL_SMALL
    cfg = HybridConfig(**spec, layer_types=layer_types(spec["num_hidden_layers"]))
    device = torch.device("cuda", 0)
    model = random_model(cfg, device, seed=0)
    blocks = len([t for t in cfg.layer_types if t == "full_attention"])
    if not a.original:
        for i, layer in enumerate(migration_order(model, blocks)):
            torch.manual_seed(i)
            install(model, layer, {"head_size": 64, "backend": "cuda", "lora_rank": None, "gate_lora_rank": None})
    runner = Runner(model)
    g = torch.Generator(device=device).manual_seed(7)
    prompt = torch.randint(0, cfg.vocab_size, (a.prompts, a.prompt), device=device, generator=g)
    events = []

    def mark(*_):
        events.append(torch.cuda.Event(enable_timing=True))
        events[-1].record()

    def run(rows):
        events.clear()
        if rows is None:
            ids, scores, _ = beam_search(runner, prompt, a.new, a.beams, on_token=mark, graph=a.graph)
            assert scores.isfinite().all()
        else:
            generate(runner, rows, a.new, on_token=mark, graph=a.graph and not a.original)
        torch.cuda.synchronize()
        return between(events)

    run(None)  # measures the GEMM tile choices
    search = run(None)
    rows = prompt.repeat_interleave(a.beams, 0)
    run(rows)
    greedy = run(rows)
    G, K, V = a.prompts, a.beams, cfg.vocab_size
    logits = torch.randn(G, K, V, device=device, generator=g).to(torch.bfloat16)
    scores, ends = torch.zeros(G, K, device=device), torch.zeros(G, K, dtype=torch.bool, device=device)
    lengths = torch.ones(G, K, dtype=torch.int32, device=device)
    select = median_us(lambda: beam_select(logits, scores, lengths, ends))
    states = [layer[name] for layer in runner.cache.layers if "recurrent" in layer for name in ("conv", "recurrent")]
    parents = torch.arange(K, device=device).expand(G, K).clone()
    parents[:, K // 2:] = parents[:, :K - K // 2]  # half of the slots follow others
    reorder = median_us(lambda: reorder_states_(states, parents))
    print(json.dumps({"bench": "beam_search", "model": f"qwen3.5-hybrid-{a.model}", "original": a.original,
                      "prompts": a.prompts, "beams": a.beams, "prompt": a.prompt, "new_tokens": a.new, "dtype": "bf16",
                      "cuda_graph": a.graph, "step": search, "greedy_same_rows": greedy, "select_us": select,
                      "reorder_half_us": reorder, "data": "uniform-random prompt ids; random-init weights"}), flush=True)


if __name__ == "__main__":
    main()
