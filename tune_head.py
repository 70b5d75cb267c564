#!/usr/bin/env python3
"""Tune the vocabulary head of a completed migration on the teacher's recorded logits and on next tokens, and export it.

The config's training chunks are recorded with the original attention blocks, the head is tuned against the record on
the assembled model's hidden states of the same chunks, and the scores on validation text of the teacher and of the
assembled model before and after are printed as JSON (single GPU).

    python tune_head.py --checkpoint RUN_DIR --steps 200 [--chunks 32] [--top 64] [--kl-weight 0.5] --output EXPORT_DIR
"""
import argparse
import json

import torch

from rwkv_theseus_b200.assembly import _base_with_students, _require_same_base
from rwkv_theseus_b200.checkpoint import read_checkpoint
from rwkv_theseus_b200.data import reader_for
from rwkv_theseus_b200.head_tuning import hidden_states, record_teacher, score, tune_head
from rwkv_theseus_b200.inference import save_export
from rwkv_theseus_b200.models.runner import Runner
from rwkv_theseus_b200.validation import original_attention, validation_batches


class _Local:
    rank, world = 0, 1


def run(checkpoint, output, steps, chunks=32, top=64, temperature=1.0, kl_weight=0.5, lr=1e-5, device="cuda"):
    directory, meta, delta = read_checkpoint(checkpoint)
    if not meta["complete"] or set(delta) != set(meta["order"]):
        raise ValueError("Head tuning requires all layers to have completed training")
    cfg = meta["config"]
    _require_same_base(cfg, meta, "Base weights changed")
    device = torch.device(device)
    model = _base_with_students(cfg, delta, meta["order"], device)
    runner = Runner(model)
    reader = reader_for(dict(cfg, training_mode="sampled"), _Local())
    train = [reader.next() for _ in range(chunks)]
    held_out = validation_batches(cfg, _Local())
    with original_attention(model, cfg["model"]):
        records = record_teacher(runner, train, device, top, temperature)
        teacher = score(runner, held_out, device)[0]
    states = hidden_states(runner, train, device)
    before, tokens = score(runner, held_out, device)
    losses = tune_head(model, train, states, records, device, steps, lr, kl_weight, temperature)
    after = score(runner, held_out, device)[0]
    report = {"tokens": tokens, "teacher": teacher, "before": before, "after": after,
              "first_loss": losses[0] if losses else None, "last_loss": losses[-1] if losses else None}
    if output:
        save_export(model.cpu(), output, cfg, meta["order"], meta["base_fingerprint"], checkpoint=directory)
    return report


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--checkpoint", required=True, help="complete checkpoint, its run directory or 'latest'")
    p.add_argument("--output", help="directory of the export (omit to report only)")
    p.add_argument("--steps", type=int, default=200, help="0: the scores alone")
    p.add_argument("--chunks", type=int, default=32, help="training chunks to record and tune on")
    p.add_argument("--top", type=int, default=64, help="recorded log-probabilities per token")
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--kl-weight", type=float, default=0.5)
    p.add_argument("--lr", type=float, default=1e-5)
    p.add_argument("--device", default="cuda")
    a = p.parse_args(argv)
    print(json.dumps(run(a.checkpoint, a.output, a.steps, a.chunks, a.top, a.temperature, a.kl_weight, a.lr, a.device),
                     indent=2))


if __name__ == "__main__":
    main()
