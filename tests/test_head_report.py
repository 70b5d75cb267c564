"""The head-tuning command without a step: the scores alone, the head as it was."""
import math

import torch

from fixtures import make_config
from rwkv_theseus_b200.inference import load_export
from test_resume import rewrite, train
from tune_head import run


def test_scores_without_a_step(tmp_path):
    cfg, path = make_config(tmp_path, 2)
    rewrite(path, cfg, stage_steps=1, warmup_steps=0, constant_steps=0)
    train(path, 1)
    report = run(tmp_path / "full" / "latest", tmp_path / "same", steps=0, chunks=2, top=8, device="cpu")
    assert report["first_loss"] is None and report["last_loss"] is None
    assert report["before"] == report["after"] and math.isfinite(report["teacher"])
    assert torch.isfinite(load_export(tmp_path / "same", device="cpu").model.lm_head.weight).all()
