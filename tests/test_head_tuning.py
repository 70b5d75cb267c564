"""Head tuning: recording, scoring and tuning on a tiny hybrid, and the command on a finished run."""
import math

import pytest
import torch
from torch.nn import functional as F

from fixtures import make_config, tiny_model
from rwkv_theseus_b200.head_tuning import hidden_states, next_tokens, record_teacher, score, tune_head
from rwkv_theseus_b200.models.runner import Runner
from test_resume import rewrite, train

CPU = torch.device("cpu")


def _chunks(n=3, T=9, vocab=64):
    g = torch.Generator().manual_seed(4)
    return [{"ids": torch.randint(0, vocab, (1, T), generator=g), "reset": i != 1} for i in range(n)]


def test_record_and_score_follow_the_models_logits():
    model, chunks = tiny_model(dtype=torch.float32), _chunks()
    runner = Runner(model)
    records = record_teacher(runner, chunks, CPU, k=5, temperature=2.0, token_block=4)
    states = hidden_states(runner, chunks, CPU)
    nats, count = score(runner, chunks, CPU)
    assert count == 3 * 8
    expected = 0.0
    for chunk, state, (indices, log_probs) in zip(chunks, states, records):
        z = state @ model.lm_head.weight.t()
        assert indices.dtype == torch.int32 and indices.shape == (1, 9, 5)
        torch.testing.assert_close(log_probs, torch.log_softmax(z / 2.0, -1).gather(-1, indices.long()))
        assert torch.equal(indices[..., 0].long(), z.argmax(-1))
        expected += F.cross_entropy(z[0], next_tokens(chunk["ids"])[0], reduction="sum", ignore_index=-100).item()
    assert math.isclose(nats, expected / count, rel_tol=1e-5)


@pytest.mark.parametrize("kl_weight", [0.0, 0.5, 1.0])
def test_tuning_brings_a_disturbed_head_back(kl_weight):
    model, chunks = tiny_model(dtype=torch.float32), _chunks()
    runner = Runner(model)
    records = record_teacher(runner, chunks, CPU, k=16)
    states = hidden_states(runner, chunks, CPU)
    with torch.no_grad():
        model.lm_head.weight.add_(0.3 * torch.randn(model.lm_head.weight.shape))
    before = model.lm_head.weight.clone()
    losses = tune_head(model, chunks, states, records, CPU, 60, lr=3e-2, kl_weight=kl_weight)
    assert len(losses) == 60 and sum(losses[-3:]) < 0.5 * sum(losses[:3])
    assert not torch.equal(before, model.lm_head.weight) and not model.lm_head.weight.requires_grad


def test_tuning_refuses():
    model, chunks = tiny_model(dtype=torch.float32), _chunks(1)
    runner = Runner(model)
    records, states = record_teacher(runner, chunks, CPU, k=4), hidden_states(runner, chunks, CPU)
    with pytest.raises(ValueError, match="kl_weight"):
        tune_head(model, chunks, states, records, CPU, 1, kl_weight=1.5)
    with pytest.raises(ValueError, match="per chunk"):
        tune_head(model, chunks, states, [], CPU, 1)
    model.config.tie_word_embeddings = True
    with pytest.raises(ValueError, match="shares its weight"):
        tune_head(model, chunks, states, records, CPU, 1)


def test_the_command_on_a_finished_run(tmp_path):
    from rwkv_theseus_b200.inference import load_export
    from tune_head import run
    cfg, path = make_config(tmp_path, 2)
    rewrite(path, cfg, stage_steps=1, warmup_steps=0, constant_steps=0)
    train(path, 1)
    out = tmp_path / "tuned"
    report = run(tmp_path / "full" / "latest", out, steps=20, chunks=4, top=8, lr=1e-2, device="cpu")
    assert report["tokens"] == 2 * 2 and report["last_loss"] < report["first_loss"]
    assert all(math.isfinite(report[key]) for key in ("teacher", "before", "after"))
    assert load_export(out, device="cpu").model.lm_head.weight.shape == (64, 32)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA unavailable")
def test_one_step_on_cuda_matches_the_plain_definition():
    """The same chunk, record and head through the kernels and through the plain definition on the CPU. The hidden
    states and weight are the same bf16 values; the gradients differ by bf16 roundings (3 x 2^-8 of their parts, see
    test_head_losses_gpu.py), so do the updates' inputs; losses agree to fp32 sums over 64 products."""
    from rwkv_theseus_b200.head_tuning import head_loss
    from rwkv_theseus_b200.losses import top_log_probs
    g = torch.Generator().manual_seed(0)
    hidden = torch.randn(2, 37, 64, generator=g).to(torch.bfloat16)
    weight = (torch.randn(513, 64, generator=g) * 0.2).to(torch.bfloat16)
    ids = torch.randint(0, 513, (2, 37), generator=g)
    log_probs, indices = top_log_probs((hidden.float() + torch.randn(hidden.shape, generator=g)) @ weight.float().t(), 12)
    out = []
    for device in ("cpu", "cuda"):
        live = weight.to(device).requires_grad_()
        record = (indices.to(torch.int32).to(device), log_probs.to(device))
        loss = head_loss(hidden.to(device), live, next_tokens(ids).to(device), record, 1.0, 0.5)
        out.append((loss.item(), torch.autograd.grad(loss, live)[0].float().cpu()))
    (a, ga), (b, gb) = out
    assert abs(a - b) <= 1e-4 * abs(a)
    assert (ga - gb).norm() <= 4 * 3 * 2.0 ** -8 * ga.norm()
