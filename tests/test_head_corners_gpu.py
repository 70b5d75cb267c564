"""Corners of the vocabulary-head operators on the GPU against 64-bit formulas: students that are sure of their record,
records of the whole vocabulary, logits of any size, masks of the type's lowest value, NaN.

Tolerances are those of test_head_losses_gpu.py (u = 2^-8; a gradient is off by (3 u + 4 dz) times the same product of
absolute values, dz the bound of a logit's error) unless a test derives its own.
"""
import math

import pytest
import torch

from rwkv_theseus_b200.losses import linear_cross_entropy, top_log_probs
from test_head_losses_gpu import U, _check, _inputs, _record

pytestmark = pytest.mark.gpu
cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA unavailable")


def _sure(T, V, gap, mass, entries=4):
    """Rows whose student is `gap` nats surer of its `entries` recorded tokens than of the rest, where the teacher's
    record holds `mass`. Feature j of the width stands for the j-th group of tokens and is zero for all others."""
    g = torch.Generator(device="cuda").manual_seed(T + V + int(gap))
    weight = torch.randn(V, 64, device="cuda", generator=g) * 0.15
    hidden = torch.randn(T, 64, device="cuda", generator=g)
    weight[:, :8] = 0.0
    hidden[:, :8] = 0.0
    for j in range(8):
        weight[j * entries:(j + 1) * entries, j] = 1.0
    group = torch.randint(0, 8, (T,), device="cuda", generator=g)
    hidden[torch.arange(T, device="cuda"), group] = gap
    index = group[:, None] * entries + torch.arange(entries, device="cuda")
    p = torch.rand(T, entries, device="cuda", generator=g) + 0.2
    return hidden.to(torch.bfloat16), weight.to(torch.bfloat16), index, (p / p.sum(-1, keepdim=True) * mass).log()


@cuda
@pytest.mark.parametrize("T", [5, 100, 150])
@pytest.mark.parametrize("gap", [80.0, 100.0, 300.0])
@pytest.mark.parametrize("mass,entries", [(0.5, 4), (0.9, 1), (0.999999, 4)])
def test_a_student_that_is_sure_of_its_record(T, gap, mass, entries):
    """The rest of the vocabulary has a probability of e^-gap, and is all that pushes mass back to it."""
    hidden, weight, index, log_probs = _sure(T, 1003, gap, mass, entries)
    _check(hidden, weight, index, log_probs, 1.0, True, "mean")
    _check(hidden, weight, index, log_probs, 0.5, True, "none")
    _check(hidden, weight, index, log_probs, 1.0, False, "mean")


@cuda
@pytest.mark.parametrize("T", [5, 100, 150])
@pytest.mark.parametrize("V", [8, 64, 700])
def test_a_record_of_the_whole_vocabulary_without_all_its_mass(T, V):
    """Nothing is left for the rest's class, in the loss and in its gradient."""
    hidden, weight, _, g = _inputs(T, V, 64)
    log_probs, index = _record(hidden, weight, V, 1.0, g)
    _check(hidden, weight, index, log_probs + math.log(0.6), 1.0, True, "mean")
    log_probs[:, 1:3] = -math.inf
    _check(hidden, weight, index, log_probs, 1.0, True, "none")


@cuda
@pytest.mark.parametrize("T", [20, 100, 150])
def test_the_largest_of_very_large_logits(T):
    """Two equal logits share each row, one of them its target; all others are far below. They are exact (one product
    and zeros), so the other one's gradient is 1/2 up to the 16-bit form of its logit (2^-10 octaves, 7e-4) and two
    roundings to bf16."""
    hidden = torch.zeros(T, 64, device="cuda")
    hidden[:, 0] = torch.linspace(8192, 32000, T, device="cuda").to(torch.bfloat16)
    weight = torch.zeros(600, 64, device="cuda")
    weight[5, 0], weight[300, 0], weight[300, 1] = 1.0, 1.0, 1.0
    hidden = hidden.to(torch.bfloat16).requires_grad_()
    weight = weight.to(torch.bfloat16).requires_grad_()
    loss = linear_cross_entropy(hidden, weight, torch.full((T,), 5, device="cuda"), reduction="sum")
    dh, dw = torch.autograd.grad(loss, (hidden, weight))
    half = torch.full((T,), 0.5, device="cuda", dtype=torch.float64)
    torch.testing.assert_close(dh[:, 1].double(), half, rtol=0, atol=0.5 * (7e-4 + 2 * U))
    half = 0.5 * hidden[:, 0].detach().double().sum()
    torch.testing.assert_close(dw[300, 0].double(), half, rtol=7e-4 + 2 * U, atol=0)
    torch.testing.assert_close(dw[5, 0].double(), -half, rtol=7e-4 + 2 * U, atol=0)


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 20011, 248077])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
def test_top_log_probs_of_masks_of_the_lowest_value(dtype, V, temperature):
    """Logits masked by the type's lowest number: most of a row, all but one entry, all of it, and beside the largest.
    Expected in 64 bits, rounded to fp32 (a masked entry may be -inf there); the bound is that of
    test_head_losses_gpu.py for the unmasked logits, and the magnitude's rounding for the masked ones."""
    g = torch.Generator(device="cuda").manual_seed(V)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = torch.randn(6, V, device="cuda", generator=g).mul_(3).to(dtype)
    logits[0, : V // 2] = low
    logits[1, 20:] = low
    logits[2, 1:] = low
    logits[3] = low
    logits[4, 7] = high
    logits[5, ::2], logits[5, 1::2] = low, -math.inf
    got, index = top_log_probs(logits, 30, temperature)
    z = logits.double()
    order = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :30]
    expected = torch.log_softmax(z / temperature, -1).gather(1, order).float()
    assert torch.equal(index, order)
    torch.testing.assert_close(got, expected, rtol=2.0 ** -21, atol=8 * 2.0 ** -24 * (20 / temperature + 32))


@cuda
@pytest.mark.parametrize("T", [20, 150])
def test_a_weight_without_numbers(T):
    """Logits that are NaN have NaN gradients, held or not."""
    hidden, weight, targets, _ = _inputs(T, 700, 64)
    weight[:, 3] = math.nan
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = linear_cross_entropy(hidden, weight, targets)
    dh, dw = torch.autograd.grad(loss, (hidden, weight))
    assert torch.isnan(loss) and torch.isnan(dh).all() and torch.isnan(dw).all()
