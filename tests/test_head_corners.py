"""Corners of the vocabulary-head operators' plain definitions and of their public functions' checks, on CPU."""
import math

import pytest
import torch

from rwkv_theseus_b200.losses import linear_cross_entropy, linear_topk_kl, top_log_probs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
def test_top_log_probs_of_masks_of_the_lowest_value(dtype, temperature):
    """A row without an unmasked logit is uniform, whatever the temperature makes of the type's lowest number."""
    low = torch.finfo(dtype).min
    logits = torch.tensor([[1.0, low, 3.0, low, low], [low] * 5], dtype=dtype)
    log_probs, index = top_log_probs(logits, 5, temperature)
    assert index.tolist() == [[2, 0, 1, 3, 4], [0, 1, 2, 3, 4]]
    expected = torch.log_softmax(logits.double() / temperature, -1).gather(1, index).float()
    torch.testing.assert_close(log_probs, expected, rtol=2.0 ** -20, atol=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
@pytest.mark.parametrize("value", [math.nan, math.inf, -3e38])
def test_masked_rows_hold_anything(dtype, value):
    """Rows without a target or a record have loss 0 and gradient 0 and leave the weight's gradient alone."""
    g = torch.Generator().manual_seed(5)
    hidden = torch.randn(6, 8, generator=g).to(dtype)
    weight = torch.randn(20, 8, generator=g).to(dtype)
    targets = torch.tensor([1, -100, 19, -100, 0, 7])
    masked = targets == -100
    log_probs, indices = top_log_probs(torch.randn(6, 20, generator=g), 3)
    indices[masked] = -1
    for call in (lambda h, w: linear_cross_entropy(h, w, targets),
                 lambda h, w: linear_topk_kl(h, w, indices, log_probs, 2.0),
                 lambda h, w: linear_topk_kl(h, w, indices, log_probs, tail=False, reduction="sum")):
        results = []
        for content in (0.0, value):
            h = hidden.masked_fill(masked[:, None], content).requires_grad_()
            w = weight.clone().requires_grad_()
            loss = call(h, w)
            results.append((loss.detach(), *torch.autograd.grad(loss, (h, w))))
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert not results[1][1][masked].any()


@pytest.mark.parametrize("temperature", [math.inf, math.nan, 1e-31, 1e31])
def test_temperatures_that_leave_no_scale(temperature):
    """1 / temperature times a logit has to stay a number of fp32's range (at infinity 0 x -inf is none)."""
    hidden, weight = torch.randn(3, 8), torch.randn(20, 8)
    log_probs, indices = top_log_probs(torch.randn(3, 20), 4)
    with pytest.raises(ValueError, match="temperature"):
        linear_topk_kl(hidden, weight, indices, log_probs, temperature)
    with pytest.raises(ValueError, match="temperature"):
        top_log_probs(torch.randn(3, 20), 4, temperature)
