"""Corners of the vocabulary-head operators' plain definitions and of their public functions' checks, on CPU."""
import pytest
import torch

from rwkv_theseus_b200.losses import top_log_probs


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
