"""Distillation statistics (reference ``theseus/losses.py:5-30``) and losses of the vocabulary head.

``statistics`` returns the differentiable sums ``[sum NMSE, sum cosine, count]``
over tokens, with per-token NMSE = mean((x-y)^2) / max(mean(y^2), eps). On CUDA
the fused loss kernel computes the same three sums in one pass (and the NMSE
gradient in the same kernel, see ``ops.loss``); this module is the
device-agnostic definition used on CPU and as the test oracle.

``linear_cross_entropy``, ``linear_topk_kl`` and ``top_log_probs`` score and train through the vocabulary head: the
first two take hidden states and the head's weight and never keep the logits, the third makes the teacher's record
that the second learns from.

On CUDA the two losses are fp32 and off by about 2e-7 of a logit (width / 16 x 2^-26 of it where its products add up
without rounding, 4.8e-6 at width 5120). Their gradients are bf16: the logits' gradient is rounded to bf16 once (without
the factors that all tokens share), the result once, and once more for an upstream factor that is no power of two. A
loss that is summed or averaged while gradients are recorded forms them in the forward call, all that are required, and
keeps them until its backward (outside saved-tensor hooks): score under ``torch.no_grad()``. reduction "none" forms them
in backward. There is no second and no forward-mode derivative. ``top_log_probs`` has no gradient.
"""
import math

import torch
from torch.nn import functional as F

from .ops import native, reference


def statistics(prediction, target, epsilon=1e-6, mask=None):
    x, y = prediction.float(), target.float()
    nmse = (x - y).square().mean(-1) / y.square().mean(-1).clamp_min(epsilon)
    cosine = F.cosine_similarity(x, y, dim=-1, eps=epsilon)
    weight = torch.ones_like(nmse) if mask is None else mask.float()
    return torch.stack([(nmse * weight).sum(), (cosine * weight).sum(), weight.sum()])


def loss_sum(stats, cosine_weight):
    """Training objective of summed statistics: sum NMSE + w * (token count - sum cosine)."""
    nmse_total, cos_total, count = stats[0], stats[1], stats[2]
    return nmse_total + cosine_weight * (count - cos_total)


def metrics(stats):
    """Per-token means of summed statistics: NMSE, its root (RRMS), cosine, and the token count."""
    totals = [float(v) for v in stats.detach().double().cpu()]
    tokens = totals[2]
    if not tokens > 0:
        raise ValueError("No valid validation tokens")
    per_token = totals[0] / tokens
    return {"nmse": per_token, "rrms": math.sqrt(per_token), "cosine": totals[1] / tokens, "tokens": int(tokens)}


def kl_sum(student_logits, teacher_logits):
    """Sum over tokens of KL(teacher || student) on the full vocabulary.

    CUDA tensors take the one-pass kernel (``csrc/fused/kl.cu``: online max / sums per row, per-row results
    summed here in a fixed order); otherwise two log_softmax passes (reference ``theseus/losses.py:27-30``)."""
    if student_logits.is_cuda:
        V = student_logits.shape[-1]
        s = student_logits.reshape(-1, V)
        t = teacher_logits.reshape(-1, V)
        if s.dtype not in (torch.bfloat16, torch.float32) or s.dtype != t.dtype:
            s, t = s.float(), t.float()
        return native().kl_rows(s.contiguous(), t.contiguous()).sum()
    teacher = F.log_softmax(teacher_logits.float(), dim=-1)
    student = F.log_softmax(student_logits.float(), dim=-1)
    return (teacher.exp() * (teacher - student)).sum()


def _check_temperature(temperature):
    """Its inverse times a logit has to stay in fp32's range, and a mask of -inf has to stay one."""
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be positive (1e-30 to 1e30), got {temperature}")


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _head_loss(hidden, weight, index, log_probs, ignore, scale, tail, reduction):
    """Checks what both head losses share and runs the CUDA kernels or the plain definition."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"Unknown reduction: {reduction}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"expected hidden [..., C] and weight [V, C], got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    if index.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"vocabulary indices must be int32 or int64, got {index.dtype}")
    if weight.device != hidden.device or index.device != hidden.device:
        raise ValueError("hidden states, weight and indices are on different devices")
    if index.shape != hidden.shape[:-1] + (() if log_probs is None else index.shape[-1:]):
        raise ValueError(f"indices {tuple(index.shape)} do not match hidden {tuple(hidden.shape)}")
    if not hidden.is_cuda:
        if log_probs is None:
            index = index.unsqueeze(-1)
        return reference.head_loss(hidden, weight, index.long(), log_probs, ignore, scale, tail, reduction)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("the CUDA head losses take bf16 hidden states and weight")
    if weight.stride(1) != 1 or weight.stride(0) % 8 or weight.shape[1] % 8 or weight.data_ptr() % 16:
        raise ValueError("the CUDA head losses need a width and weight row stride that are multiples of 8, unit inner "
                         "stride and 16-byte alignment")
    return native().head_loss(hidden, weight, index, log_probs, ignore, scale, tail, _REDUCTIONS[reduction])


def linear_cross_entropy(hidden, weight, targets, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of ``hidden @ weight.T`` (hidden [..., C], weight [V, C]) with ``targets`` [...], without
    keeping the logits; differentiable in ``hidden`` and ``weight``.

    Tokens whose target is ``ignore_index`` have loss 0 and gradient 0 whatever their hidden state holds, and are not
    counted by the mean (which is 0 when none is left). fp32 result: [...] for reduction "none", else a scalar. On
    CUDA a target outside the vocabulary makes its token's loss NaN and its gradient 0; on CPU it raises."""
    return _head_loss(hidden, weight, targets, None, ignore_index, 1.0, False, reduction)


def linear_topk_kl(hidden, weight, indices, log_probs, temperature=1.0, tail=True, reduction="mean"):
    """KL from a teacher's recorded top log-probabilities to the student ``softmax(hidden @ weight.T / temperature)``,
    without keeping the logits; differentiable in ``hidden`` and ``weight``.

    ``indices``, ``log_probs`` [..., K] are a record as ``top_log_probs`` makes it at the same temperature, K <= 1024;
    the indices of a token are distinct, negative ones are padding, and a token without any has loss 0 and gradient 0
    and is not counted by the mean. With ``tail`` the vocabulary outside a token's record is one more class, which
    holds the teacher's remaining mass; without it the sum runs over the recorded entries alone. ``log_probs`` get no
    gradient. fp32 result: [...] for reduction "none", else a scalar. On CUDA an index beyond the vocabulary makes its
    token's loss NaN and its gradient 0; on CPU it raises."""
    if log_probs.shape != indices.shape or log_probs.device != indices.device:
        raise ValueError(f"indices {tuple(indices.shape)} and log_probs {tuple(log_probs.shape)} must match")
    if indices.dim() < 1 or not 1 <= indices.shape[-1] <= 1024:
        raise ValueError(f"a record holds 1 to 1024 entries per token, got {tuple(indices.shape)}")
    if not log_probs.is_floating_point():
        raise TypeError("log_probs must be floating point")
    _check_temperature(temperature)
    return _head_loss(hidden, weight, indices, log_probs.detach(), -1, 1.0 / temperature, tail, reduction)


def top_log_probs(logits, k, temperature=1.0):
    """(log_probs fp32, indices int64), both [..., k]: the k largest log-probabilities of
    ``softmax(logits / temperature)`` over the last axis, largest first, equal logits by the lowest index. CUDA logits
    are bf16 or fp32 and k is at most 1024."""
    if logits.dim() < 1 or not 1 <= k <= min(logits.shape[-1], 1024):
        raise ValueError(f"k must be in 1..min(V, 1024), got {k} for logits {tuple(logits.shape)}")
    _check_temperature(temperature)
    if logits.is_cuda:
        if logits.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("top_log_probs takes bf16 or fp32 logits on CUDA")
        return native().top_log_probs(logits, k, 1.0 / temperature)
    with torch.no_grad():
        return reference.top_log_probs(logits, k, 1.0 / temperature)
