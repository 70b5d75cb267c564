"""Losses of the vocabulary head on CUDA, from hidden states without logits.

``head_loss`` covers the cross entropy (``log_probs`` None, ``index`` [rows, 1] targets) and the KL from a recorded
top-k (``index``, ``log_probs`` [rows, K]); the mathematics stands in ``csrc/head/head_loss.cu``. A reduced loss forms
its gradients in the forward call, from the same pass over the vocabulary as the loss; backward multiplies them by the
upstream scalar (no pass over them when it is one). An unreduced loss forms them in backward, from the upstream
gradient of each row. Backward through the same call a second time computes them again.
"""
import torch

from . import native

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, index, log_probs, ignore, scale, tail, reduction):
        ctx.args = (ignore, scale, tail)
        ctx.reduction = reduction
        ctx.save_for_backward(hidden, weight, index, log_probs)
        need_h, need_w = ctx.needs_input_grad[:2]
        eager = reduction != 0
        loss, dh, dw = native().head_loss(hidden, weight, index, log_probs, ignore, scale, tail, reduction, None,
                                          eager and need_h, eager and need_w)
        ctx.ready = (dh, dw) if eager else None
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        need_h, need_w = ctx.needs_input_grad[:2]
        hidden, weight, index, log_probs = ctx.saved_tensors
        upstream = upstream.float().contiguous()
        if ctx.reduction == 0:
            _, dh, dw = native().head_loss(hidden, weight, index, log_probs, *ctx.args, 0, upstream, need_h, need_w)
        else:
            if ctx.ready is None:
                ctx.ready = native().head_loss(hidden, weight, index, log_probs, *ctx.args, ctx.reduction, None,
                                               need_h, need_w)[1:]
            dh, dw = ctx.ready
            ctx.ready = None
            for grad, need in ((dh, need_h), (dw, need_w)):
                if need:
                    native().scale_bf16_(grad, upstream)
        return (dh if need_h else None, dw if need_w else None) + (None,) * 6


def head_loss(hidden, weight, index, log_probs, ignore, scale, tail, reduction):
    """Loss of hidden [..., C] against a record index / log_probs [..., K]; [...] or a scalar, fp32."""
    lead = hidden.shape[:-1]
    rows = hidden.reshape(-1, hidden.shape[-1])
    if rows.stride(-1) != 1 or rows.stride(0) % 8 or rows.data_ptr() % 16:
        rows = rows.contiguous()
    index = index.reshape(rows.shape[0], index.shape[-1]).to(torch.int64).contiguous()
    if log_probs is not None:
        log_probs = log_probs.reshape(index.shape).detach().float().contiguous()
    out = _HeadLoss.apply(rows, weight, index, log_probs, ignore, scale, tail, REDUCTIONS[reduction])
    return out.view(lead) if reduction == "none" else out

