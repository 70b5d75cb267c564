"""Plain PyTorch definitions of every teacher/student op.

These are the CPU execution path (Gloo tests, tiny fixtures) and the oracles
the CUDA kernels are tested against. They follow the math of the Qwen3.5
hybrid text model (HF ``modeling_qwen3_5.py``: RMSNorm with (1+w) at
HF:711-723, gated RMSNorm HF:175-190, causal conv1d HF:210-226, gated delta
rule HF:318-353, attention HF:647-692) with one deliberate difference: the
convolution and delta-rule state are always carried across chunks, which the
chunked HF 5.5 path does not do (it restarts both at every multi-token call).
"""
import torch
from torch.nn import functional as F


def rmsnorm_1p(x, weight, eps):
    """Qwen RMSNorm: normalise in fp32, scale by (1 + w), cast back to x.dtype."""
    xf = x.float()
    out = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (out * (1.0 + weight.float())).type_as(x)


def gated_rmsnorm(x, gate, weight, eps):
    """GDN output norm: w * norm(x) (in x.dtype) times SiLU(gate) in fp32."""
    dtype = x.dtype
    xf = x.float()
    xf = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    out = weight * xf.to(dtype)
    out = out * F.silu(gate.float())
    return out.to(dtype)


def causal_conv1d_silu(x, state, weight):
    """Depthwise causal conv over time + SiLU with carried state.

    x: [B, T, C] (channels last), state: [B, K-1, C] previous inputs (oldest
    first), weight: [C, K] (tap K-1 multiplies the newest input).
    Returns (y [B, T, C] in x.dtype, new_state [B, K-1, C]).
    """
    K = weight.shape[-1]
    full = torch.cat([state.to(x.dtype), x], 1)
    taps = full.unfold(1, K, 1)  # [B, T, C, K]
    y = (taps.float() * weight.float()).sum(-1)
    new_state = full[:, full.shape[1] - (K - 1):]
    return F.silu(y).to(x.dtype), new_state.contiguous()


def l2norm(x, eps=1e-6):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + eps)


def gated_delta_rule(q, k, v, g, beta, state):
    """Recurrent gated delta rule with in-kernel q/k L2 norm and GQA.

    q, k: [B, T, Hk, Dk]; v: [B, T, Hv, Dv]; g (log decay), beta: [B, T, Hv];
    state: [B, Hv, Dk, Dv] fp32. Value head h reads key head h // (Hv / Hk).
    Returns (out [B, T, Hv, Dv] in v.dtype, new state fp32).
    """
    dtype = v.dtype
    rep = v.shape[2] // q.shape[2]
    q = l2norm(q.float()).repeat_interleave(rep, dim=2) * q.shape[-1] ** -0.5
    k = l2norm(k.float()).repeat_interleave(rep, dim=2)
    v, g, beta = v.float(), g.float(), beta.float()
    s = state.float()
    out = []
    for t in range(q.shape[1]):
        s = s * g[:, t, :, None, None].exp()
        mem = (s * k[:, t, :, :, None]).sum(-2)
        delta = (v[:, t] - mem) * beta[:, t, :, None]
        s = s + k[:, t, :, :, None] * delta[:, :, None, :]
        out.append((s * q[:, t, :, :, None]).sum(-2))
    return torch.stack(out, 1).to(dtype), s


def rope_tables(inv_freq, positions, dtype):
    freqs = positions.float()[:, None] * inv_freq.float()[None]
    emb = torch.cat([freqs, freqs], -1)
    return emb.cos().to(dtype), emb.sin().to(dtype)


def apply_rope(x, cos, sin):
    """Partial rotary embedding on the first ``cos.shape[-1]`` dims. x: [B,T,H,D]."""
    rot = cos.shape[-1]
    xr, xp = x[..., :rot], x[..., rot:]
    half = rot // 2
    rotated = torch.cat([-xr[..., half:], xr[..., :half]], -1)
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    return torch.cat([xr * c + rotated * s, xp], -1)


def attention(q, k_all, v_all, offset):
    """Causal GQA attention of T queries against a cache of L >= T keys.

    q: [B, T, Hq, D]; k_all, v_all: [B, L, Hkv, D]; query t sits at absolute
    position offset + t and sees keys 0..offset+t. Returns [B, T, Hq, D].
    """
    B, T, Hq, D = q.shape
    L, Hkv = k_all.shape[1], k_all.shape[2]
    rep = Hq // Hkv
    qh = q.transpose(1, 2)
    kh = k_all.transpose(1, 2).repeat_interleave(rep, 1)
    vh = v_all.transpose(1, 2).repeat_interleave(rep, 1)
    rows = torch.arange(T, device=q.device)[:, None] + offset
    cols = torch.arange(L, device=q.device)[None]
    mask = cols <= rows
    out = F.scaled_dot_product_attention(qh, kh, vh, attn_mask=mask, scale=D ** -0.5)
    return out.transpose(1, 2)


def head_loss(hidden, weight, index, log_probs, ignore, scale, tail, reduction):
    """Vocabulary-head loss against a record (see ``losses.linear_topk_kl``), in fp32 (fp64 for fp64 operands)."""
    wide = torch.float64 if hidden.dtype == torch.float64 else torch.float32
    held = (index != ignore) if log_probs is None else (index >= 0)
    if bool((held & ((index < 0) | (index >= weight.shape[0]))).any()):
        raise IndexError(f"vocabulary index outside 0..{weight.shape[0] - 1}")
    valid = held.any(-1)
    # what a row without an entry holds never meets the weight, whose gradient it would make NaN
    z = (hidden.to(wide).masked_fill(~valid[..., None], 0.0) @ weight.to(wide).t()) * scale
    log_q = z - z.logsumexp(-1, keepdim=True)
    logp = torch.zeros(index.shape, dtype=wide, device=z.device) if log_probs is None else log_probs.to(wide)
    logp = logp.masked_fill(~held, float("-inf"))
    p = logp.exp()
    index = index.masked_fill(~held, 0)
    # p log p is 0 at p = 0 (padding, and recorded log-probabilities of -inf)
    terms = p * (logp.masked_fill(p == 0, 0.0) - log_q.gather(-1, index))
    loss = terms.masked_fill(p == 0, 0.0).sum(-1)
    if tail:
        inside = torch.zeros(z.shape, dtype=torch.int32, device=z.device).scatter_add_(-1, index, held.int()) > 0
        rest = (1.0 - p.sum(-1)).clamp_min(0.0)
        counted = (rest > 0) & ~inside.all(-1) & valid
        log_rest = log_q.masked_fill(inside & counted[..., None], float("-inf")).logsumexp(-1)
        loss = loss + (rest * (rest.masked_fill(~counted, 1.0).log() - log_rest)).masked_fill(~counted, 0.0)
    loss = loss.masked_fill(~valid, 0.0)
    if reduction == "none":
        return loss
    return loss.sum() if reduction == "sum" else loss.sum() / valid.sum().clamp_min(1)


def top_log_probs(logits, k, scale):
    """k largest log-probabilities of softmax(scale * logits) and their indices, equal logits by the lowest index."""
    z = logits.float() if logits.dtype != torch.float64 else logits
    index = torch.sort(z, dim=-1, descending=True, stable=True)[1][..., :k]
    wide = z.double()  # masks of the lowest value leave fp32's range when they are scaled
    below = (wide - wide.amax(-1, keepdim=True)) * scale
    return torch.log_softmax(below, -1).gather(-1, index).to(z.dtype), index
