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


@torch.no_grad()
def place_children(parents):
    """Slots of a group's K chosen candidates, given by rank (``parents`` [G, K]): a parent's best child keeps the
    parent's slot, the others fill the slots that are left in order. Returns [G, K]: the rank that each slot takes."""
    held = torch.empty_like(parents)
    for g, row in enumerate(parents.tolist()):
        slots = {}
        for rank, parent in enumerate(row):
            slots.setdefault(parent, rank)
        rest = [rank for rank in range(len(row)) if rank not in slots.values()]
        for slot in range(len(row)):
            held[g, slot] = slots[slot] if slot in slots else rest.pop(0)
    return held


@torch.no_grad()
def beam_select(logits, scores, lengths, finished, end_token, length_penalty):
    """One step of beam search over [G, K, V] (see ``beams.beam_select``), ranked in 64 bits."""
    G, K, V = logits.shape
    value = scores.double()[..., None] + torch.log_softmax(logits.double(), -1)
    fit = scores.isfinite()
    value = value.masked_fill(~((value < float("inf")) & (fit & ~finished)[..., None]), float("-inf"))
    if end_token >= 0:
        value[..., end_token] = torch.where(finished & fit, scores.double(), value[..., end_token])
    length = lengths + (~finished).to(lengths.dtype)
    rank = value / length.clamp_min(1).double().pow(length_penalty)[..., None]
    # of equal ranks the lowest beam, then the largest logit (a score of 1e16 swallows it), then the lowest token
    order = logits.double().masked_fill(value == float("-inf"), float("-inf"))
    order = order.sort(dim=-1, descending=True, stable=True)[1]
    rank = rank.gather(-1, order).flatten(1)
    best = rank.sort(dim=1, descending=True, stable=True)[1][:, :K]
    best = best // V * V + order.flatten(1).gather(1, best)
    best = best.gather(1, place_children(best // V))
    parents, tokens = best // V, best % V
    return (tokens, parents, value.flatten(1).gather(1, best).float(), length.gather(1, parents),
            finished.gather(1, parents) | (tokens == end_token))


def parent_rows(parents):
    """Rows [G * K] of the parents [G, K]; an index outside a group stands for the slot itself."""
    G, K = parents.shape
    own = torch.arange(K, device=parents.device).expand(G, K)
    inside = torch.where((parents >= 0) & (parents < K), parents, own)
    return (inside + torch.arange(G, device=parents.device)[:, None] * K).flatten()


@torch.no_grad()
def advance_pages(pool, table, lengths, refs, tokens, parents, live):
    """Row after row, as ``paged.advance_pages`` defines it. Returns (table, lengths, refs, status)."""
    pages, page, (R, width) = pool.shape[0], pool.shape[4], table.shape
    old, length, count = table.tolist(), lengths.tolist(), refs.tolist()
    status = 0
    source = list(range(R))
    if parents is not None:
        source = parent_rows(parents).tolist()
        status = 4 * bool(((parents < 0) | (parents >= parents.shape[1])).any())
    alive = [True] * R if live is None else live.flatten().tolist()
    new = [list(old[source[r]]) if alive[r] else [-1] * width for r in range(R)]
    length = [min(max(length[source[r]], 0), width * page) if alive[r] else 0 for r in range(R)]
    for rows, change in ((old, -1), (new, 1)):
        for row in rows:
            for entry in row:
                if 0 <= entry < pages:
                    count[entry] += change
    free = iter([p for p in range(pages) if count[p] <= 0])

    def take():
        nonlocal status
        found = next(free, -1)
        if found < 0:
            status |= 1
        else:
            count[found] = 1
        return found

    for r in range(R):
        if not alive[r] or tokens == 0:
            continue
        have, need, fill = -(-length[r] // page), -(-(length[r] + tokens) // page), length[r] % page
        if need > width:
            status |= 2
            continue
        last = new[r][have - 1] if fill else -1
        if 0 <= last < pages and count[last] > 1:
            new[r][have - 1] = found = take()
            count[last] -= 1
            if found >= 0:
                pool[found, ..., :fill, :] = pool[last, ..., :fill, :]
        for slot in range(have, need):
            new[r][slot] = take()
        length[r] += tokens
    return (torch.tensor(new, dtype=torch.int32).view(R, width), torch.tensor(length, dtype=torch.int32),
            torch.tensor(count, dtype=torch.int32), torch.tensor([status], dtype=torch.int32))


@torch.no_grad()
def compact_pages(pool, table, refs):
    """Pages in use moved into the free ones before them (see ``paged.compact_pages``). Returns (table, refs, used)."""
    taken = refs > 0
    used = int(taken.sum())
    holes = (~taken[:used]).nonzero()[:, 0]
    behind = taken[used:].nonzero()[:, 0] + used
    pool[holes] = pool[behind]
    target = torch.arange(len(refs))
    target[behind] = holes
    inside = (table >= 0) & (table < len(refs))
    table = torch.where(inside, target[table.long().clamp(0, len(refs) - 1)].to(torch.int32), table)
    refs = refs.clone()
    refs[holes] = refs[behind]
    refs[behind] = 0
    return table, refs, torch.tensor([used], dtype=torch.int32)


def _slots(pool, table, positions):
    """(valid, page, slot) of the positions [R, T] of each row."""
    page = pool.shape[4]
    at = (positions.clamp_min(0) // page).long()
    inside = (positions >= 0) & (at < table.shape[1])
    entry = table.gather(1, at.clamp_max(table.shape[1] - 1)).long()
    return inside & (entry >= 0) & (entry < pool.shape[0]), entry, (positions.clamp_min(0) % page).long()


@torch.no_grad()
def store_pages(pool, block, table, lengths, keys, values):
    """``keys``, ``values`` [N, T, H, D] as the last T tokens of every (R / N)-th row."""
    N, T = keys.shape[:2]
    every = table.shape[0] // N
    positions = lengths[::every, None] - T + torch.arange(T)
    valid, entry, slot = _slots(pool, table[::every], positions)
    for kind, x in enumerate((keys, values)):
        pool[entry[valid], block, kind, :, slot[valid]] = x[valid].to(pool.dtype)


@torch.no_grad()
def append_heads(x, pool, block, table, lengths, q_weight, k_weight, inv_freq, heads, eps):
    """Norm and rotation of a token's queries and keys, keys and values into their pages (see ``paged.append_heads``)."""
    H, D = pool.shape[3], pool.shape[5]
    R = x.shape[0]
    q = x[:, :2 * heads * D].reshape(R, heads, 2 * D)[..., :D]
    k, v = x[:, 2 * heads * D:].reshape(R, 2, H, D).unbind(1)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    angle = (lengths - 1).clamp_min(0).double()[:, None] * inv_freq.double()
    cos, sin = torch.cat([angle, angle], -1).cos().to(wide), torch.cat([angle, angle], -1).sin().to(wide)

    def turned(y, weight):
        y = y.to(wide)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * (1.0 + weight.to(wide))
        return apply_rope(y[None], cos, sin)[0]  # rows as time: its [B, T, H, D] has one angle per T

    q, k = turned(q, q_weight), turned(k, k_weight)
    store_pages(pool, block, table, lengths, k[:, None], v[:, None])
    return q.to(x.dtype)


@torch.no_grad()
def paged_attention(q, pool, block, table, lengths, gate):
    """One token per row over the keys of its pages (see ``paged.paged_attention``)."""
    R, Hq, D = q.shape
    H, page, width = pool.shape[3], pool.shape[4], table.shape[1]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros(R, Hq, D, dtype=wide)
    positions = torch.arange(width * page).expand(R, -1)
    valid, entry, slot = _slots(pool, table, positions)
    valid = valid & (positions < lengths[:, None])
    for r in range(R):
        if not valid[r].any():
            continue
        k, v = (pool[entry[r][valid[r]], block, kind, :, slot[r][valid[r]]].to(wide) for kind in (0, 1))  # [n, H, D]
        s = torch.einsum("hgd,nhd->hgn", q[r].to(wide).view(H, -1, D), k) * D ** -0.5
        out[r] = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(Hq, D)
    if gate is not None:
        out = out * torch.sigmoid(gate.to(wide))
    return out.to(q.dtype)
