"""Measured cases of the vocabulary-head operators: next-token cross entropy and distillation from a teacher's
recorded top log-probabilities, both computed from hidden states and the head's weight with their gradients, and
the operator that records those log-probabilities from logits.

``run`` takes one pass through an operator: in plain torch operations (``own`` false), or through the package's
public functions in ``rwkv_theseus_b200.losses`` (``own`` true). ``exact`` is the same result in 64 bits.

The two head sizes are the benchmark's: vocabulary 248077 x width 5120 (27B) and 4096 x 1024 (small).
"""
import math

import torch

own = False

IGNORE = -100
BIG = {"V": 248077, "C": 5120}
SMALL = {"V": 4096, "C": 1024}


def listed():
    return [
        # Cross entropy of each token, no gradients: scoring.
        # One validation block of the small model: the smallest call, launch latency counts.
        dict(name="ce_score_small", op="ce", T=16, **SMALL, ignored=0, grad_h=False, grad_w=False),
        # One token of the 27B head, as a decoder that reports log-likelihoods scores it: reads the head once.
        dict(name="ce_score_token", op="ce", T=1, **BIG, ignored=0, grad_h=False, grad_w=False),
        # Perplexity of one training-sized chunk under the 27B head.
        dict(name="ce_score_chunk", op="ce", T=1024, **BIG, ignored=0, grad_h=False, grad_w=False),
        # Cross entropy with gradients: tuning the head (and what is below it) on next tokens.
        # A short ragged document of the small model.
        dict(name="ce_tune_small", op="ce", T=131, **SMALL, ignored=7, grad_h=True, grad_w=True),
        # One chunk of the 27B head.
        dict(name="ce_tune_chunk", op="ce", T=1024, **BIG, ignored=32, grad_h=True, grad_w=True),
        # A whole ragged context of chat data, whose prompt tokens carry no loss.
        dict(name="ce_tune_context", op="ce", T=4001, **BIG, ignored=1203, grad_h=True, grad_w=True),
        # Distillation from recorded top log-probabilities.
        # One validation block of the small model, eight recorded tokens.
        dict(name="kd_small", op="kd", T=16, **SMALL, K=8, ignored=0, ragged=False, temperature=1.0, tail=True,
             grad_h=True, grad_w=True),
        # One chunk through a frozen 27B head (the blocks below it learn), softened teacher, the rest as one class.
        dict(name="kd_frozen_chunk", op="kd", T=1024, **BIG, K=64, ignored=0, ragged=False, temperature=2.0,
             tail=True, grad_h=True, grad_w=False),
        # An odd chunk with the head learning too, records of uneven length, some tokens without one.
        dict(name="kd_tune_chunk", op="kd", T=1000, **BIG, K=20, ignored=77, ragged=True, temperature=1.0,
             tail=False, grad_h=True, grad_w=True),
        # Recording the teacher's top log-probabilities.
        # One decoded token.
        dict(name="top_token", op="top", T=1, V=BIG["V"], K=64, dtype="bf16", temperature=1.0),
        # One chunk of 27B logits.
        dict(name="top_chunk", op="top", T=1024, V=BIG["V"], K=64, dtype="bf16", temperature=2.0),
        # 32-bit logits of an odd vocabulary and a long record.
        dict(name="top_wide_f32", op="top", T=333, V=32003, K=200, dtype="f32", temperature=1.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "kd", "kd", "top"])
    T = _log_int(rng, 1, 2500)
    V = _log_int(rng, 700, BIG["V"])
    if op == "top":
        return dict(op=op, T=min(T, 1024), V=V, K=_log_int(rng, 1, 256), dtype=rng.choice(["bf16", "f32"]),
                    temperature=rng.choice([1.0, 2.0, 0.7]))
    C = 8 * _log_int(rng, 8, BIG["C"] // 8)
    case = dict(op=op, T=T, V=V, C=C, ignored=rng.choice([0, T // 5, T // 2]))
    grad_h = rng.choice([False, True, True, True])
    case.update(grad_h=grad_h, grad_w=grad_h and rng.choice([False, True, True]))
    if op == "kd":
        case.update(K=_log_int(rng, 1, 256), ragged=rng.choice([False, True]),
                    temperature=rng.choice([1.0, 2.0, 0.7]), tail=rng.choice([False, True]))
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    """Inputs of one pass. Hidden states have unit RMS as after the final norm, plus a pull of random strength
    towards their next token, so that its probability is anywhere from negligible to about 0.9."""
    g = _generator(seed)
    T, V = case["T"], case["V"]
    if case["op"] == "top":
        # Logits as a head gives them: a wide bulk and a few leading tokens per row.
        logits = torch.randn(T, V, device="cuda", generator=g).mul_(2.0)
        lead = torch.randint(0, V, (T, 6), device="cuda", generator=g)
        logits.scatter_(1, lead, torch.rand(T, 6, device="cuda", generator=g) * 8 + 8)
        return dict(case, logits=logits.to(torch.bfloat16) if case["dtype"] == "bf16" else logits)
    C = case["C"]
    weight = (torch.randn(V, C, device="cuda", generator=g) * (1.4 / math.sqrt(C))).to(torch.bfloat16)
    targets = torch.randint(0, V, (T,), device="cuda", generator=g)
    pull = torch.rand(T, 1, device="cuda", generator=g) * ((math.log(V) + 3) * case.get("temperature", 1.0) / 1.96)
    hidden = torch.randn(T, C, device="cuda", generator=g) + pull * weight[targets].float()
    dropped = torch.randperm(T, device="cuda", generator=g)[:case["ignored"]]
    state = dict(case)
    if case["op"] == "ce":
        targets[dropped] = IGNORE
        state["targets"] = targets
    else:
        # The teacher sees a hidden state near the student's; its record is made once, outside the pass.
        teacher = (hidden + torch.randn(T, C, device="cuda", generator=g)).to(torch.bfloat16)
        indices, log_probs = [], []
        for start in range(0, T, 1024):
            z = (teacher[start:start + 1024] @ weight.t()).float() / case["temperature"]
            top, index = z.topk(case["K"], dim=-1)
            log_probs.append(top - z.logsumexp(-1, keepdim=True))
            indices.append(index)
        indices, log_probs = torch.cat(indices), torch.cat(log_probs)
        if case["ragged"]:
            length = torch.randint(1, case["K"] + 1, (T, 1), device="cuda", generator=g)
            indices.masked_fill_(torch.arange(case["K"], device="cuda") >= length, -1)
        indices[dropped] = -1
        state.update(indices=indices, log_probs=log_probs)
    state["hidden"] = hidden.to(torch.bfloat16).requires_grad_(case["grad_h"])
    state["weight"] = weight.requires_grad_(case["grad_w"])
    return state


def _wanted(state):
    return [state[name] for name, flag in (("hidden", "grad_h"), ("weight", "grad_w")) if state[flag]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from rwkv_theseus_b200 import losses
    if state["op"] == "top":
        return losses.top_log_probs(state["logits"], state["K"], temperature=state["temperature"])
    if state["op"] == "ce":
        loss = losses.linear_cross_entropy(state["hidden"], state["weight"], state["targets"], ignore_index=IGNORE,
                                           reduction="mean" if state["grad_h"] else "none")
    else:
        loss = losses.linear_topk_kl(state["hidden"], state["weight"], state["indices"], state["log_probs"],
                                     temperature=state["temperature"], tail=state["tail"])
    wanted = _wanted(state)
    grads = torch.autograd.grad(loss, wanted) if wanted else ()
    return (loss.detach(), *grads)


@torch.no_grad()
def _run_plain(state):
    if state["op"] == "top":
        return _plain_top(state)
    h, w = state["hidden"].float(), state["weight"].float()
    scale = 1.0 if state["op"] == "ce" else 1.0 / state["temperature"]
    z = (h @ w.t()) * scale
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp_()
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    if state["op"] == "ce":
        valid = state["targets"] != IGNORE
        count = valid.sum().clamp_min(1)
        index = state["targets"].clamp_min(0)[:, None]
        loss = torch.where(valid, (lse - z.gather(1, index))[:, 0], 0.0)
        if not state["grad_h"]:
            return (loss,)
        loss = loss.sum() / count
        dz = e.div_(total)
        dz.scatter_add_(1, index, torch.full_like(lse, -1.0))
    else:
        index, logp = state["indices"], state["log_probs"].float()
        held = index >= 0
        valid = held.any(-1)
        count = valid.sum().clamp_min(1)
        index = index.clamp_min(0)
        p = torch.where(held, logp.exp(), 0.0)
        zk = z.gather(1, index)
        kl = torch.where(held & (p > 0), p * (logp - (zk - lse)), 0.0).sum(-1)
        dz = e.div_(total)
        if state["tail"]:
            rest = (1.0 - p.sum(-1, keepdim=True)).clamp_min(0.0)
            tail_z = _drop(z, index, held)
            tail_top = tail_z.amax(-1, keepdim=True)
            tail_e = tail_z.sub_(tail_top).exp_()
            tail_sum = tail_e.sum(-1, keepdim=True)
            tail_log_q = tail_top + tail_sum.log() - lse
            kl = kl + torch.where(rest > 0, rest * (rest.log() - tail_log_q), 0.0)[:, 0]
            dz.mul_(p.sum(-1, keepdim=True) + rest)
            dz.sub_(tail_e.mul_(rest / tail_sum))
        else:
            dz.mul_(p.sum(-1, keepdim=True))
        dz.scatter_add_(1, index, -p)
        loss = torch.where(valid, kl, 0.0).sum() / count
    out = [loss]
    if state["grad_h"]:
        dz.mul_((valid.float() * scale / count)[:, None])
        out.append((dz @ w).to(torch.bfloat16))
    if state["grad_w"]:
        out.append((dz.t() @ h).to(torch.bfloat16))
    return tuple(out)


def _drop(z, index, held):
    """Copy of ``z`` with the held entries of each row at -inf."""
    keep = torch.zeros_like(z, dtype=torch.int8)
    keep.scatter_add_(1, index, held.to(torch.int8))
    return z.masked_fill(keep > 0, float("-inf"))


def _plain_top(state):
    """Unique 64-bit keys (the value's order above, the lower index first below) make equal logits exact."""
    z = state["logits"].float() + 0.0
    bits = z.view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, (~bits) & 0xFFFFFFFF, bits | 0x80000000) - 0x80000000
    key = (order << 31) + (0x7FFFFFFF - torch.arange(z.shape[1], device=z.device))
    index = 0x7FFFFFFF - (key.topk(state["K"], dim=-1)[0] & 0x7FFFFFFF)
    z = z / state["temperature"]
    top = z.amax(-1, keepdim=True)
    lse = top + (z - top).exp_().sum(-1, keepdim=True).log()
    return z.gather(1, index) - lse, index


def work(case):
    T, V = case["T"], case["V"]
    if case["op"] == "top":
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": T * V * size + T * case["K"] * 12, "flops": 2 * T * V}
    C = case["C"]
    live = T - case["ignored"]
    moved = 2 * V * C + 2 * live * C + 4
    moved += 8 * T if case["op"] == "ce" else 12 * T * case["K"]
    moved += 2 * T * C * case["grad_h"] + 2 * V * C * case["grad_w"]
    return {"bytes": moved, "flops": 2 * live * V * C * (1 + case["grad_h"] + case["grad_w"])}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "top":
        z = state["logits"].double() + 0.0
        index = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :case["K"]]
        return torch.log_softmax(z / case["temperature"], -1).gather(1, index), index
    h = state["hidden"].detach().double().requires_grad_(case["grad_h"])
    w = state["weight"].detach().double().requires_grad_(case["grad_w"])
    if case["op"] == "ce":
        loss = torch.nn.functional.cross_entropy(h @ w.t(), state["targets"], ignore_index=IGNORE,
                                                 reduction="mean" if case["grad_h"] else "none")
    else:
        log_q = torch.log_softmax(h @ w.t() / case["temperature"], -1)
        held = state["indices"] >= 0
        index = state["indices"].clamp_min(0)
        logp = state["log_probs"].double().masked_fill(~held, 0.0)
        p = logp.exp() * held
        kl = (p * (logp - log_q.gather(1, index))).sum(-1)
        if case["tail"]:
            inside = torch.zeros(log_q.shape, dtype=torch.int32, device="cuda").scatter_add_(1, index, held.int()) > 0
            rest = 1 - p.sum(-1)
            tail = rest * (rest.clamp_min(1e-300).log() - log_q.masked_fill(inside, -math.inf).logsumexp(-1))
            kl = kl + tail.masked_fill(rest <= 0, 0.0)
        valid = held.any(-1)
        loss = kl.masked_fill(~valid, 0.0).sum() / valid.sum().clamp_min(1)
    wanted = [t for t in (h, w) if t.requires_grad]
    grads = torch.autograd.grad(loss, wanted) if wanted else ()
    return (loss.detach(), *(grad.detach() for grad in grads))
