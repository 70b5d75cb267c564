"""Tuning the vocabulary head of an assembled model on the teacher's logits and on the text itself.

The migration trains every student at its own block; what is left is how the assembled model's last hidden states
meet the head. ``record_teacher`` runs the original blocks once and keeps the top log-probabilities of every token
(``losses.top_log_probs``: 12 bytes per entry instead of a vocabulary of logits). ``tune_head`` then minimises

    kl_weight * KL(teacher's record || student) + (1 - kl_weight) * next-token cross entropy

over the head's weight with AdamW on an fp32 master copy, the hidden states being those of the assembled model; and
``score`` is the mean next-token cross entropy. The losses form no logits (``losses.linear_topk_kl`` and
``losses.linear_cross_entropy``); nothing here is part of the reference, which stops at the assembled model.

Chunks are the batches of ``validation.validation_batches`` (``ids`` [B, T] on the CPU and ``reset``).
"""
import torch

from .losses import linear_cross_entropy, linear_topk_kl, top_log_probs
from .validation import _logits, replay

IGNORE = -100


def next_tokens(ids):
    """Targets of a chunk: the following token of each position, none for the last (its follower is in another chunk)."""
    return torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], IGNORE)], 1)


@torch.no_grad()
def record_teacher(runner, chunks, device, k=64, temperature=1.0, token_block=256):
    """Per chunk, on the CPU: (indices int32, log_probs fp32) [B, T, k] of the model as it stands in `runner`."""
    head = runner.model.lm_head.weight
    records = []

    def keep(_, hidden):
        parts = [top_log_probs(_logits(hidden[:, t:t + token_block], head), k, temperature)
                 for t in range(0, hidden.shape[1], token_block)]
        records.append((torch.cat([index for _, index in parts], 1).to(torch.int32).cpu(),
                        torch.cat([log_probs for log_probs, _ in parts], 1).cpu()))

    replay(runner, chunks, device, keep)
    return records


@torch.no_grad()
def hidden_states(runner, chunks, device):
    """Per chunk, on the CPU: the final hidden states [B, T, C] of the model as it stands in `runner`."""
    states = []
    replay(runner, chunks, device, lambda _, hidden: states.append(hidden.to(runner.model.lm_head.weight.dtype).cpu()))
    return states


@torch.no_grad()
def score(runner, chunks, device):
    """(mean next-token cross entropy in nats, number of scored tokens)."""
    head = runner.model.lm_head.weight
    total = torch.zeros(2, dtype=torch.float64)

    def add(index, hidden):
        targets = next_tokens(chunks[index]["ids"]).to(device)
        loss = linear_cross_entropy(hidden.to(head.dtype), head, targets, IGNORE, "none")
        total[0] += loss.double().sum().cpu()
        total[1] += (targets != IGNORE).sum().cpu()

    replay(runner, chunks, device, add)
    return (total[0] / total[1].clamp_min(1)).item(), int(total[1])


def head_loss(hidden, weight, targets, record, temperature, kl_weight):
    """The tuning objective of one chunk; a part with weight 0 is not computed."""
    loss = 0.0
    if kl_weight > 0:
        indices, log_probs = record
        loss = kl_weight * linear_topk_kl(hidden, weight, indices, log_probs, temperature)
    if kl_weight < 1:
        loss = loss + (1 - kl_weight) * linear_cross_entropy(hidden, weight, targets, IGNORE)
    return loss


def tune_head(model, chunks, states, records, device, steps, lr=1e-5, kl_weight=0.5, temperature=1.0, on_step=None):
    """`steps` AdamW updates of ``model.lm_head.weight`` in place, one chunk each, in order and again from the first.

    `states` and `records` are what ``hidden_states`` of the assembled model and ``record_teacher`` returned for
    `chunks`. Returns the losses."""
    if model.config.tie_word_embeddings:
        raise ValueError("the head shares its weight with the embedding: tuning it would change the model's input")
    if not 0 <= kl_weight <= 1:
        raise ValueError("kl_weight must lie in 0..1")
    if len(states) != len(chunks) or len(records) != len(chunks) or not chunks:
        raise ValueError("one set of hidden states and one record per chunk")
    weight = model.lm_head.weight
    master = weight.detach().float().clone()
    optimizer = torch.optim.AdamW([master], lr=lr, weight_decay=0.0)
    losses = []
    for step in range(steps):
        at = step % len(chunks)
        live = weight.detach().requires_grad_()
        record = tuple(part.to(device) for part in records[at])
        loss = head_loss(states[at].to(device), live, next_tokens(chunks[at]["ids"]).to(device), record, temperature,
                         kl_weight)
        master.grad, = (grad.float() for grad in torch.autograd.grad(loss, live))
        optimizer.step()
        with torch.no_grad():
            weight.copy_(master)
        losses.append(loss.item())
        if on_step is not None:
            on_step(step, losses[-1])
    return losses
