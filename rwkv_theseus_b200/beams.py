"""Beam search over assembled, partly migrated and original models.

``beam_select`` chooses a step's hypotheses over beams and vocabulary, ``reorder_states_`` lets recurrent states follow
them in place, ``paged`` does the same for keys and values without moving them, and ``beam_search`` is the decode loop
over all three (greedy decoding is ``inference.generate``).

Nothing of a step is read back by the host, and every buffer keeps its address, so a step can be captured as a CUDA
graph, key/value cache included. None of this records gradients; nothing here is part of the reference.
"""
import math

import torch

from .models.runner import adapters, isolated_state
from .ops import native, reference
from .paged import PagedCache, check_parents
from .validation import _logits

MAX_BEAMS = 32  # of a group on CUDA


def beam_select(logits, scores, lengths, finished, end_token=-1, length_penalty=0.0):
    """(tokens int64, parents int64, scores fp32, lengths int32, finished bool), all [G, K]: one step of beam search
    for G groups of K beams.

    ``logits`` [G, K, V] of the next token (on CUDA bf16 or fp32, at most 32 beams and 4161536 tokens); ``scores``
    [G, K] fp32, the sums of the beams' log-probabilities; ``lengths`` [G, K] int32, their generated tokens;
    ``finished`` [G, K] bool. A running beam offers each token at score + log_softmax(logits), and is one token longer
    with it; a finished one offers itself alone, as one more ``end_token`` at its old score and length. A beam whose
    score is not finite, or whose logits hold a NaN or +inf or are all -inf, offers nothing better than -inf. Of a
    group's K * V candidates the K with the largest score / max(length, 1)^length_penalty are kept, ranked in 64 bits,
    equal ones by the lowest beam, then the largest logit, then the lowest token.

    They are not sorted: a parent's best child takes the parent's slot, and the others fill the slots that are left in
    order of rank, so that what a surviving beam holds stays where it is. ``parents`` are slots of the same group;
    ``end_token`` -1: no token ends a beam. To start from one state per group, give its K beams the same logits and
    the scores 0, -inf, -inf, ..."""
    if logits.is_cuda:
        return tuple(native().beam_select(logits, scores, lengths, finished, end_token, length_penalty))
    if logits.dim() != 3 or logits.numel() == 0:
        raise ValueError(f"expected logits [groups, beams, vocabulary], got {tuple(logits.shape)}")
    G, K, V = logits.shape
    for name, part, dtype in (("scores", scores, torch.float32), ("lengths", lengths, torch.int32),
                              ("finished", finished, torch.bool)):
        if part.shape != (G, K):
            raise ValueError(f"{name} {tuple(part.shape)} does not match logits {tuple(logits.shape)}")
        if part.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {part.dtype}")
        if part.device != logits.device:
            raise ValueError(f"{name} and logits are on different devices")
    if not -1 <= end_token < V:
        raise ValueError(f"end_token must be -1 or in 0..{V - 1}, got {end_token}")
    if not -16.0 <= length_penalty <= 16.0:
        raise ValueError(f"length_penalty must lie in -16..16, got {length_penalty}")
    if not logits.is_floating_point():
        raise TypeError("logits must be floating point")
    return reference.beam_select(logits, scores, lengths, finished, end_token, length_penalty)


def reorder_states_(states, parents):
    """Rows of each tensor of ``states`` ([G * K, ...], contiguous, any type) replaced by their parents' rows, in
    place: slot k of group g takes what slot ``parents[g, k]`` held (int64 [G, K], any indices of the group; one
    outside it leaves its slot alone). Rows that stay are not touched. The tensors must not overlap; on CUDA a group has
    at most 32 beams."""
    if parents.is_cuda:
        return native().reorder_rows_(list(states), parents)
    states = list(states)
    rows, device = parents.numel(), parents.device
    check_parents(parents, rows, device)
    spans = [(parents.data_ptr(), parents.data_ptr() + parents.nbytes)] if parents.is_contiguous() else []
    for state in states:
        if state.dim() < 1 or state.shape[0] != rows:
            raise ValueError(f"expected states of {rows} rows, got {tuple(state.shape)}")
        if not state.is_contiguous():
            raise ValueError("states must be contiguous")
        if state.device != device:
            raise ValueError("states and parents are on different devices")
        size = state.nbytes
        if size:
            start = state.data_ptr()
            spans.append((start, start + size))
    spans.sort()
    if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
        raise ValueError("states and parents must not overlap")
    source = reference.parent_rows(parents)
    with torch.no_grad():
        for state in states:
            state.copy_(state[source])


def _spread(state, beams):
    return {name: part.repeat_interleave(beams, 0) for name, part in state.items()}


def _to_beams(runner, beams, new_tokens, page):
    """The cache of G prompts as that of G * beams sequences: recurrent states repeated, keys and values in pages
    that a group's beams share. Returns the ``PagedCache`` (None without full-attention blocks)."""
    cache = runner.cache
    for adapter in adapters(runner.model).values():
        adapter.state = _spread(adapter.state, beams)
    kept = [layer for layer in cache.layers if "keys" in layer]
    for layer in cache.layers:
        if "recurrent" in layer:
            layer.update(_spread({name: layer[name] for name in ("conv", "recurrent")}, beams))
    if not kept:
        return None
    groups, _, heads, dim = kept[0]["keys"].shape
    prompt = cache.cursor
    device, dtype = kept[0]["keys"].device, kept[0]["keys"].dtype
    # every beam may end up with pages of its own behind the prompt's whole ones
    pages = groups * (prompt // page + beams * (-(-(prompt % page + new_tokens) // page)))
    paged = PagedCache(len(kept), heads, dim, groups * beams, prompt + new_tokens, max(pages, 1), page, device, dtype)
    first = torch.zeros(groups, beams, dtype=torch.bool, device=device)
    first[:, 0] = True
    paged.advance_(prompt, live=first)
    for index, layer in enumerate(kept):
        paged.store_(index, layer["keys"][:, :prompt], layer["values"][:, :prompt])
        for name in ("keys", "values", "length"):
            del layer[name]
        layer["paged"] = (paged, index, beams)
    paged.advance_(0, parents=torch.zeros(groups, beams, dtype=torch.int64, device=device))
    return paged


class _Search:
    """A search between two steps. Its tensors keep their addresses."""

    def __init__(self, runner, logits, beams, new_tokens, end_token, length_penalty, page):
        groups, device = logits.shape[0], logits.device
        self.runner, self.end_token, self.length_penalty = runner, end_token, length_penalty
        self.head = runner.model.lm_head.weight
        scores = torch.full((groups, beams), -math.inf, device=device)
        scores[:, 0] = 0.0
        none = torch.zeros(groups, beams, dtype=torch.int32, device=device)
        self.tokens, self.parents, self.scores, self.lengths, self.finished = beam_select(
            logits[:, None].expand(groups, beams, -1), scores, none, none.bool(), end_token, length_penalty)
        # one state per prompt: nothing has to move after the first selection
        self.parents.copy_(torch.arange(beams, device=device).expand(groups, beams))
        self.paged = _to_beams(runner, beams, new_tokens, page)
        self.history = torch.zeros(groups * beams, new_tokens, dtype=torch.int64, device=device)
        self.at = torch.zeros(1, dtype=torch.int64, device=device)

    def recurrent(self):
        """(holder, name) of each recurrent state."""
        layers = [(layer, name) for layer in self.runner.cache.layers if "recurrent" in layer
                  for name in ("conv", "recurrent")]
        return layers + [(adapter.state, name) for adapter in adapters(self.runner.model).values()
                         for name in adapter.state]

    def record(self, *states):
        """The last selection's tokens join the histories, which (and ``states``) follow it first."""
        reorder_states_([*states, self.history], self.parents)
        self.history.index_copy_(1, self.at, self.tokens.view(-1, 1))
        self.at += 1

    def step(self):
        self.record(*(holder[name] for holder, name in self.recurrent()))
        if self.paged is not None:
            self.paged.advance_(1, self.parents, ~self.finished)
        hidden = self.runner.forward(self.tokens.view(-1, 1))
        logits = _logits(hidden[:, -1], self.head).view(*self.tokens.shape, -1)
        chosen = beam_select(logits, self.scores, self.lengths, self.finished, self.end_token, self.length_penalty)
        for mine, new in zip((self.tokens, self.parents, self.scores, self.lengths, self.finished), chosen):
            mine.copy_(new)

    def result(self):
        """(ids [G, K, tokens so far], scores [G, K], lengths [G, K]), best first."""
        rank = self.scores.double() / self.lengths.clamp_min(1).double().pow(self.length_penalty)
        order = rank.sort(dim=1, descending=True, stable=True)[1]
        ids = self.history.view(*order.shape, -1)
        return (ids.gather(1, order[..., None].expand_as(ids)), self.scores.gather(1, order),
                self.lengths.gather(1, order))


class _StepGraph:
    """A search's step captured as a CUDA graph (after an eager one, which has measured the GEMM tiles).

    The forward returns new convolution windows and student states; the captured step copies them back into the
    buffers that it read, so that replays advance like eager steps."""

    def __init__(self, search):
        self.search = search
        cache = search.runner.cache
        buffers = [(holder, name, holder[name]) for holder, name in search.recurrent()]
        states = {index: dict(adapter.state) for index, adapter in adapters(search.runner.model).items()}
        cursor = cache.cursor
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            search.step()
            for (_, _, buffer), (holder, name) in zip(buffers, search.recurrent()):
                if holder[name] is not buffer:
                    buffer.copy_(holder[name])
        # capture ran nothing: the states are still the buffers'
        for holder, name, buffer in buffers:
            holder[name] = buffer
        for index, adapter in adapters(search.runner.model).items():
            adapter.state = states[index]
        cache.cursor = cursor

    def step(self):
        self.graph.replay()
        self.search.runner.cache.cursor += 1


@torch.no_grad()
def beam_search(runner, prompt, new_tokens, beams=4, end_token=-1, length_penalty=0.0, prefill_chunk=4096, page=64,
                on_token=None, graph=False):
    """The ``beams`` best continuations of each prompt of ``prompt`` [G, T] that a beam search finds, best first:
    (ids [G, beams, new_tokens], scores [G, beams], lengths [G, beams]).

    A continuation ends with ``end_token`` (its ids are followed by more of them, and its length counts the first) or
    after ``new_tokens``. Scores are sums of log-probabilities; the order is that of score / length^length_penalty
    (see ``beam_select``). ``page``: tokens in a page of the key/value cache (of full-attention blocks that were
    not replaced, whose heads have 64, 128 or 256 components on CUDA). ``on_token(step)`` is called after each decode
    step. ``graph=True`` replays the steps as a CUDA graph after the first. The runner's own cache and states are left as
    they are."""
    if prompt.dim() != 2 or prompt.numel() == 0:
        raise ValueError(f"expected prompts [groups, tokens], got {tuple(prompt.shape)}")
    if new_tokens < 1 or beams < 1 or prefill_chunk < 1:
        raise ValueError("beam search needs at least one beam, one new token and one token per prefill chunk")
    if graph and not prompt.is_cuda:
        raise ValueError("graph steps need CUDA")
    if prompt.is_cuda and beams > MAX_BEAMS:
        raise ValueError(f"beam search takes at most {MAX_BEAMS} beams on CUDA, got {beams}")
    every = 16  # steps between two looks at whether all beams have ended
    with isolated_state(runner):
        for start in range(0, prompt.shape[1], prefill_chunk):
            hidden = runner.forward(prompt[:, start:start + prefill_chunk])
        logits = _logits(hidden[:, -1], runner.model.lm_head.weight)
        search = stepper = _Search(runner, logits, beams, new_tokens, end_token, length_penalty, page)
        for step in range(1, new_tokens):
            if end_token >= 0 and step % every == 0 and bool(search.finished.all()):
                break  # what follows would add end tokens alone
            stepper.step()
            if on_token is not None:
                on_token(step)
            if graph and stepper is search and step + 1 < new_tokens:
                stepper = _StepGraph(search)
        search.record()
        if search.paged is not None:
            search.paged.check()
        ids, scores, lengths = search.result()
        if end_token >= 0:
            ids = ids.masked_fill(torch.arange(new_tokens, device=ids.device) >= lengths[..., None], end_token)
        return ids, scores, lengths
