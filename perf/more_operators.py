"""Measured cases of the beam-search operators: joint selection over beams and vocabulary, reordering of recurrent
states, a paged key/value cache (forking with copy on write, compaction), per-head norms with rotation written into its
pages, and the attention that reads them.

``run`` takes one pass through an operator: in plain torch operations (``own`` false), or through the package's public
functions in ``rwkv_theseus_b200.beams`` and ``rwkv_theseus_b200.paged`` (``own`` true). ``exact`` is the same result
in 64 bits.

The model sizes are the benchmark's: 27B (vocabulary 248077, 24 query and 4 key/value heads of 256, 16 attention
blocks, 48 gated-delta blocks of 48 heads of 128 x 128) and small (4096; 8 and 2 heads of 128; 2 and 6 blocks).
"""
import math

import torch

own = False

# Row widths of the recurrent states of one sequence: (dtype, elements) with how many blocks have one.
STATES = {
    "small": [("f32", 8 * 128 * 128, 6), ("bf16", 3 * 2048, 6), ("f32", 16 * 64 * 64, 2), ("bf16", 1024, 2)],
    "27b": [("f32", 48 * 128 * 128, 48), ("bf16", 3 * 10240, 48), ("f32", 80 * 64 * 64, 16), ("bf16", 5120, 16)],
}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i64": torch.int64}
ROTATED = 0.25  # share of a head that is rotated
THETA = 1e7
EPS = 1e-6


def listed():
    small = dict(layers=2, heads=2, dim=128)
    big = dict(layers=16, heads=4, dim=256)
    return [
        # One step of four beams of the small model: the smallest call, launch latency counts.
        dict(name="select_small", op="select", G=1, K=4, V=4096, dtype="bf16", end=True, penalty=0.0, first=False),
        # A batch of eight prompts with eight beams each under the 27B head, length-normalised, 32-bit logits.
        dict(name="select_batch", op="select", G=8, K=8, V=248077, dtype="f32", end=True, penalty=0.6, first=False),
        # After a selection: one of four slots has changed its parent, small model.
        dict(name="reorder_small", op="reorder", G=1, K=4, moves=1, model="small"),
        # The same for two prompts of the assembled 27B model (172 MB of states per beam).
        dict(name="reorder_27b", op="reorder", G=2, K=4, moves=2, model="27b"),
        # A token's room in every beam of one prompt, one slot forked: small model, short pages.
        dict(name="advance_small", op="advance", G=1, K=4, moves=1, page=16, prompt=35, new=9, step=0, **small),
        # Eight prompts of uneven length on the 27B cache, half of the slots forked: partly filled pages are copied.
        dict(name="advance_27b", op="advance", G=8, K=4, moves=2, page=64, prompt=517, new=45, step=37, **big),
        # Moving a small cache's pages to its front before it is saved.
        dict(name="compact_small", op="compact", R=4, each=5, pages=64, moves=13, page=16, **small),
        # The 27B cache after a batch whose longest prompts ended.
        dict(name="compact_27b", op="compact", R=12, each=17, pages=400, moves=101, page=64, **big),
        # Queries and keys of one step of four beams, small model.
        dict(name="append_small", op="append", G=1, K=4, page=16, prompt=35, new=9, step=0, queries=8, **small),
        # Four prompts with sixteen beams each at far positions of the 27B model.
        dict(name="append_27b", op="append", G=4, K=16, page=64, prompt=30011, new=70, step=101, queries=24,
             **{**big, "layers": 1}),
        # Eight beams of one long prompt: its pages are shared, the generated ones are not.
        dict(name="attend_long", op="attend", G=1, K=8, page=64, prompt=32001, new=100, step=0, queries=24, gate=True,
             **{**big, "layers": 2}),
        # Sixteen short uneven prompts with four beams each.
        dict(name="attend_batch", op="attend", G=16, K=4, page=64, prompt=300, new=45, step=97, queries=24, gate=True,
             **{**big, "layers": 2}),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "advance", "compact", "append", "attend", "attend"])
    if op == "select":
        G, K, V = _log_int(rng, 1, 8), rng.randint(1, 32), _log_int(rng, 50, 248077)
        return dict(op=op, G=G, K=min(K, 64 // G), V=V, dtype=rng.choice(["bf16", "f32"]),
                    end=rng.choice([True, False]), penalty=rng.choice([0.0, 0.0, 0.6, 1.0]),
                    first=rng.choice([False, False, False, True]))
    if op == "reorder":
        model = rng.choice(["small", "27b"])
        K = rng.randint(2, 4) if model == "27b" else _log_int(rng, 2, 32)
        G = 1 if model == "27b" else _log_int(rng, 1, 8)
        return dict(op=op, G=G, K=K, moves=rng.randint(1, K - 1), model=model)
    heads, dim = rng.choice([(1, 64), (2, 64), (2, 128), (4, 256), (3, 128)])
    shape = dict(heads=heads, dim=dim, page=rng.choice([16, 32, 64]))
    if op == "compact":
        R, each = _log_int(rng, 1, 12), _log_int(rng, 1, 17)
        pages = _log_int(rng, R * each + 1, 3 * R * each + 1)
        return dict(op=op, R=R, each=each, pages=pages, moves=rng.randint(1, min(pages - R * each, R * each)),
                    layers=_log_int(rng, 1, 16), **shape)
    G, K = _log_int(rng, 1, 8), _log_int(rng, 1, 16)
    if op == "advance":
        K = min(K, max(1, 32 // G))
        return dict(op=op, G=G, K=K, moves=rng.randint(0, K - 1), prompt=_log_int(rng, 1, 517),
                    new=_log_int(rng, 1, 130), step=rng.randint(0, 60), layers=_log_int(rng, 1, 4), **shape)
    shape.update(G=G, K=K, queries=heads * rng.choice([1, 2, 4, 6, 8, 12]), layers=rng.randint(1, 2))
    if op == "append":
        return dict(op=op, prompt=_log_int(rng, 1, 4000), new=_log_int(rng, 1, 130), step=rng.randint(0, 60), **shape)
    return dict(op=op, prompt=_log_int(rng, 1, 32001 // (G * K)), new=_log_int(rng, 1, 130),
                step=rng.randint(0, 60), gate=rng.choice([True, False]), **shape)


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _host(seed):
    return torch.Generator().manual_seed(seed)


def _parents(case, seed):
    """[G, K]: ``moves`` slots of each group take over another slot's history, the others keep their own; the slots
    that are taken over from are used evenly."""
    g = _host(seed + 1)
    rows = []
    for _ in range(case["G"]):
        order = torch.randperm(case["K"], generator=g)
        gone, kept = order[:case["moves"]], order[case["moves"]:]
        parents = torch.arange(case["K"])
        for i, slot in enumerate(gone.tolist()):
            parents[slot] = kept[i % len(kept)]
        rows.append(parents)
    return torch.stack(rows).cuda()


def _prompt_length(case, group):
    """Uneven prompts: a case's step times the group, folded into half of its longest prompt."""
    return max(1, case["prompt"] - group * case["step"] % (case["prompt"] // 2 + 1))


def _row_lengths(case):
    return [_prompt_length(case, g) + case["new"] for g in range(case["G"]) for _ in range(case["K"])]


def _page_lists(case):
    """Per row the numbers 0, 1, ... of its pages: a group's whole prompt pages are one for all of its beams, what
    was generated behind them is each beam's own. Returns (lists, number of pages in use)."""
    page, used, lists = case["page"], 0, []
    for g in range(case["G"]):
        length = _prompt_length(case, g)
        shared = list(range(used, used + length // page))
        used += len(shared)
        for _ in range(case["K"]):
            mine = -(-(length + case["new"]) // page) - len(shared)
            lists.append(shared + list(range(used, used + mine)))
            used += mine
    return lists, used


def _pool(case, pages, g):
    shape = (pages, case["layers"], 2, case["heads"], case["page"], case["dim"])
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16)


def _cache(case, seed, g):
    """A cache as a search has it in the middle: pages in any order in a pool with free ones between them."""
    lists, used = _page_lists(case)
    pages = used + used // 8 + 2 * len(lists)
    place = torch.randperm(pages, generator=_host(seed + 2)).to(torch.int32)
    width = max(len(entry) for entry in lists) + 2
    table = torch.full((len(lists), width), -1, dtype=torch.int32)
    for row, entry in enumerate(lists):
        table[row, :len(entry)] = place[entry]
    held = table[table >= 0].long()
    refs = torch.zeros(pages, dtype=torch.int32).index_add_(0, held, torch.ones(len(held), dtype=torch.int32))
    return dict(pool=_pool(case, pages, g), table=table.cuda(), refs=refs.cuda(),
                lengths=torch.tensor(_row_lengths(case), dtype=torch.int32).cuda())


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["op"] == "select":
        G, K, V = case["G"], case["K"], case["V"]
        # Logits as a head gives them: a wide bulk and a few leading tokens per beam.
        logits = torch.randn(G, K, V, device="cuda", generator=g).mul_(2.0)
        lead = torch.randint(0, V, (G, K, 12), device="cuda", generator=g)
        logits.scatter_(2, lead, torch.rand(G, K, 12, device="cuda", generator=g) * 8 + 6)
        state["logits"] = logits.to(DTYPES[case["dtype"]])
        scores = -torch.rand(G, K, device="cuda", generator=g) * 4 - 15
        lengths = torch.full((G, K), 12, dtype=torch.int32, device="cuda")
        finished = torch.zeros(G, K, dtype=torch.bool, device="cuda")
        if case["first"]:  # the first step: one beam stands for all
            scores.zero_()
            scores[:, 1:] = -math.inf
            lengths.zero_()
        elif case["end"]:
            finished = torch.rand(G, K, device="cuda", generator=g) < 0.25
            ended = torch.randint(1, 13, (G, K), device="cuda", generator=g).to(torch.int32)
            lengths = torch.where(finished, ended, lengths)
        state.update(scores=scores, lengths=lengths, finished=finished, end_token=V - 2 if case["end"] else -1)
    elif case["op"] == "reorder":
        rows = case["G"] * case["K"]
        # one buffer per kind of state, [blocks, rows, width]; the states are its blocks' tensors
        state["buffers"] = [torch.randn(count, rows, width, device="cuda", generator=g, dtype=DTYPES[dtype])
                            for dtype, width, count in STATES[case["model"]]]
        state["states"] = [tensor for buffer in state["buffers"] for tensor in buffer.unbind()]
        state["parents"] = _parents(case, seed)
    elif case["op"] == "compact":
        used = case["R"] * case["each"]
        h = _host(seed)
        places = torch.cat([torch.randperm(used, generator=h)[:used - case["moves"]],
                            used + torch.randperm(case["pages"] - used, generator=h)[:case["moves"]]])
        places = places[torch.randperm(used, generator=h)].to(torch.int32)
        refs = torch.zeros(case["pages"], dtype=torch.int32)
        refs[places.long()] = 1
        state.update(pool=_pool(case, case["pages"], g), refs=refs.cuda(),
                     table=torch.nn.functional.pad(places.view(case["R"], case["each"]), (0, 2), value=-1).cuda())
    else:
        state.update(_cache(case, seed, g))
        rows, D = case["G"] * case["K"], case["dim"]
        state["layer"] = case["layers"] - 1
        if case["op"] == "advance":
            state["parents"] = _parents(case, seed)
        else:
            # Rows of a block's input projection: per query head [query | gate], then keys, then values.
            Hq, Hkv = case["queries"], case["heads"]
            x = torch.randn(rows, (2 * Hq + 2 * Hkv) * D, device="cuda", generator=g, dtype=torch.bfloat16)
            if case["op"] == "append":
                rotated = int(D * ROTATED)
                state.update(x=x, q_weight=torch.randn(D, device="cuda", generator=g) * 0.1,
                             k_weight=torch.randn(D, device="cuda", generator=g) * 0.1,
                             inv_freq=1.0 / THETA ** (torch.arange(0, rotated, 2, device="cuda").float() / rotated))
            else:
                state["q"] = torch.randn(rows, Hq, D, device="cuda", generator=g, dtype=torch.bfloat16) * 1.5
                state["gate"] = x[:, :2 * Hq * D].view(rows, Hq, 2 * D)[..., D:] if case["gate"] else None
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from rwkv_theseus_b200 import beams, paged
    op = state["op"]
    if op == "select":
        return beams.beam_select(state["logits"], state["scores"], state["lengths"], state["finished"],
                                 end_token=state["end_token"], length_penalty=state["penalty"])
    if op == "reorder":
        beams.reorder_states_(state["states"], state["parents"])
        return state["buffers"]
    if op == "advance":
        table, lengths, refs, status = paged.advance_pages(state["pool"], state["table"], state["lengths"],
                                                           state["refs"], tokens=1, parents=state["parents"])
        return state["pool"], table, lengths, refs, status
    if op == "compact":
        table, refs, used = paged.compact_pages(state["pool"], state["table"], state["refs"])
        return state["pool"], table, refs, used
    if op == "append":
        q = paged.append_heads(state["x"], state["pool"], state["layer"], state["table"], state["lengths"],
                               state["q_weight"], state["k_weight"], state["inv_freq"], state["queries"], EPS)
        return q, state["pool"]
    return paged.paged_attention(state["q"], state["pool"], state["layer"], state["table"], state["lengths"],
                                 gate=state["gate"], group=state["K"])


@torch.no_grad()
def _run_plain(state):
    return {"select": _plain_select, "reorder": _plain_reorder, "advance": _plain_advance, "compact": _plain_compact,
            "append": _plain_append, "attend": _plain_attend}[state["op"]](state)


def _place(parents):
    """Slots of candidates given in order of rank ([G, K] parents): a parent's best child keeps the parent's slot, the
    others fill the remaining slots in order. Returns [G, K]: the rank that each slot holds."""
    G, K = parents.shape
    rank = torch.arange(K, device=parents.device)
    first = torch.full_like(parents, K).scatter_reduce_(1, parents, rank.expand(G, K), "amin")  # by parent
    keeps = first.gather(1, parents) == rank
    free = torch.sort((first < K).to(torch.int8), dim=1, stable=True)[1]  # unused slots first, in order
    order = (~keeps).long().cumsum(1) - 1
    slot = torch.where(keeps, parents, free.gather(1, order.clamp_min(0)))
    return torch.empty_like(parents).scatter_(1, slot, rank.expand(G, K))


def _plain_select(state):
    """Each beam's own best tokens first (their order is the logits', and needs no 64 bits: unique keys of the value
    above and the lower index first below), then the beams' candidates against each other in 64 bits."""
    z = state["logits"].float() + 0.0
    G, K, V = z.shape
    n = min(K, V)
    scores, lengths, finished, end = state["scores"].double(), state["lengths"], state["finished"], state["end_token"]
    top = z.amax(-1).double()
    total = (z.double() - top[..., None]).exp_().sum(-1)
    alive = total.isfinite() & top.isfinite() & scores.isfinite() & ~finished
    bits = z.view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, (~bits) & 0xFFFFFFFF, bits | 0x80000000) - 0x80000000
    order = torch.where(alive[..., None], order, torch.zeros((), dtype=torch.int64, device=z.device))
    if end >= 0:
        order[..., end] += (finished & scores.isfinite()).long()
    key = (order << 31) + (0x7FFFFFFF - torch.arange(V, device=z.device))
    token = 0x7FFFFFFF - (key.topk(n, dim=-1)[0] & 0x7FFFFFFF)
    step = z.gather(2, token).double() - top[..., None] - total.log()[..., None]
    score = torch.where(alive[..., None], scores[..., None] + step, -math.inf)
    ends = (finished & scores.isfinite())[..., None] & (token == end)
    score = torch.where(ends, scores[..., None], score)
    length = lengths + (~finished).to(torch.int32)
    rank = score / length.clamp_min(1).double().pow(state["penalty"])[..., None]
    flat = (torch.arange(K, device=z.device)[:, None] * V + token).view(G, K * n)
    flat, by_index = flat.sort(1)
    best = rank.view(G, -1).gather(1, by_index).sort(dim=1, descending=True, stable=True)[1][:, :K]
    flat, score = flat.gather(1, best), score.view(G, -1).gather(1, by_index).gather(1, best)
    held = _place(flat // V)
    flat, score = flat.gather(1, held), score.gather(1, held)
    parents, tokens = flat // V, flat % V
    return (tokens, parents, score.float(), length.gather(1, parents), finished.gather(1, parents) | (tokens == end))


def _plain_reorder(state):
    G, K = state["parents"].shape
    rows = (state["parents"] + torch.arange(G, device="cuda")[:, None] * K).view(-1)
    for tensor in state["states"]:
        tensor.copy_(tensor[rows])
    return state["buffers"]


def _count(table, pages):
    """References of each page in a table (-1 counts nowhere)."""
    entries = torch.where(table >= 0, table, pages).long().view(-1)
    return torch.zeros(pages + 1, dtype=torch.int32, device=table.device).index_add_(
        0, entries, torch.ones_like(entries, dtype=torch.int32))[:pages]


def _plain_advance(state):
    pool, page = state["pool"], state["page"]
    pages, (R, width) = pool.shape[0], state["table"].shape
    G, K = state["parents"].shape
    rows = (state["parents"] + torch.arange(G, device="cuda")[:, None] * K).view(-1)
    table, lengths = state["table"][rows], state["lengths"][rows]
    refs = _count(table, pages)
    fill = lengths % page
    at = (lengths // page).long()[:, None]  # the page that takes the new token
    last = torch.where(fill > 0, table.gather(1, at)[:, 0], -1)
    # of the rows that share a partly filled page the highest keeps it, if nobody else holds it
    before = ((last[:, None] == last[None]) & torch.ones(R, R, dtype=torch.bool, device="cuda").tril(-1)).sum(1)
    copies = (last >= 0) & (refs[last.clamp_min(0).long()] - before > 1)
    wants = copies | (fill == 0)
    free = torch.sort((refs > 0).to(torch.int8), stable=True)[1]
    fresh = free[(wants.long().cumsum(0) - 1).clamp_min(0)].to(torch.int32)
    target = torch.where(wants, fresh, last)
    table.scatter_(1, at, target[:, None])
    source, target = torch.where(copies, last, target).long(), target.long()
    kept = torch.arange(page, device="cuda") < torch.where(copies, fill, 0)[:, None]
    pool[target] = torch.where(kept[:, None, None, None, :, None], pool[source], pool[target])
    return pool, table, lengths + 1, _count(table, pages), torch.zeros(1, dtype=torch.int32, device="cuda")


def _plain_compact(state):
    pool, table, refs = state["pool"], state["table"], state["refs"]
    pages = len(refs)
    page = torch.arange(pages, device="cuda")
    used = (refs > 0).sum()
    behind = (refs > 0) & (page >= used)
    hole = (refs == 0) & (page < used)
    holes = torch.sort((~hole).to(torch.int8), stable=True)[1]  # in order, then the rest
    target = torch.where(behind, holes[(behind.long().cumsum(0) - 1).clamp_min(0)], page)
    filler = page.new_zeros(pages + 1).scatter_(0, torch.where(behind, target, pages), page)[:pages]
    source = torch.where(hole & (filler > 0), filler, page)
    for start in range(0, pages, 64):  # holes lie before what fills them
        pool[start:start + 64] = pool[source[start:start + 64]]
    table = torch.where(table >= 0, target[table.clamp_min(0).long()].to(torch.int32), table)
    refs = torch.where(page < used, refs[source], 0)
    return pool, table, refs, used.to(torch.int32)[None]


def _normed(x, weight, angle):
    """Norm of each head ([R, H, D]) scaled by 1 + weight, then the rotation of its first components."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + weight)
    half = angle.shape[-1]
    cos, sin = angle.cos()[:, None].to(x.dtype), angle.sin()[:, None].to(x.dtype)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _append(state, dtype):
    x, pool, page = state["x"], state["pool"], state["page"]
    R, Hq, Hkv, D = len(x), state["queries"], state["heads"], state["dim"]
    position = state["lengths"].long() - 1
    angle = position.double()[:, None] * state["inv_freq"].double()  # far positions need 64 bits
    q = x[:, :2 * Hq * D].view(R, Hq, 2 * D)[..., :D].to(dtype)
    k, v = x[:, 2 * Hq * D:].view(R, 2, Hkv, D).unbind(1)
    q = _normed(q, state["q_weight"].to(dtype), angle)
    k = _normed(k.to(dtype), state["k_weight"].to(dtype), angle)
    at = state["table"].gather(1, (position // page)[:, None])[:, 0].long()
    return q, k, v, at, position % page


def _plain_append(state):
    q, k, v, at, slot = _append(state, torch.float32)
    pool = state["pool"]
    pool[at, state["layer"], 0, :, slot] = k.to(torch.bfloat16)
    pool[at, state["layer"], 1, :, slot] = v
    return q.to(torch.bfloat16), pool


def _attend(state, dtype):
    R, Hq, D = state["q"].shape
    Hkv = state["heads"]
    out = torch.empty(R, Hq, D, dtype=dtype, device="cuda")
    for row in range(R):  # a row's pages as one run of keys and values
        pages = state["table"][row].clamp_min(0).long()
        kv = state["pool"][pages, state["layer"]].to(dtype).permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, D)
        s = state["q"][row].to(dtype).view(Hkv, -1, D) @ kv[0].transpose(1, 2) * D ** -0.5
        hidden = torch.arange(s.shape[-1], device="cuda") >= state["lengths"][row]
        s = s.masked_fill(hidden, -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp()
        out[row] = ((p / p.sum(-1, keepdim=True)) @ kv[1].masked_fill(hidden[:, None], 0.0)).view(Hq, D)
    if state["gate"] is not None:
        out = out / (1.0 + (-state["gate"].to(dtype)).exp())
    return out


def _plain_attend(state):
    return _attend(state, torch.float32).to(torch.bfloat16)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "select":
        rows = case["G"] * case["K"]
        return {"bytes": rows * (case["V"] * DTYPES[case["dtype"]].itemsize + 9 + 25), "flops": 3 * rows * case["V"]}
    if op == "reorder":
        width = sum(DTYPES[dtype].itemsize * size * count for dtype, size, count in STATES[case["model"]])
        read = min(case["moves"], case["K"] - case["moves"])
        return {"bytes": case["G"] * ((case["moves"] + read) * width + 8 * case["K"]), "flops": 0}
    token = case["layers"] * 2 * case["heads"] * case["dim"] * 2  # bytes of a token in every block
    if op == "compact":
        table = 4 * (case["R"] * (case["each"] + 2) + case["pages"])
        return {"bytes": 2 * case["moves"] * case["page"] * token + 2 * table, "flops": 0}
    lists, used = _page_lists(case)
    lengths = _row_lengths(case)
    if op == "advance":
        copied = sum(case["moves"] * (lengths[g * case["K"]] % case["page"]) for g in range(case["G"]))
        table = 4 * (len(lists) * (max(map(len, lists)) + 3) + used)
        return {"bytes": 2 * copied * token + 2 * table + 8 * len(lists), "flops": 0}
    rows, D = len(lists), case["dim"]
    if op == "append":
        values = rows * (case["queries"] + 2 * case["heads"]) * D
        return {"bytes": 4 * values + 8 * D + 8 * rows, "flops": 8 * values}
    shared = sum(_prompt_length(case, g) // case["page"] * case["page"] * (1 - case["K"]) for g in range(case["G"]))
    keys = sum(lengths) + shared
    moved = keys * token // case["layers"] + rows * case["queries"] * D * 2 * (2 + case["gate"])
    return {"bytes": moved + 4 * sum(map(len, lists)), "flops": 4 * sum(lengths) * case["queries"] * D}


# ---------------------------------------------------------------- the definitions in 64 bits
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "select":
        return _exact_select(state)
    if op == "reorder":
        moved = []
        for buffer in state["buffers"]:
            groups = buffer.view(len(buffer), case["G"], case["K"], -1)
            moved.append(torch.stack([groups[:, g, p] for g, row in enumerate(state["parents"].tolist()) for p in row], 1))
        return moved
    if op == "append":
        q, k, v, at, slot = _append(state, torch.float64)
        pool = state["pool"].double()
        pool[at, state["layer"], 0, :, slot] = k
        pool[at, state["layer"], 1, :, slot] = v.double()
        return q, pool
    if op == "attend":
        return _attend(state, torch.float64)
    return _exact_advance(state) if op == "advance" else _exact_compact(state)


def _exact_select(state):
    """From the whole list of a group's candidates."""
    G, K, V = state["logits"].shape
    rows = []
    for g in range(G):
        z = state["logits"][g].double()
        scores, lengths, finished = (state[name][g] for name in ("scores", "lengths", "finished"))
        value = scores.double()[:, None] + torch.log_softmax(z, -1)
        value[~(value < math.inf)] = -math.inf  # NaN as well
        value[finished] = -math.inf
        if state["end_token"] >= 0:
            value[finished, state["end_token"]] = scores.double()[finished]
        length = lengths + (~finished).int()
        rank = (value / length.clamp_min(1).double()[:, None] ** state["penalty"]).view(-1)
        # the K largest, equal ones by the lowest index: everything above the K-th, then its equals in order
        border = rank.topk(K)[0][-1]
        above, equal = (rank > border).nonzero()[:, 0], (rank == border).nonzero()[:, 0]
        chosen = torch.cat([above, equal[:K - len(above)]]).tolist()
        chosen.sort(key=lambda flat: (-rank[flat].item(), flat))
        slots, rest = {}, []
        for flat in chosen:
            rest.append(flat) if flat // V in slots else slots.setdefault(flat // V, flat)
        for slot in range(K):
            if slot not in slots:
                slots[slot] = rest.pop(0)
        flat = torch.tensor([slots[slot] for slot in range(K)], device="cuda")
        token, parent = flat % V, flat // V
        rows.append((token, parent, value.view(-1)[flat], length[parent],
                     finished[parent] | (token == state["end_token"])))
    return tuple(torch.stack(part) for part in zip(*rows))


def _exact_advance(state):
    """Row after row, on the host."""
    page, pool = state["page"], state["pool"].clone()
    table, lengths = state["table"].tolist(), state["lengths"].tolist()
    G, K = state["parents"].shape
    parents = [g * K + p for g, row in enumerate(state["parents"].tolist()) for p in row]
    table, lengths = [list(table[p]) for p in parents], [lengths[p] for p in parents]
    refs = [0] * pool.shape[0]
    for row in table:
        for entry in row:
            if entry >= 0:
                refs[entry] += 1
    free = iter([p for p, count in enumerate(refs) if count == 0])
    for row, length in enumerate(lengths):
        at, fill = divmod(length, page)
        old = table[row][at]
        if fill == 0 or refs[old] > 1:
            table[row][at] = new = next(free)
            refs[new] = 1
            if fill:
                refs[old] -= 1
                pool[new, :, :, :, :fill] = pool[old, :, :, :, :fill]
    ints = [torch.tensor(part, dtype=torch.int32, device="cuda") for part in (table, [n + 1 for n in lengths], refs, [0])]
    return (pool, *ints)


def _exact_compact(state):
    pool, table, refs = state["pool"].clone(), state["table"].clone(), state["refs"].tolist()
    used = sum(count > 0 for count in refs)
    holes = [p for p in range(used) if refs[p] == 0]
    for hole, source in zip(holes, [p for p in range(used, len(refs)) if refs[p] > 0]):
        pool[hole] = pool[source]
        table[table == source] = hole
        refs[hole], refs[source] = refs[source], 0
    return (pool, table, torch.tensor(refs, dtype=torch.int32, device="cuda"),
            torch.tensor([used], dtype=torch.int32, device="cuda"))
