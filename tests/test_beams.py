"""Beam search on CPU: the plain definitions against independent ones, whole searches, and the refusals of the public
functions."""
import itertools
import math

import pytest
import torch

from fixtures import tiny_model
from rwkv_theseus_b200.beams import beam_search, beam_select, reorder_states_
from rwkv_theseus_b200.inference import generate
from rwkv_theseus_b200.models.runner import Runner, install
from rwkv_theseus_b200.paged import (PagedCache, advance_pages, append_heads, compact_pages, paged_attention,
                                     store_pages)


# ---------------------------------------------------------------- selection
def _step(G=2, K=3, V=11, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(G, K, V, generator=g) * 3
    return (logits, -torch.rand(G, K, generator=g) * 5, torch.randint(1, 6, (G, K), generator=g).int(),
            torch.zeros(G, K, dtype=torch.bool))


def _by_hand(logits, scores, lengths, finished, end, penalty):
    """Candidate by candidate: (rank, beam, token, value) of each group, best first."""
    G, K, V = logits.shape
    groups = []
    for g in range(G):
        found = []
        for b, v in itertools.product(range(K), range(V)):
            z = logits[g, b].double()
            value = -math.inf
            score = scores[g, b].double().item()
            if math.isfinite(score):
                if finished[g, b]:
                    value = score if v == end else -math.inf
                else:
                    below = z - z.max()  # (next to a mask of -3.4e38 the logarithm of a sum would vanish)
                    value = score + (below[v] - below.logsumexp(0)).item()
                    value = value if value < math.inf else -math.inf
            length = lengths[g, b].item() + (not finished[g, b])
            found.append((value / max(length, 1) ** penalty, b, v, value))
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        groups.append(found[:K])
    return groups


def _check_step(args, end, penalty):
    logits, scores, lengths, finished = args
    tokens, parents, new_scores, new_lengths, ended = beam_select(*args, end_token=end, length_penalty=penalty)
    for g, chosen in enumerate(_by_hand(*args, end, penalty)):
        got = [(parents[g, k].item(), tokens[g, k].item()) for k in range(len(chosen))]
        assert sorted(got) == sorted((b, v) for _, b, v, _ in chosen)
        values = {(b, v): value for _, b, v, value in chosen}
        firsts, rest = {}, []
        for _, b, v, _ in chosen:
            if b in firsts:
                rest.append((b, v))
            else:
                firsts[b] = (b, v)
        for k, pair in enumerate(got):
            assert pair == (firsts[k] if k in firsts else rest.pop(0))
            b, v = pair
            if math.isinf(values[pair]):
                assert new_scores[g, k] == values[pair]
            else:
                assert abs(new_scores[g, k].item() - values[pair]) <= 2 ** -23 * abs(values[pair])
            assert new_lengths[g, k] == lengths[g, b] + (not finished[g, b])
            assert ended[g, k] == bool(finished[g, b] or v == end)


@pytest.mark.parametrize("penalty", [0.0, 0.7, -0.5])
@pytest.mark.parametrize("case", ["plain", "finished", "all_finished", "first", "masked", "dead", "equal", "short"])
def test_selection_against_all_candidates(case, penalty):
    args = _step()
    logits, scores, lengths, finished = args
    end = 4
    if case == "plain":
        end = -1
    elif case == "finished":
        finished[0, 1] = finished[1, 0] = finished[1, 2] = True
    elif case == "all_finished":
        finished[:] = True
        scores[0, 1] = -math.inf
    elif case == "first":
        scores[:] = 0
        scores[:, 1:] = -math.inf
        lengths.zero_()
    elif case == "masked":
        logits[0, :, 2:] = -math.inf
        logits[1, 0] = torch.finfo(torch.float32).min
        logits[1, 1, 3:] = torch.finfo(torch.float32).min
    elif case == "dead":
        logits[0, 0, 3] = math.nan
        logits[0, 1] = -math.inf
        logits[1, 0, 2] = math.inf
        scores[1, 1], scores[1, 2] = math.nan, math.inf
    elif case == "equal":
        logits[:] = 1.5
        scores[:] = -2.0
        lengths[:] = 3
    elif case == "short":
        args = (logits[..., :1], scores, lengths, finished)
        end = 0
    _check_step(args, end, penalty)


@pytest.mark.parametrize("score", [-1e14, -1e17, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("penalty", [0.0, 0.7])
def test_scores_that_swallow_logits_leave_their_order(score, penalty):
    logits, scores, lengths, finished = _step(V=40)
    scores[:, 1:] = -math.inf
    scores[:, 0] = score
    tokens, parents, new_scores, _, _ = beam_select(logits, scores, lengths, finished, length_penalty=penalty)
    assert (parents == 0).all() and torch.equal(new_scores, torch.full((2, 3), score))
    assert torch.equal(tokens, logits[:, 0].sort(dim=1, descending=True)[1][:, :3])


def test_selection_refuses():
    logits, scores, lengths, finished = _step()
    with pytest.raises(ValueError, match="expected logits"):
        beam_select(logits[0], scores, lengths, finished)
    with pytest.raises(ValueError, match="expected logits"):
        beam_select(logits[..., :0], scores, lengths, finished)
    with pytest.raises(ValueError, match="does not match"):
        beam_select(logits, scores[:, :2], lengths, finished)
    with pytest.raises(TypeError, match="lengths must be"):
        beam_select(logits, scores, lengths.long(), finished)
    with pytest.raises(TypeError, match="scores must be"):
        beam_select(logits, scores.double(), lengths, finished)
    with pytest.raises(ValueError, match="end_token"):
        beam_select(logits, scores, lengths, finished, end_token=11)
    with pytest.raises(ValueError, match="length_penalty"):
        beam_select(logits, scores, lengths, finished, length_penalty=math.nan)
    with pytest.raises(TypeError, match="floating point"):
        beam_select(logits.long(), scores, lengths, finished)


# ---------------------------------------------------------------- states
def test_states_follow_their_parents():
    states = [torch.randn(6, 5), torch.arange(12).view(6, 2), torch.randn(6, 0), torch.randn(6)]
    parents = torch.tensor([[1, 2, 0], [2, 2, 7]])
    expected = [state[[1, 2, 0, 5, 5, 5]] for state in states]
    reorder_states_(states, parents)
    for state, value in zip(states, expected):
        assert torch.equal(state, value)
    reorder_states_([], parents)


def test_states_refuse():
    parents = torch.zeros(2, 3, dtype=torch.int64)
    state = torch.randn(6, 4)
    with pytest.raises(ValueError, match="6 rows"):
        reorder_states_([state[:5]], parents)
    with pytest.raises(ValueError, match="contiguous"):
        reorder_states_([torch.randn(4, 6).t()], parents)
    with pytest.raises(ValueError, match="overlap"):
        reorder_states_([state, state], parents)
    with pytest.raises(ValueError, match="overlap"):
        reorder_states_([parents.view(-1)], parents)
    with pytest.raises(TypeError, match="int64"):
        reorder_states_([state], parents.int())
    with pytest.raises(ValueError, match="expected parents"):
        reorder_states_([state], parents.view(-1))


# ---------------------------------------------------------------- pages
def _cache(rows=4, pages=12, page=16, width=4, blocks=2, heads=1, dim=4):
    cache = PagedCache(blocks, heads, dim, rows, width * page, pages, page, dtype=torch.float64)
    cache.pool.copy_(torch.arange(cache.pool.numel(), dtype=torch.float64).view(cache.pool.shape))
    return cache


def _count(table, pages):
    return torch.bincount(table[table >= 0].long(), minlength=pages).int()


def test_a_cache_holds_what_lists_hold():
    """Random steps of a search: every row's tokens equal those of a plain list that is copied whole."""
    g = torch.Generator().manual_seed(3)
    cache = _cache(rows=6, pages=24, width=5)
    lists = [[] for _ in range(6)]
    for step in range(60):
        parents = torch.randint(0, 3, (2, 3), generator=g)
        live = torch.rand(6, generator=g) < 0.9
        tokens = int(torch.randint(0, 4, (1,), generator=g))
        if step % 20 == 19:
            live[:] = False
        cache.advance_(tokens, parents, live.view(2, 3))
        lists = [list(lists[r // 3 * 3 + parents.view(-1)[r]]) if live[r] else [] for r in range(6)]
        if any(len(entry) + tokens > 80 for entry in lists):
            with pytest.raises(RuntimeError, match="outgrew"):
                cache.check()
        else:
            cache.check()
        for row in range(6):
            if live[row] and len(lists[row]) + tokens <= 80:
                lists[row] += torch.randn(tokens, 2, 2, 1, 4, generator=g, dtype=torch.float64).unbind()
        assert cache.lengths.tolist() == [len(entry) for entry in lists]
        assert torch.equal(cache.refs, _count(cache.table, 24))
        for row in range(6):
            grown = [x for x in lists[row][max(len(lists[row]) - tokens, 0):]]
            for i, x in enumerate(grown):
                t = len(lists[row]) - len(grown) + i
                cache.pool[cache.table[row, t // 16], :, :, :, t % 16] = x
        if step % 7 == 6:
            used = cache.compact_()
            assert used == int((cache.refs > 0).sum()) and bool((cache.refs[:used] > 0).all())
        if step % 11 == 10:
            saved = cache.state_dict()
            cache = _cache(rows=6, pages=30, width=5)
            cache.load_state_dict(saved)
            cache.pool, cache.refs = cache.pool[:24].clone(), cache.refs[:24].clone()
        for row in range(6):
            for t, x in enumerate(lists[row]):
                assert torch.equal(cache.pool[cache.table[row, t // 16], :, :, :, t % 16], x)


def test_forking_copies_only_a_partly_filled_page():
    cache = _cache()
    cache.advance_(20, live=torch.tensor([True, False, False, False]))
    before = cache.pool.clone()
    parents = torch.zeros(1, 4, dtype=torch.int64)
    cache.advance_(0, parents)
    assert cache.refs[:2].tolist() == [4, 4] and torch.equal(cache.pool, before)
    cache.advance_(1)
    # rows 0 to 2 take pages 2 to 4 with the 4 tokens of page 1, the last row keeps page 1
    assert cache.table[:, :2].tolist() == [[0, 2], [0, 3], [0, 4], [0, 1]]
    assert torch.equal(cache.pool[2:5, ..., :4, :], before[1, ..., :4, :].expand(3, -1, -1, -1, -1, -1))
    assert torch.equal(cache.pool[2:5, ..., 4:, :], before[2:5, ..., 4:, :])
    cache.check()
    cache.free_(torch.tensor([False, True, True, True]))
    assert cache.refs[:5].tolist() == [1, 0, 1, 0, 0] and cache.lengths.tolist() == [21, 0, 0, 0]
    # a page that somebody outside the table holds is not written to either
    cache.refs[2] += 1
    cache.advance_(1)
    assert cache.table[0, 1] == 1 and cache.refs[:3].tolist() == [1, 1, 1]


def test_a_pool_that_runs_out_says_so():
    cache = _cache(rows=2, pages=3, width=2)
    cache.advance_(16)
    cache.advance_(3)
    with pytest.raises(RuntimeError, match="ran out"):
        cache.check()
    assert cache.table.tolist() == [[0, 2], [1, -1]] and cache.lengths.tolist() == [19, 19]
    cache.check()
    cache.advance_(20)
    with pytest.raises(RuntimeError, match="outgrew"):
        cache.check()
    assert cache.lengths.tolist() == [19, 19]
    cache.advance_(0, torch.tensor([[0, 5]]))
    with pytest.raises(RuntimeError, match="outside its group"):
        cache.check()
    # the missing page's tokens are stored nowhere and not seen
    store_pages(cache.pool, 1, cache.table, cache.lengths, torch.ones(2, 3, 1, 4).double(), torch.ones(2, 3, 1, 4).double())
    q = torch.randn(2, 2, 4, dtype=torch.float64)
    cut = cache.lengths.clone()
    cut[1] = 16
    assert torch.equal(cache.attend(1, q), paged_attention(q, cache.pool, 1, cache.table, cut))


def test_attention_and_append_against_formulas():
    g = torch.Generator().manual_seed(1)
    cache = _cache(rows=3, pages=9, width=3, heads=2, dim=8)
    cache.pool.normal_(generator=g)
    cache.table.copy_(torch.tensor([[5, 2, -1], [0, 7, 8], [3, -1, -1]]))
    cache.lengths.copy_(torch.tensor([21, 48, 0]))
    x = torch.randn(3, (2 * 6 + 4) * 8, generator=g, dtype=torch.float64)
    wq, wk = torch.randn(8, generator=g).double(), torch.randn(8, generator=g).double()
    freq = torch.tensor([1.0, 0.25])
    before = cache.pool.clone()
    q = cache.append_(1, x, wq, wk, freq, 6, 1e-6)

    def turned(y, w, position):
        y = y * (y.square().mean() + 1e-6).rsqrt() * (1 + w)
        out = y.clone()
        for i, f in enumerate(freq.tolist()):
            c, s = math.cos(position * f), math.sin(position * f)
            out[i], out[i + 2] = y[i] * c - y[i + 2] * s, y[i + 2] * c + y[i] * s
        return out

    for row, (page, slot) in enumerate([(2, 4), (8, 15), (None, None)]):
        position = max(int(cache.lengths[row]) - 1, 0)
        for h in range(6):
            torch.testing.assert_close(q[row, h], turned(x[row, 16 * h:16 * h + 8], wq, position), rtol=1e-12, atol=1e-12)
        for h in range(2):
            if page is None:
                continue
            key = x[row, 96 + 8 * h:104 + 8 * h]
            torch.testing.assert_close(cache.pool[page, 1, 0, h, slot], turned(key, wk, position), rtol=1e-12, atol=1e-12)
            assert torch.equal(cache.pool[page, 1, 1, h, slot], x[row, 112 + 8 * h:120 + 8 * h])
    changed = (cache.pool != before).any(-1).nonzero().tolist()
    assert sorted(changed) == sorted([p, 1, kind, h, s] for p, s in ((2, 4), (8, 15)) for kind in (0, 1) for h in (0, 1))
    gate = torch.randn(3, 6, 8, generator=g, dtype=torch.float64)
    out = cache.attend(1, q, gate, group=3)
    for row, pages in enumerate([[5, 2], [0, 7, 8], []]):
        if not pages:
            assert not out[row].any()
            continue
        n = int(cache.lengths[row])
        for h in range(6):
            k, v = (torch.cat([cache.pool[p, 1, kind, h // 3] for p in pages])[:n] for kind in (0, 1))
            p = torch.softmax(k @ q[row, h] / 8 ** 0.5, 0)
            torch.testing.assert_close(out[row, h], (p @ v) * torch.sigmoid(gate[row, h]), rtol=1e-12, atol=1e-12)


def test_pages_refuse():
    cache = _cache()
    pool, table, lengths, refs = cache.pool, cache.table, cache.lengths, cache.refs
    with pytest.raises(ValueError, match="expected a pool"):
        advance_pages(pool[0], table, lengths, refs)
    with pytest.raises(ValueError, match="page holds"):
        PagedCache(1, 1, 4, 1, 8, 1, page=8)
    with pytest.raises(ValueError, match="at least one"):
        PagedCache(1, 1, 4, 0, 8, 1)
    with pytest.raises(ValueError, match="contiguous"):
        advance_pages(pool[..., ::2], table, lengths, refs)
    with pytest.raises(TypeError, match="table must be"):
        advance_pages(pool, table.long(), lengths, refs)
    with pytest.raises(ValueError, match="lengths"):
        advance_pages(pool, table, lengths[:2], refs)
    with pytest.raises(ValueError, match="refs"):
        compact_pages(pool, table, refs[:5].clone())
    with pytest.raises(ValueError, match="tokens must"):
        advance_pages(pool, table, lengths, refs, tokens=-1)
    with pytest.raises(ValueError, match="expected parents"):
        advance_pages(pool, table, lengths, refs, parents=torch.zeros(1, 3, dtype=torch.int64))
    with pytest.raises(ValueError, match="live must be"):
        advance_pages(pool, table, lengths, refs, live=torch.ones(4))
    status = torch.zeros(1, dtype=torch.int32)
    both = torch.zeros(table.numel() + 1, dtype=torch.int32)
    for out in ((both[1:].view(table.shape), lengths, refs, status), (table, lengths, refs, refs[:1])):
        with pytest.raises(ValueError, match="apart"):
            advance_pages(pool, both[:-1].view(table.shape), lengths, refs, out=out)
    with pytest.raises(ValueError, match="apart"):
        compact_pages(pool, both[:-1].view(table.shape), refs, out=(both[1:].view(table.shape), refs))
    q = torch.randn(4, 2, 4, dtype=torch.float64)
    with pytest.raises(IndexError, match="block 2"):
        paged_attention(q, pool, 2, table, lengths)
    with pytest.raises(ValueError, match="expected q"):
        paged_attention(q[0], pool, 0, table, lengths)
    with pytest.raises(ValueError, match="gate"):
        paged_attention(q, pool, 0, table, lengths, gate=q[:, :1])
    with pytest.raises(ValueError, match="groups of 3"):
        paged_attention(q, pool, 0, table, lengths, group=3)
    with pytest.raises(ValueError, match="query heads"):
        append_heads(q.view(4, 8), pool, 0, table, lengths, q[0, 0], q[0, 0], q[0, 0, :1], 0, 1e-6)
    with pytest.raises(ValueError, match="x .*does not match"):
        append_heads(q.view(4, 8), pool, 0, table, lengths, q[0, 0], q[0, 0], q[0, 0, :1], 2, 1e-6)
    with pytest.raises(ValueError, match="frequencies"):
        append_heads(torch.randn(4, 24).double(), pool, 0, table, lengths, q[0, 0], q[0, 0], torch.ones(3), 2, 1e-6)
    with pytest.raises(ValueError, match="expected keys"):
        store_pages(pool, 0, table, lengths, torch.zeros(3, 1, 1, 4), torch.zeros(3, 1, 1, 4))
    with pytest.raises(ValueError, match="do not fit"):
        cache.load_state_dict(dict(cache.state_dict(), table=table[:, :2]))


# ---------------------------------------------------------------- searches
def _sharp(replaced=()):
    model = tiny_model()
    with torch.no_grad():
        model.lm_head.weight.mul_(200)  # logits that differ by more than bf16 rounds
    for layer in replaced:
        install(model, layer, {"head_size": 8, "backend": "reference"})
        with torch.no_grad():  # it starts at zero: the block would add nothing
            model.model.layers[layer].self_attn.core.output.weight.normal_(0, 0.2)
    return model


def _fresh(model):
    runner = Runner(model)
    runner.reset()
    return runner


@pytest.mark.parametrize("replaced", [(), (1,), (1, 3)])
def test_one_beam_is_greedy(replaced):
    runner = Runner(_sharp(replaced))
    prompt = torch.randint(0, 64, (2, 21))
    ids, scores, lengths = beam_search(runner, prompt, 9, beams=1, page=16)
    assert torch.equal(ids[:, 0], generate(runner, prompt, 9))
    assert (scores < 0).all() and (lengths == 9).all()


@pytest.mark.parametrize("replaced", [(), (1, 3)])
def test_scores_are_those_of_a_single_pass(replaced):
    model = _sharp(replaced)
    prompt = torch.randint(0, 64, (2, 21))
    runner = Runner(model)
    live = runner.forward(prompt[:1, :5])
    cursor = runner.cache.cursor
    ids, scores, _ = beam_search(runner, prompt, 6, beams=4, page=16, prefill_chunk=8)
    assert runner.cache.cursor == cursor and live.shape[1] == 5  # the runner's own state is untouched
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    for g in range(2):
        assert len({tuple(row) for row in ids[g].tolist()}) == 4
        for k in range(4):
            hidden = _fresh(model).forward(torch.cat([prompt[g], ids[g, k]])[None])
            logits = (hidden.to(model.lm_head.weight.dtype) @ model.lm_head.weight.t())[0].float()
            single = torch.log_softmax(logits, -1)[20:26].gather(1, ids[g, k, :, None]).sum()
            # bf16 activations of two schedules: six tokens' logits of magnitude 16 to 32, each off by a few bf16 steps
            assert abs(single - scores[g, k]) < 6 * 0.125 * 2


def test_a_wide_search_finds_the_best_pair_of_tokens():
    """With as many beams as tokens, two steps see every pair: the best ones must come out."""
    model = _sharp((1, 3))
    prompt = torch.randint(0, 64, (1, 5))
    ids, scores, _ = beam_search(Runner(model), prompt, 2, beams=64)
    runner = _fresh(model)
    head = model.lm_head.weight
    first = torch.log_softmax((runner.forward(prompt)[:, -1].to(head.dtype) @ head.t()).float(), -1)[0]
    runner = _fresh(model)
    hidden = runner.forward(torch.cat([prompt.expand(64, -1), torch.arange(64)[:, None]], 1))
    pairs = first[:, None] + torch.log_softmax((hidden[:, -1].to(head.dtype) @ head.t()).float(), -1)
    best = pairs.flatten().topk(64)[0]
    assert (best - scores[0]).abs().max() < 2 * 0.125 * 2  # as above, two tokens


def test_ended_beams_stay_and_cost_nothing():
    model = _sharp()
    runner = Runner(model)
    prompt = torch.randint(0, 64, (2, 7))
    free, _, _ = beam_search(runner, prompt, 24, beams=3, page=16)
    end = int(free[0, 0, 3])
    ids, scores, lengths = beam_search(runner, prompt, 24, beams=3, end_token=end, length_penalty=0.6, page=16)
    rank = scores.double() / lengths.double() ** 0.6
    assert (rank[:, :-1] >= rank[:, 1:]).all()
    for row, length in zip(ids.view(6, 24).tolist(), lengths.view(-1).tolist()):
        assert end not in row[:length - 1] and all(token == end for token in row[length:])
        assert length == 24 or row[length - 1] == end
    assert (lengths < 24).any()


def test_search_refuses():
    runner = Runner(tiny_model())
    with pytest.raises(ValueError, match="expected prompts"):
        beam_search(runner, torch.zeros(0, 3, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="at least one beam"):
        beam_search(runner, torch.zeros(1, 3, dtype=torch.int64), 0)
    with pytest.raises(ValueError, match="page holds"):
        beam_search(runner, torch.zeros(1, 3, dtype=torch.int64), 4, page=5)


def test_search_refuses_chunks_and_graphs_that_cannot_be():
    runner = Runner(tiny_model())
    with pytest.raises(ValueError, match="prefill chunk"):
        beam_search(runner, torch.zeros(1, 3, dtype=torch.int64), 4, prefill_chunk=-1)
    with pytest.raises(ValueError, match="graph steps need CUDA"):
        beam_search(runner, torch.zeros(1, 3, dtype=torch.int64), 4, graph=True)
