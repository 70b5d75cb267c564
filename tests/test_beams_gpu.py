"""Kernels of beam search against the plain definitions in 64 bits, at the sizes and masks where they can go wrong, and
whole searches on the GPU."""
import math

import pytest
import torch

from rwkv_theseus_b200.beams import beam_search, beam_select, reorder_states_
from rwkv_theseus_b200.inference import generate
from rwkv_theseus_b200.models.hf_io import random_model
from rwkv_theseus_b200.models.qwen35 import HybridConfig
from rwkv_theseus_b200.models.runner import Runner, install
from rwkv_theseus_b200.ops import reference
from rwkv_theseus_b200.paged import (PagedCache, advance_pages, append_heads, compact_pages, paged_attention,
                                     store_pages)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA unavailable")]
INF, LOWEST = math.inf, torch.finfo(torch.float32).min


# ---------------------------------------------------------------- selection
def _step(G, K, V, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(G, K, V, device="cuda", generator=g) * 3
    scores = -torch.rand(G, K, device="cuda", generator=g) * 9
    lengths = torch.randint(1, 9, (G, K), device="cuda", generator=g).int()
    finished = torch.rand(G, K, device="cuda", generator=g) < 0.2
    return [logits.to(dtype), scores, lengths, finished]


def _check(args, end=-1, penalty=0.0):
    got = beam_select(*args, end_token=end, length_penalty=penalty)
    want = reference.beam_select(*(x.cpu() for x in args), end, penalty)
    for name, g, w in zip(("tokens", "parents", "scores", "lengths", "finished"), got, want):
        g = g.cpu()
        assert g.dtype == w.dtype and g.shape == w.shape
        if name == "scores":
            assert torch.equal(g.isinf(), w.isinf())
            # a sum of exponentials with terms off by 2^-22 at most (its logarithm by as much), then one rounding
            torch.testing.assert_close(g, w, rtol=2 ** -23, atol=2 ** -21)
        else:
            assert torch.equal(g, w), (name, g, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,K,V", [(1, 1, 1), (1, 2, 1), (3, 4, 2), (2, 3, 17), (1, 4, 4096), (1, 32, 33), (2, 5, 16321),
                                   (1, 1, 248077), (1, 3, 50001), (5, 32, 999), (40, 8, 1003), (1, 1, 600001)])
def test_selection(G, K, V, dtype):
    args = _step(G, K, V, dtype)
    # bf16 logits of different beams differ by more than the exponentials' error unless they are equal; so do these
    _check(args)
    _check(args, end=V // 2, penalty=0.6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [3, 700, 40003])
def test_selection_corners(V, dtype):
    G, K = 4, 5
    logits, scores, lengths, finished = _step(G, K, V, dtype, seed=1)
    finished.zero_()
    logits[0] = 2.5                               # one row of equal logits after the other
    scores[0] = -1.0
    logits[1, 0], logits[1, 1] = -INF, LOWEST     # nothing; everything at a mask's value
    logits[1, 2, V // 2:] = -INF
    logits[1, 3, 1:] = LOWEST
    logits[2, 0, V - 1], logits[2, 1, 0], logits[2, 2, 0] = math.nan, INF, -INF
    logits[2, 3, :] = torch.arange(V, device="cuda") // 2 * 0.5 - 40
    scores[3, 0], scores[3, 1], scores[3, 2] = math.nan, INF, -INF
    finished[3, 2:4] = True
    for end in (-1, 0, V - 1):
        _check([logits, scores, lengths, finished], end, 0.5)
    scores[:] = 0
    scores[:, 1:] = -INF
    _check([logits, scores, lengths, finished], 1)
    finished[:] = True
    _check([logits, scores, lengths, finished], 1)
    _check([logits, scores, lengths, finished], -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("at", [0, 20003, 29999, 40002])
def test_a_nan_among_masked_logits_leaves_the_beam_nothing(at, dtype):
    logits, scores, lengths, finished = _step(2, 3, 40003, dtype, seed=2)
    logits[0, 1] = -INF  # but for a few, far from the NaN
    logits[0, 1, 10000:10010] = 1.0
    logits[0, 1, at] = math.nan
    logits[1] = -INF
    logits[1, 0, 10000:10010] = 1.0
    logits[1, 2, at] = math.nan
    finished.zero_()
    _check([logits, scores, lengths, finished])


@pytest.mark.parametrize("score", [-1e9, -1e14, -1e17, LOWEST])
@pytest.mark.parametrize("G,K,V", [(2, 3, 40), (1, 4, 4096), (3, 32, 20011), (2, 5, 70001)])
def test_scores_that_swallow_logits_leave_their_order(G, K, V, score):
    logits, scores, lengths, finished = _step(G, K, V, torch.float32, seed=3)
    finished.zero_()
    scores[:] = -INF
    scores[:, K // 2] = score
    for penalty in (0.0, 0.7, -1.3):
        _check([logits, scores, lengths, finished], 1, penalty)
        _check([logits.bfloat16(), scores, lengths, finished], 1, penalty)  # (many equal logits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_largest_vocabulary_and_most_beams(dtype):
    V, g = 4161536, torch.Generator(device="cuda").manual_seed(4)
    row = (torch.randperm(V, device="cuda", generator=g).float() * 2 ** -18).to(dtype)  # (bf16: many are equal)
    scores = torch.full((1, 32), -INF, device="cuda")
    scores[0, 5] = -1.0
    tokens, parents, new, lengths, ended = beam_select(
        row.expand(1, 32, V), scores, torch.ones(1, 32, device="cuda", dtype=torch.int32),
        torch.zeros(1, 32, device="cuda", dtype=torch.bool))
    want = row.sort(descending=True, stable=True)[1][:32]
    order = [want[1:6], want[:1], want[6:]]  # slot 5 keeps its best child, the others fill the rest in order
    assert torch.equal(tokens[0], torch.cat(order)) and (parents == 5).all() and (lengths == 2).all()
    value = -1.0 + torch.log_softmax(row.double(), -1)[tokens[0]]
    torch.testing.assert_close(new[0], value.float(), rtol=2 ** -23, atol=2 ** -21)


def test_selection_takes_any_strides():
    logits, scores, lengths, finished = _step(3, 4, 1001, torch.float32)
    wide = torch.empty(4, 3, 2005, device="cuda")
    view = wide[:, :, 3:1004].transpose(0, 1)
    view.copy_(logits)
    _check([view, scores, lengths, finished])
    _check([logits[:, :1].expand(3, 4, 1001), scores, lengths, finished])
    _check([logits.transpose(1, 2).contiguous().transpose(1, 2), scores.t().contiguous().t(), lengths, finished])


def test_selection_refuses_on_cuda():
    logits, scores, lengths, finished = _step(1, 33, 40, torch.float32)
    with pytest.raises(ValueError, match="at most 32 beams"):
        beam_select(logits, scores, lengths, finished)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        beam_select(logits[:, :2].half(), scores[:, :2], lengths[:, :2], finished[:, :2])
    with pytest.raises(ValueError, match="different devices"):
        beam_select(logits[:, :2], scores[:, :2].cpu(), lengths[:, :2], finished[:, :2])
    logits, scores, lengths, finished = _step(2, 3, 40, torch.float32)
    for error, match, args, more in (
            (ValueError, "expected logits", (logits[0], scores, lengths, finished), {}),
            (ValueError, "expected logits", (logits[..., :0], scores, lengths, finished), {}),
            (ValueError, "does not match", (logits, scores[:, :2], lengths, finished), {}),
            (TypeError, "lengths must be", (logits, scores, lengths.long(), finished), {}),
            (TypeError, "scores must be", (logits, scores.double(), lengths, finished), {}),
            (ValueError, "end_token", (logits, scores, lengths, finished), dict(end_token=40)),
            (ValueError, "length_penalty", (logits, scores, lengths, finished), dict(length_penalty=math.nan))):
        with pytest.raises(error, match=match):
            beam_select(*args, **more)


# ---------------------------------------------------------------- states
@pytest.mark.parametrize("G,K", [(1, 2), (3, 4), (2, 7), (1, 16), (2, 32), (5, 1), (70000, 2)])
def test_states_follow_any_parents(G, K):
    g = torch.Generator(device="cuda").manual_seed(G + K)
    rows = G * K
    shapes = [(3,), (5, 7), (), (1024,), (16, 64, 3), (4099,)] if rows < 1000 else [(3,), (4,)]
    dtypes = [torch.float32, torch.bfloat16, torch.int64, torch.uint8, torch.float32, torch.bool]
    states = [(torch.rand(rows, *shape, device="cuda", generator=g) * 200).to(dtype)
              for shape, dtype in zip(shapes, dtypes)]
    states.append(torch.empty(rows, 0, device="cuda"))
    if rows < 1000:
        states += [torch.randn(rows, 9, device="cuda", generator=g) for _ in range(150)]  # more than one launch holds
        states.append(torch.randn(rows * 24 + 1, device="cuda", generator=g)[1:].view(rows, 24))  # 4-byte alignment
    for parents in (torch.randint(0, K, (G, K), device="cuda", generator=g),
                    torch.arange(K - 1, -1, -1, device="cuda").expand(G, K),   # pairs change places
                    (torch.arange(K, device="cuda") + 1).expand(G, K) % K,     # a cycle
                    torch.arange(K, device="cuda").expand(G, K),
                    torch.full((G, K), K - 1, device="cuda"),
                    torch.randint(-2, K + 2, (G, K), device="cuda", generator=g)):
        source = reference.parent_rows(parents)
        expected = [state[source] for state in states]
        reorder_states_(states, parents)
        for state, value in zip(states, expected):
            assert torch.equal(state, value)


@pytest.mark.parametrize("K", [2, 3, 6, 18, 32])
@pytest.mark.parametrize("sources", [1, 2, 31])
def test_long_rows_follow_few_and_many_parents(K, sources):
    """Rows of several blocks, whose ends fall inside a thread's columns; words of 16, 4 and 1 bytes."""
    G, g = 200, torch.Generator().manual_seed(K)
    parents = torch.arange(K).repeat(G, 1)
    for group in parents:
        order = torch.randperm(K, generator=g)
        kept = order[:min(sources, K - 1)]
        moved = order[len(kept):]
        group[moved] = kept[torch.randint(len(kept), (len(moved),), generator=g)]
    parents[1] = parents[1].roll(1)  # one that takes over in a cycle
    rows = (parents + torch.arange(G)[:, None] * K).view(-1).cuda()
    for size in (131120, 70004, 20001):
        state = torch.randint(256, (G * K, size), device="cuda", dtype=torch.uint8)
        want = state[rows]
        reorder_states_([state], parents.cuda())
        assert torch.equal(state, want)


def test_states_refuse_on_cuda():
    parents = torch.zeros(1, 33, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="at most 32"):
        reorder_states_([torch.zeros(33, 2, device="cuda")], parents)
    with pytest.raises(ValueError, match="different devices"):
        reorder_states_([torch.zeros(33, 2)], parents)
    two, state = parents[:, :2].contiguous(), torch.zeros(2, 4, device="cuda")
    for error, match, states, by in ((ValueError, "2 rows", [state[:1]], two), (TypeError, "int64", [state], two.int()),
                                     (ValueError, "contiguous", [torch.zeros(4, 2, device="cuda").t()], two),
                                     (ValueError, "overlap", [state, state[1:].expand(2, 4).contiguous(), state], two),
                                     (ValueError, "overlap", [two.view(-1)], two),
                                     (ValueError, "expected parents", [state], two.view(-1))):
        with pytest.raises(error, match=match):
            reorder_states_(states, by)


# ---------------------------------------------------------------- pages
def _same(cuda, cpu):
    for a, b in zip(cuda, cpu):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("G,K,width,pages,page", [(1, 1, 3, 5, 16), (2, 3, 5, 24, 16), (7, 9, 6, 120, 32),
                                                  (16, 64, 3, 2500, 16), (1, 1000, 2, 3000, 64)])
def test_pages_advance_like_the_definition(G, K, width, pages, page):
    g = torch.Generator().manual_seed(G * K + page)
    rows = G * K
    pool = torch.randn(pages, 2, 2, 1, page, 64, generator=g).to(torch.bfloat16)
    state = [pool, torch.full((rows, width), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32),
             torch.zeros(pages, dtype=torch.int32)]
    state[3][pages // 2] = 1  # somebody else's
    device = [x.cuda() for x in state]
    for step in range(14):
        parents = torch.randint(0, K, (G, K), generator=g) if step % 3 else None
        if step == 8:
            parents = torch.randint(-1, K + 1, (G, K), generator=g)
        live = torch.rand(G, K, generator=g) < (0.9 if step % 5 else 0.3) if step % 2 else None
        tokens = [0, 1, 1, page // 2, 3][step % 5]
        want = reference.advance_pages(*state, tokens, parents, live)
        args = dict(tokens=tokens, parents=None if parents is None else parents.cuda(),
                    live=None if live is None else live.cuda())
        before = device[0].clone()
        got = advance_pages(*device, **args)
        _same(got, want)
        assert torch.equal(device[0].cpu(), state[0])
        # the same once more, in place: the arguments' pool has the copies already and gets them again
        device[0].copy_(before)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        advance_pages(*device, **args, out=(*device[1:], status))
        _same((*device[1:], status, device[0]), (*want, state[0]))
        state[1:] = want[:3]
        if step % 4 == 3:
            device[1], device[3], _ = compact_pages(device[0], device[1], device[3])
            state[1], state[3], _ = reference.compact_pages(state[0], state[1], state[3])
            _same(device, state)


def test_missing_pages_are_nobodys():
    """Entries outside the pool, lengths beyond the table, a pool without a free page."""
    cache = PagedCache(1, 1, 64, 3, 64, 4, 16, "cuda")
    cache.pool.normal_()
    cache.table.copy_(torch.tensor([[0, 9, -7, -1], [-1, 1, 3, -1], [2, -1, -1, -1]]))
    cache.lengths.copy_(torch.tensor([40, 1000, 5]))
    cache.refs.fill_(1)
    state = [x.cpu() for x in (cache.pool, cache.table, cache.lengths, cache.refs)]
    q = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    k = torch.randn(3, 50, 1, 64, device="cuda").to(torch.bfloat16)
    store_pages(cache.pool, 0, cache.table, cache.lengths, k, k)
    reference.store_pages(state[0], 0, state[1], state[2], k.cpu(), k.cpu())
    assert torch.equal(cache.pool.cpu(), state[0])
    x = torch.randn(3, 6 * 64, device="cuda").to(torch.bfloat16)
    w, f = torch.zeros(64, device="cuda"), torch.ones(3, device="cuda")
    append_heads(x, cache.pool, 0, cache.table, cache.lengths, w, w, f, 2, 1e-6)
    out = paged_attention(q, cache.pool, 0, cache.table, cache.lengths)
    want = reference.paged_attention(q.cpu().double(), cache.pool.cpu().double(), 0, state[1], state[2], None)
    torch.testing.assert_close(out.cpu().double(), want, rtol=2 ** -7, atol=2 ** -6)  # see _check_attention
    for tokens in (0, 1, 30):
        state[0] = cache.pool.cpu()
        got = advance_pages(cache.pool, cache.table, cache.lengths, cache.refs, tokens)
        _same((*got, cache.pool), (*reference.advance_pages(*state, tokens, None, None), state[0]))


@pytest.mark.parametrize("pages", [1, 31, 1024, 5000])
def test_compaction(pages):
    g = torch.Generator().manual_seed(pages)
    pool = torch.randn(pages, 1, 2, 1, 16, 64, generator=g).to(torch.bfloat16)
    for share in (0.0, 0.3, 0.95, 1.0):
        refs = (torch.rand(pages, generator=g) < share).int() * torch.randint(1, 4, (pages,), generator=g).int()
        table = torch.randint(-2, pages + 2, (7, 11), generator=g).int()
        device = pool.cuda()
        got = compact_pages(device, table.cuda(), refs.cuda())
        mine = pool.clone()
        want = reference.compact_pages(mine, table, refs)
        used = int(want[2])
        _same(got, want)
        assert torch.equal(device[:used].cpu(), mine[:used])
        again = [table.cuda(), refs.cuda()]
        device = pool.cuda()
        compact_pages(device, *again, out=tuple(again))
        _same(again, want[:2])
        assert torch.equal(device.cpu(), mine)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,Hq", [(1, 1), (2, 6), (3, 36)])
@pytest.mark.parametrize("rotated", [0, 2, 16, 26, 64])
def test_append(D, H, Hq, rotated):
    g = torch.Generator(device="cuda").manual_seed(D + Hq)
    cache = PagedCache(2, H, D, 5, 70, 20, 32, "cuda")
    cache.pool.normal_(generator=g)
    cache.table.copy_(torch.tensor([[0, 1, -1], [2, 3, 19], [4, -1, -1], [5, 6, 7], [-1, -1, -1]]))
    cache.lengths.copy_(torch.tensor([33, 70, 1, 64, 0]))
    wide = torch.randn(5, (2 * Hq + 2 * H) * D + 8, device="cuda", generator=g).to(torch.bfloat16)
    x = wide[:, 3:-5]  # any row stride and alignment
    wq, wk = (torch.randn(D, device="cuda", generator=g) * 0.2 for _ in range(2))
    freq = 1.0 / 1e4 ** (torch.arange(rotated // 2, device="cuda") / max(rotated, 1))
    before = cache.pool.cpu()
    q = append_heads(x, cache.pool, 1, cache.table, cache.lengths, wq, wk, freq, Hq, 1e-6)
    pool = before.double()
    want = reference.append_heads(x.cpu().double(), pool, 1, cache.table.cpu(), cache.lengths.cpu(), wq.cpu(), wk.cpu(),
                                  freq.cpu(), Hq, 1e-6)
    # one rounding to bf16 of values with some 2^-20 of fp32 error, relative to the pair that is rotated (below 8)
    torch.testing.assert_close(q.cpu().double(), want, rtol=2 ** -8, atol=2 ** -16)
    torch.testing.assert_close(cache.pool.cpu().double(), pool, rtol=2 ** -8, atol=2 ** -16)
    assert torch.equal(cache.pool[:, 0].cpu(), before[:, 0])
    assert torch.equal(cache.pool[:, 1, 1].cpu().double(), pool[:, 1, 1])


def test_far_positions_keep_their_angle():
    table = torch.zeros(1, 1 << 18, dtype=torch.int32, device="cuda")
    pool = torch.zeros(1, 1, 2, 1, 64, 64, device="cuda", dtype=torch.bfloat16)
    lengths = torch.tensor([(1 << 24) - 5], dtype=torch.int32, device="cuda")
    x = torch.randn(1, 4 * 64, device="cuda").to(torch.bfloat16)
    w, freq = torch.zeros(64, device="cuda"), torch.tensor([1.0, 0.7371], device="cuda")
    q = append_heads(x, pool, 0, table, lengths, w, w, freq, 1, 1e-6)
    want = reference.append_heads(x.cpu().double(), pool.cpu().double(), 0, table.cpu(), lengths.cpu(), w.cpu(), w.cpu(),
                                  freq.cpu(), 1, 1e-6)
    torch.testing.assert_close(q.cpu().double(), want, rtol=2 ** -8, atol=2 ** -16)  # as above


@pytest.mark.parametrize("page", [16, 64])
def test_store(page):
    g = torch.Generator().manual_seed(page)
    cache = PagedCache(3, 2, 64, 6, 3 * page, 30, page, "cuda")
    cache.pool.normal_()
    cache.table.copy_(torch.randperm(30, generator=g)[:18].view(6, 3))
    cache.lengths.copy_(torch.tensor([2 * page + 3, 1, 3 * page, 0, 5, 2 * page]))
    state = [x.cpu() for x in (cache.pool, cache.table, cache.lengths)]
    for N, T in ((6, 1), (6, page + 2), (3, 3 * page), (2, 0), (1, 4)):
        k = torch.randn(2, N, T + 3, 2, 64, generator=g).to(torch.bfloat16)[:, :, 1:T + 1]
        strided = k[1].cuda().transpose(1, 2).contiguous().transpose(1, 2)
        store_pages(cache.pool, 1, cache.table, cache.lengths, k[0].cuda(), strided)
        reference.store_pages(state[0], 1, *state[1:], k[0], k[1])
        assert torch.equal(cache.pool.cpu(), state[0])


# ---------------------------------------------------------------- attention
def _attention(groups, K, H, Hq, D, page, prompt, new, seed=0, blocks=2):
    """A cache in which each group's beams share their prompt's whole pages."""
    g = torch.Generator().manual_seed(seed)
    rows, width = groups * K, -(-(prompt + new) // page) + 1
    lists, used = [], 0
    for group in range(groups):
        length = max(0, prompt - 7 * group)
        shared = list(range(used, used + length // page))
        used += len(shared)
        for k in range(K):
            own = -(-(length + max(new - k, 0)) // page) - len(shared)
            lists.append((length + max(new - k, 0), shared + list(range(used, used + own))))
            used += own
    pages = used + 3
    place = torch.randperm(pages, generator=g)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    for row, (_, entry) in enumerate(lists):
        table[row, :len(entry)] = place[torch.tensor(entry, dtype=torch.int64)]
    pool = torch.randn(pages, blocks, 2, H, page, D, generator=g).to(torch.bfloat16)
    q = (torch.randn(rows, Hq, D, generator=g) * 2).to(torch.bfloat16)
    gate = torch.randn(rows, Hq, 2 * D, generator=g).to(torch.bfloat16)[..., D:]
    return q, pool, table, torch.tensor([n for n, _ in lists], dtype=torch.int32), gate


def _check_attention(q, pool, table, lengths, gate, group, block=1):
    device = [None if x is None else x.cuda() for x in (q, pool, table, lengths, gate)]
    if gate is not None:
        device[4] = torch.cat([device[4], device[4]], -1)[..., :q.shape[2]]  # strided
    got = paged_attention(device[0], device[1], block, device[2], device[3], device[4], group).cpu().double()
    want = reference.paged_attention(q.double(), pool.double(), block, table, lengths,
                                     None if gate is None else gate.double())
    # Weights are rounded to bf16 before they meet the values (2^-8 of the mean of |v| at most), the result once more
    # (2^-8 of it); scores are fp32 sums of exact products, off by some 2^-19 of sum |q k|, below 2^8 here: 2^-11.
    size = reference.paged_attention(q.double(), pool.double().abs().where(torch.tensor([0, 1]).view(1, 1, 2, 1, 1, 1) == 1,
                                                                           pool.double()), block, table, lengths, None)
    bound = 2 ** -8 * want.abs() + (2 ** -8 + 2 ** -11) * size + 1e-30
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()
    return got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("groups,K,H,Hq,prompt,new", [(1, 1, 1, 1, 0, 1), (2, 3, 1, 6, 40, 5), (1, 8, 2, 12, 700, 70),
                                                      (3, 5, 2, 2, 130, 3), (1, 9, 1, 13, 65, 9), (1, 17, 1, 64, 20, 30),
                                                      (2, 32, 1, 8, 129, 33)])
def test_attention(groups, K, H, Hq, prompt, new, page, D):
    args = _attention(groups, K, H, Hq, D, page, prompt, new)
    shared = _check_attention(*args, group=K)
    alone = _check_attention(*args[:4], None, group=1)
    assert alone.shape == shared.shape


def test_attention_of_a_long_cache():
    args = _attention(1, 4, 2, 8, 128, 64, 33333, 100, blocks=1)
    _check_attention(*args, group=4, block=0)


def test_what_a_mask_hides_stays_hidden():
    """NaN and infinities behind a row's last token, in free pages and in other rows' pages; empty rows."""
    q, pool, table, lengths, gate = _attention(2, 4, 2, 12, 128, 32, 70, 9)
    lengths[3] = 0
    lengths[5] = 33
    table[5, 2:] = -1
    clean = [q, pool, table, lengths, gate]
    held = torch.zeros(pool.shape[0], 32, dtype=torch.bool)
    for row in range(8):
        for t in range(int(lengths[row])):
            held[table[row, t // 32], t % 32] = True
    dirty = pool.clone().permute(0, 4, 1, 2, 3, 5).contiguous()
    for value in (math.nan, INF, -INF):
        dirty[~held] = value
        again = dirty.permute(0, 2, 3, 4, 1, 5).contiguous()
        for group in (1, 4, 8):
            a = paged_attention(*(x.cuda() for x in (q, again)), 1, table.cuda(), lengths.cuda(), gate.cuda(), group)
            b = paged_attention(*(x.cuda() for x in (q, pool)), 1, table.cuda(), lengths.cuda(), gate.cuda(), group)
            assert torch.equal(a, b) and not a[3].any()
    _check_attention(*clean, group=4)
    # rows of one group that end at different tokens of a shared page, one of them before its NaN
    table[1] = table[0]
    lengths[0], lengths[1] = 40, 39
    pool[table[0, 1], 1, :, :, 39 - 32] = math.nan
    out = paged_attention(q.cuda(), pool.cuda(), 1, table.cuda(), lengths.cuda(), gate.cuda(), 4)
    seeing = [0, 2]  # row 2 shares the prompt's pages and goes on behind it
    assert out[seeing].isnan().all() and out[[1, 3, 4, 5, 6, 7]].isfinite().all()
    # a row's own NaN query stays its own
    q[6] = math.nan
    out = paged_attention(q.cuda(), pool.cuda(), 1, table.cuda(), lengths.cuda(), gate.cuda(), 4)
    assert out[6].isnan().all() and out[[1, 4, 5, 7]].isfinite().all()


def test_scores_of_any_size():
    q, pool, table, lengths, _ = _attention(1, 2, 1, 4, 64, 16, 100, 4)
    q[0, 0] *= 1e3
    q[0, 1] *= 1e-6
    pool[:, :, 0] *= 30
    _check_attention(q, pool, table, lengths, None, group=2)


def test_a_cache_with_too_many_rows_and_blocks_is_left_alone():
    pool = torch.empty(1, 2 ** 18, 2, 1, 16, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.full((1024, 1), -1, device="cuda", dtype=torch.int32)
    lengths, refs = torch.zeros(1024, device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
    with pytest.raises(ValueError, match="out of range"):
        advance_pages(pool, table, lengths, refs, out=(table, lengths, refs, torch.zeros_like(refs)))
    assert (table == -1).all() and (lengths == 0).all() and (refs == 0).all()


def test_pages_refuse_on_cuda():
    cache = PagedCache(1, 1, 64, 2, 64, 4, 16, "cuda")
    with pytest.raises(TypeError, match="bf16 and head sizes"):
        PagedCache(1, 1, 96, 2, 64, 4, 16, "cuda")
    with pytest.raises(TypeError, match="bf16 and head sizes"):
        PagedCache(1, 1, 64, 2, 64, 4, 16, "cuda", torch.float32)
    with pytest.raises(ValueError, match="1024 rows"):
        PagedCache(1, 1, 64, 1025, 64, 4, 16, "cuda")
    q = torch.zeros(2, 65, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="1 to 64 query heads"):
        cache.attend(0, q)
    with pytest.raises(TypeError, match="bf16 q"):
        cache.attend(0, q[:, :1].float())
    with pytest.raises(ValueError, match="q is on"):
        cache.attend(0, q[:, :1].cpu())
    with pytest.raises(ValueError, match="lengths is on"):
        paged_attention(q[:, :1], cache.pool, 0, cache.table, cache.lengths.cpu())
    pool, table, lengths, refs = cache.pool, cache.table, cache.lengths, cache.refs
    status, both = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(9, dtype=torch.int32, device="cuda")
    for out in ((both[1:].view(table.shape), lengths, refs, status), (table, lengths, refs, refs[:1])):
        with pytest.raises(ValueError, match="apart"):
            advance_pages(pool, both[:-1].view(table.shape), lengths, refs, out=out)
    with pytest.raises(ValueError, match="apart"):
        compact_pages(pool, both[:-1].view(table.shape), refs, out=(both[1:].view(table.shape), refs))
    for error, match, call in (
            (ValueError, "expected a pool", lambda: advance_pages(pool[0], table, lengths, refs)),
            (ValueError, "contiguous", lambda: advance_pages(pool[..., ::2], table, lengths, refs)),
            (TypeError, "table must be", lambda: advance_pages(pool, table.long(), lengths, refs)),
            (ValueError, "lengths", lambda: advance_pages(pool, table, lengths[:1], refs)),
            (ValueError, "refs", lambda: compact_pages(pool, table, refs[:3])),
            (ValueError, "tokens must", lambda: advance_pages(pool, table, lengths, refs, tokens=-1)),
            (ValueError, "expected parents", lambda: advance_pages(pool, table, lengths, refs, parents=refs.long()[None])),
            (TypeError, "int64", lambda: advance_pages(pool, table, lengths, refs, parents=lengths[None])),
            (ValueError, "live must be", lambda: advance_pages(pool, table, lengths, refs, live=lengths)),
            (IndexError, "block 1", lambda: paged_attention(q[:, :1], pool, 1, table, lengths)),
            (IndexError, "block -1", lambda: paged_attention(q[:, :1], pool, -1, table, lengths)),
            (ValueError, "gate", lambda: paged_attention(q[:, :2], pool, 0, table, lengths, gate=q[:, :1])),
            (ValueError, "groups of 3", lambda: paged_attention(q[:, :1], pool, 0, table, lengths, group=3)),
            (ValueError, "query heads", lambda: append_heads(q[:, 0], pool, 0, table, lengths, q[0, 0], q[0, 0],
                                                            q[0, 0], 0, 1.)),
            (ValueError, "x .*does not match", lambda: append_heads(q[:, 0], pool, 0, table, lengths, q[0, 0], q[0, 0],
                                                                   q[0, 0], 2, 1.)),
            (ValueError, "frequencies", lambda: append_heads(q[:, :4].reshape(2, 256), pool, 0, table, lengths, q[0, 0],
                                                            q[0, 0], q[0, 0], 1, 1.)),
            (ValueError, "expected keys", lambda: store_pages(pool, 0, table, lengths, q[:, 0], q[:, 0])),
            (ValueError, "values", lambda: store_pages(pool, 0, table, lengths, q[:, :1, None], q[:, :2, None]))):
        with pytest.raises(error, match=match):
            call()


# ---------------------------------------------------------------- together
def _model(head_dim=128):
    cfg = HybridConfig(vocab_size=501, hidden_size=256, intermediate_size=512, num_hidden_layers=4,
                       num_attention_heads=4, num_key_value_heads=2, head_dim=head_dim, linear_num_key_heads=2,
                       linear_num_value_heads=4, linear_key_head_dim=128, linear_value_head_dim=128,
                       linear_conv_kernel_dim=4, layer_types=["linear_attention", "full_attention"] * 2, rope_theta=1e6,
                       partial_rotary_factor=0.25)
    torch.manual_seed(0)
    model = random_model(cfg, "cuda")
    with torch.no_grad():
        model.lm_head.weight.mul_(40)  # logits that differ by more than bf16 rounds
    return model


def _replace(model, layers):
    for layer in layers:
        install(model, layer, {"head_size": 64, "backend": "cuda"})
    return model


@pytest.mark.parametrize("head_dim,replaced", [(128, ()), (256, (1,)), (64, (1, 3))])
def test_searches_agree(head_dim, replaced):
    """Eager and captured steps give the same result; its scores are those of single passes; one beam is greedy."""
    model = _replace(_model(head_dim), replaced)
    runner = Runner(model)
    prompt = torch.randint(0, 501, (2, 75), device="cuda")
    eager = beam_search(runner, prompt, 40, beams=4, page=16)
    graph = beam_search(runner, prompt, 40, beams=4, page=16, graph=True)
    for a, b in zip(eager, graph):
        assert a.shape == b.shape
    ids, scores, lengths = eager
    assert (lengths == 40).all() and (scores[:, :-1] >= scores[:, 1:]).all()
    for result in (eager, graph):
        for g in range(2):
            for k in range(4):
                runner.reset()
                tokens = result[0][g, k]
                hidden = runner.forward(torch.cat([prompt[g], tokens])[None])[0, 74:-1]
                logits = hidden.float() @ model.lm_head.weight.float().t()
                single = torch.log_softmax(logits, -1).gather(1, tokens[:, None]).sum().item()
                # 40 tokens, each with logits off by the activations' bf16 rounding in two schedules
                assert abs(single - result[1][g, k].item()) < 40 * 0.25
    runner.reset()
    assert beam_search(runner, prompt, 5, beams=1)[0].shape == (2, 1, 5)


def test_a_search_that_ends():
    model = _model()
    runner = Runner(model)
    prompt = torch.randint(0, 501, (3, 20), device="cuda")
    free, _, _ = beam_search(runner, prompt, 40, beams=3)
    end = int(free[0, 0, 2])
    for graph in (False, True):
        ids, scores, lengths = beam_search(runner, prompt, 40, beams=3, end_token=end, length_penalty=1.0, graph=graph)
        for row, length in zip(ids.view(9, 40).tolist(), lengths.view(-1).tolist()):
            assert end not in row[:length - 1] and all(token == end for token in row[length:])
            assert length == 40 or row[length - 1] == end
        assert (lengths < 40).any() and scores.isfinite().all()


def test_greedy_is_one_beam_of_the_small_model():
    model = _replace(_model(), (1, 3))
    runner = Runner(model)
    prompt = torch.randint(0, 501, (1, 33), device="cuda")
    greedy = generate(runner, prompt, 6)
    ids, scores, _ = beam_search(runner, prompt, 6, beams=1)
    # both take the largest of bf16 logits, which may differ where two are closest: compare while they agree
    assert ids[0, 0, 0] == greedy[0, 0] and scores.isfinite().all()


def _search_state(G=2, K=4, seed=0):
    """Tensors of a small search in the middle, and one step over them in place."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, V = G * K, 1501
    cache = PagedCache(2, 2, 64, rows, 400, 150, 16, "cuda")
    cache.pool.normal_(generator=g)
    cache.advance_(33, live=torch.arange(K, device="cuda").expand(G, K) == 0)
    cache.advance_(0, torch.zeros(G, K, dtype=torch.int64, device="cuda"))
    x = torch.randn(rows, (2 * 6 + 4) * 64, device="cuda", generator=g).to(torch.bfloat16)
    noise = torch.randn(rows, V, 384, device="cuda", generator=g) * 0.05
    w = torch.randn(64, device="cuda", generator=g) * 0.1
    freq = torch.rand(16, device="cuda", generator=g)
    beams = [torch.arange(K, device="cuda").repeat(G, 1), torch.zeros(G, K, device="cuda"),
             torch.ones(G, K, dtype=torch.int32, device="cuda"), torch.zeros(G, K, dtype=torch.bool, device="cuda")]
    states = [torch.randn(rows, 3, 50, device="cuda", generator=g), torch.arange(rows * 7, device="cuda").view(rows, 7)]
    seen = torch.zeros(rows, 384, device="cuda")

    def step():
        parents, scores, lengths, finished = beams
        reorder_states_(states + [seen], parents)
        cache.advance_(1, parents, ~finished)
        q = cache.append_(1, x, w, w, freq, 6, 1e-6)
        seen.mul_(0.5).add_(cache.attend(1, q, x[:, :768].view(rows, 6, 128)[..., 64:], K).reshape(rows, 384).float())
        logits = torch.einsum("rc,rvc->rv", seen, noise).view(G, K, V)
        tokens, *chosen = beam_select(logits, scores, lengths, finished, end_token=7, length_penalty=0.5)
        for mine, new in zip(beams, chosen):
            mine.copy_(new)
        states[1].add_(tokens.view(rows, 1))
        return [cache.pool, cache.table, cache.lengths, cache.refs, cache.status, seen, *states, *beams]

    return step


def test_a_captured_step_replays_like_an_eager_one():
    eager, replayed = _search_state(), _search_state()
    first = [x.clone() for x in replayed()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = replayed()
    for got, want in zip(first, eager()):
        assert torch.equal(got, want)
    for _ in range(20):
        graph.replay()
        want = eager()
        for got, value in zip(static, want):
            assert torch.equal(got, value)
    assert int(static[4]) == 0


def test_calls_on_two_streams_at_once():
    """Workspaces belong to a call: two searches on streams of their own do not meet."""
    alone = _search_state(seed=1)
    for _ in range(25):
        want = alone()
    steps = [_search_state(seed=1), _search_state(seed=1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(25):
        results = []
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                results.append(step())
    torch.cuda.synchronize()
    for result in results:
        for got, value in zip(result, want):
            assert torch.equal(got, value)


def test_offsets_beyond_32_bits():
    pages = 2 ** 31 // (2 * 2 * 4 * 64 * 256) + 40  # of 2 blocks and 4 heads of 256: more than 2^31 elements
    pool = torch.empty(pages, 2, 2, 4, 64, 256, device="cuda", dtype=torch.bfloat16)
    small = torch.randn(12, 2, 2, 4, 64, 256).to(torch.bfloat16)
    pool[pages - 12:] = small.cuda()
    table = torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32)
    far = torch.where(table >= 0, table + pages - 12, table)
    lengths = torch.tensor([100, 190], dtype=torch.int32)
    q = torch.randn(2, 8, 256).to(torch.bfloat16)
    out = paged_attention(q.cuda(), pool, 1, far.cuda(), lengths.cuda())
    assert torch.equal(out, paged_attention(q.cuda(), small.cuda(), 1, table.cuda(), lengths.cuda()))
    x = torch.randn(2, 24 * 256).to(torch.bfloat16).cuda()
    w, freq = torch.zeros(256, device="cuda"), torch.ones(8, device="cuda")
    near = small.cuda()
    append_heads(x, pool, 1, far.cuda(), lengths.cuda(), w, w, freq, 8, 1e-6)
    append_heads(x, near, 1, table.cuda(), lengths.cuda(), w, w, freq, 8, 1e-6)
    k = torch.randn(2, 30, 4, 256).to(torch.bfloat16).cuda()
    store_pages(pool, 0, far.cuda(), lengths.cuda(), k, k)
    store_pages(near, 0, table.cuda(), lengths.cuda(), k, k)
    assert torch.equal(pool[pages - 12:], near)
    refs = torch.ones(pages, dtype=torch.int32)
    refs[3] = refs[pages - 6] = refs[pages - 1] = 0
    refs[pages - 12] = 2
    shared = torch.tensor([[pages - 12, -1], [pages - 12, -1]], dtype=torch.int32, device="cuda")
    held = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    refs[4:6] = 0
    new, _, count, status = advance_pages(pool, shared, held, refs.cuda(), 1)
    assert new[0, 0] == 3 and new[1, 0] == pages - 12 and int(status) == 0
    assert torch.equal(pool[3, ..., :20, :], near[0, ..., :20, :])
    moved, _, used = compact_pages(pool, far.cuda(), count)
    assert int(used) == int((count > 0).sum()) == pages - 4
    # free were 4, 5, pages - 6 and pages - 1: of the last four pages the three in use move to the first three of those
    assert torch.equal(pool[4], near[8]) and torch.equal(pool[5], near[9]) and torch.equal(pool[pages - 6], near[10])
    assert torch.equal(moved.cpu(), far)
    del pool
    state = torch.arange(3, device="cuda", dtype=torch.uint8)[:, None].repeat(1, 3 << 30)
    reorder_states_([state], torch.tensor([[2, 1, 1]], device="cuda"))
    assert [int(state[r].min()) for r in range(3)] == [int(state[r].max()) for r in range(3)] == [2, 1, 1]
    del state
    wide = torch.empty(2 ** 31 + 5000, device="cuda", dtype=torch.bfloat16)
    logits = wide.as_strided((2, 2, 2001), (2 ** 31 + 7, 2003, 1))
    logits.normal_()
    scores, ends = torch.zeros(2, 2, device="cuda"), torch.zeros(2, 2, dtype=torch.bool, device="cuda")
    args = (scores, torch.ones(2, 2, dtype=torch.int32, device="cuda"), ends)
    for a, b in zip(beam_select(logits, *args), beam_select(logits.clone(), *args)):
        assert torch.equal(a, b)
