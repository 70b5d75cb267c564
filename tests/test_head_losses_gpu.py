"""Vocabulary-head losses and top log-probabilities on the GPU against 64-bit formulas.

Tolerances (u = 2^-8, bf16's unit roundoff: 8 significant bits). Logits are fp32 sums of exact bf16 products, C / 16 MMA steps that each
may lose 2^-23 of a partial sum bounded by |x| |w|: dz = scale (C / 16 + 16) 2^-23 max|x| max|w|. A loss is off by at
most 2 dz, and by fp32 rounding. A gradient's factors are rounded to bf16 twice at most (its exponentials or logit
gradients, and scaled hidden rows), its result once, and the exponentials follow dz: (3 u + 4 dz) times the same
product of absolute values.
"""
import math

import pytest
import torch

from rwkv_theseus_b200.losses import linear_cross_entropy, linear_topk_kl, top_log_probs

pytestmark = pytest.mark.gpu
cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA unavailable")
U = 2.0 ** -8


def _inputs(T, V, C, seed=0, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * T + V + C)
    weight = (torch.randn(V, C, device="cuda", generator=g) * (1.4 / math.sqrt(C))).to(torch.bfloat16)
    targets = torch.randint(0, V, (T,), device="cuda", generator=g)
    pull = torch.rand(T, 1, device="cuda", generator=g) * 6
    hidden = (gain * (torch.randn(T, C, device="cuda", generator=g) + pull * weight[targets].float()))
    return hidden.to(torch.bfloat16), weight, targets, g


def _record(hidden, weight, K, temperature, g):
    noisy = hidden.float() + torch.randn(hidden.shape, device="cuda", generator=g)
    return top_log_probs(torch.nan_to_num(noisy) @ weight.float().t(), K, temperature)


def _oracle(hidden, weight, index, log_probs, ignore, scale, tail):
    """Row losses and d loss / d logits (unscaled rows) in 64 bits, from the definition."""
    z = hidden.double() @ weight.double().t() * scale
    held = index != ignore if log_probs is None else index >= 0
    valid = held.any(-1)
    log_probs = torch.zeros(index.shape, device="cuda") if log_probs is None else log_probs
    p = torch.where(held, log_probs.double().exp(), 0.0)
    inside = torch.zeros(z.shape, dtype=torch.int32, device="cuda").scatter_add_(1, index.clamp_min(0), held.int()) > 0
    q = torch.softmax(z, -1)
    log_q = torch.log_softmax(z, -1)
    log_p = torch.where(p > 0, p.log(), 0.0)
    loss = (p * (log_p - log_q.gather(1, index.clamp_min(0)))).sum(-1)
    mass = p.sum(-1, keepdim=True)
    rest = (1 - mass).clamp_min(0) * tail * (~inside).any(-1, keepdim=True)
    log_rest = log_q.masked_fill(inside, -math.inf).logsumexp(-1, keepdim=True)
    loss = loss + torch.where(rest > 0, rest * (rest.log() - log_rest), 0.0)[:, 0]
    dz = q * (mass + rest) - torch.where(inside | (rest <= 0), 0.0, rest * (log_q - log_rest).exp())
    dz = dz.scatter_add(1, index.clamp_min(0), -p)
    if index.shape[1] == 1 and not log_probs.any():  # one entry of probability one: q - 1 without cancellation
        dz = dz.scatter(1, index.clamp_min(0), -torch.where(p > 0, log_rest.exp(), 0.0))
    return loss.masked_fill(~valid, 0.0), dz.masked_fill(~valid[:, None], 0.0), valid


def _check(hidden, weight, index, log_probs, temperature, tail, reduction, grad_w=True, upstream=1.0):
    scale = 1.0 / temperature
    held = (index != -100) if log_probs is None else (index >= 0)
    clean = hidden.masked_fill(~held.any(-1)[:, None], 0.0)
    hidden = hidden.clone().requires_grad_()
    weight = weight.clone().requires_grad_(grad_w)
    if log_probs is None:
        got = linear_cross_entropy(hidden, weight, index[:, 0], reduction=reduction)
    else:
        got = linear_topk_kl(hidden, weight, index, log_probs, temperature, tail, reduction)
    loss, dz, valid = _oracle(clean, weight.detach(), index, log_probs, -100,
                              scale, tail)
    T, C = hidden.shape
    n = max(int(valid.sum()), 1)
    xmax, wmax = clean.float().norm(dim=-1).max().item(), weight.detach().float().norm(dim=-1).max().item()
    err = scale * (C / 16 + 16) * 2.0 ** -23 * xmax * wmax
    if reduction == "none":
        factor = torch.linspace(-1.0, 2.0, T, device="cuda")
        value, rows = loss, factor.double()
    else:
        factor = torch.tensor(upstream, device="cuda")
        rows = torch.full((T,), upstream / (n if reduction == "mean" else 1), device="cuda", dtype=torch.float64)
        value = loss.sum() / (n if reduction == "mean" else 1)
    slack = 2 * err * (n if reduction == "sum" else 1)
    torch.testing.assert_close(got.detach().double(), value, rtol=1e-5, atol=slack + 1e-6)
    wanted = [hidden] + ([weight] if grad_w else [])
    grads = torch.autograd.grad(got, wanted, factor.to(got.dtype))
    dz = dz * rows[:, None] * scale
    tol = 3 * U + 4 * err
    if upstream != 1.0:
        tol += U  # multiplied after its rounding
    _within(grads[0], dz @ weight.detach().double(), tol * (dz.abs() @ weight.detach().double().abs()))
    if grad_w:
        x = clean.double()
        _within(grads[1], dz.t() @ x, tol * (dz.abs().t() @ x.abs()))


def _within(got, expected, bound):
    assert got.dtype == torch.bfloat16 and torch.isfinite(got).all()
    excess = (got.double() - expected).abs() - bound - 1e-30
    assert (excess <= 0).all(), f"{(excess > 0).sum().item()} entries beyond the bound, by {excess.max().item()}"


SHAPES = [(1, 1, 8), (1, 700, 64), (3, 64, 8), (16, 4096, 1024), (127, 257, 72), (128, 256, 64), (129, 1003, 520),
          (300, 9001, 128), (33, 20000, 64)]


@cuda
@pytest.mark.parametrize("T,V,C", SHAPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_cross_entropy(T, V, C, reduction):
    hidden, weight, targets, g = _inputs(T, V, C)
    targets[: T // 3] = -100
    targets[-1] = V - 1
    _check(hidden, weight, targets[:, None], None, 1.0, False, reduction)


@cuda
@pytest.mark.parametrize("T,V,C,K", [(1, 8, 8, 8), (5, 700, 64, 1), (16, 4096, 1024, 8), (127, 257, 72, 33),
                                     (129, 1003, 520, 64), (300, 9001, 128, 256), (7, 20000, 64, 1024)])
@pytest.mark.parametrize("tail", [False, True])
def test_topk_kl(T, V, C, K, tail):
    hidden, weight, _, g = _inputs(T, V, C)
    log_probs, index = _record(hidden, weight, K, 2.0, g)
    keep = torch.randint(0, K + 1, (T, 1), device="cuda", generator=g)
    index[T // 2:] = index[T // 2:].masked_fill(torch.arange(K, device="cuda") >= keep[T // 2:], -1)
    shuffle = torch.randperm(K, device="cuda", generator=g)  # a record's order is free
    _check(hidden, weight, index[:, shuffle], log_probs[:, shuffle], 2.0, tail, "mean")
    _check(hidden, weight, index, log_probs, 2.0, tail, "none", grad_w=False)


@cuda
def test_sum_and_upstream_factor():
    hidden, weight, targets, _ = _inputs(65, 1500, 128)
    _check(hidden, weight, targets[:, None], None, 1.0, False, "sum")
    _check(hidden, weight, targets[:, None], None, 1.0, False, "mean", upstream=-0.37)


@cuda
@pytest.mark.parametrize("V", [513, 5000])
def test_masked_rows_hold_anything(V):
    hidden, weight, targets, g = _inputs(140, V, 64)
    targets[10:20] = -100
    targets[139] = -100
    hidden[10:14] = math.nan
    hidden[14:17] = math.inf
    hidden[139] = -3e38
    _check(hidden, weight, targets[:, None], None, 1.0, False, "mean")
    log_probs, index = _record(hidden, weight, 16, 1.0, g)
    index[10:20] = -1
    index[139] = -1
    log_probs[10] = math.nan
    _check(hidden, weight, index, log_probs, 1.0, True, "mean")


@cuda
def test_no_row_left():
    hidden, weight, targets, _ = _inputs(30, 300, 64)
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = linear_cross_entropy(hidden, weight, torch.full_like(targets, -100))
    dh, dw = torch.autograd.grad(loss, (hidden, weight))
    assert loss.item() == 0.0 and not dh.any() and not dw.any()
    empty = linear_cross_entropy(hidden[:0], weight, targets[:0])
    dh, dw = torch.autograd.grad(empty, (hidden, weight))
    assert empty.item() == 0.0 and not dh.any() and not dw.any()


@cuda
@pytest.mark.parametrize("gain", [12.0, 60.0])
@pytest.mark.parametrize("tail", [False, True])
def test_wide_logits(gain, tail):
    """Logits hundreds apart: targets and records far below the row's maximum, probabilities that underflow."""
    hidden, weight, targets, g = _inputs(150, 2300, 64, gain=gain)
    targets[::2] = torch.randint(0, 2300, (75,), device="cuda", generator=g)
    _check(hidden, weight, targets[:, None], None, 1.0, False, "mean")
    log_probs, index = _record(torch.randn_like(hidden), weight, 12, 1.0, g)
    _check(hidden, weight, index, log_probs, 1.0, tail, "mean")


@cuda
def test_records_inside_one_tile():
    """All entries of all rows in the first columns, as frequent tokens with low ids are."""
    hidden, weight, _, g = _inputs(200, 3000, 64)
    logits = hidden.float() @ weight.float().t()
    logits[:, 130:] = -30.0
    log_probs, index = top_log_probs(logits, 128)
    _check(hidden, weight, index, log_probs, 1.0, True, "mean")


@cuda
def test_entries_without_mass():
    hidden, weight, _, g = _inputs(40, 900, 64)
    log_probs, index = _record(hidden, weight, 10, 1.0, g)
    log_probs[:, 6:] = -math.inf
    for tail in (False, True):
        _check(hidden, weight, index, log_probs, 1.0, tail, "mean")


@cuda
def test_strided_operands_and_index_types():
    hidden, weight, targets, _ = _inputs(50, 700, 64)
    wide_h = torch.full((50, 80), math.nan, device="cuda", dtype=torch.bfloat16)
    wide_w = torch.full((700, 128), math.nan, device="cuda", dtype=torch.bfloat16)
    wide_h[:, 8:72], wide_w[:, 64:] = hidden, weight
    plain = linear_cross_entropy(hidden, weight, targets, reduction="none")
    for h in (wide_h[:, 8:72], hidden.t().contiguous().t(), hidden.view(2, 25, 64).transpose(0, 1)):
        t = targets if h.dim() == 2 else targets.view(2, 25).t()
        w = wide_w[:, 64:].detach().requires_grad_()
        h = h.detach().requires_grad_()
        got = linear_cross_entropy(h, w, t.int(), reduction="none")
        assert torch.equal(got, plain if h.dim() == 2 else plain.view(2, 25).t())
        dh, dw = torch.autograd.grad(got.sum(), (h, w))
        assert dh.shape == h.shape and dw.shape == w.shape and torch.isfinite(dh).all() and torch.isfinite(dw).all()


@cuda
def test_results_do_not_change_between_calls():
    hidden, weight, targets, g = _inputs(190, 5000, 256)
    hidden.requires_grad_()
    weight.requires_grad_()
    log_probs, index = _record(hidden.detach(), weight.detach(), 32, 1.0, g)
    first = None
    for _ in range(4):
        loss = linear_topk_kl(hidden, weight, index, log_probs)
        out = (loss.detach(), *torch.autograd.grad(loss, (hidden, weight)))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@cuda
def test_backward_twice():
    hidden, weight, targets, _ = _inputs(20, 300, 64)
    hidden.requires_grad_()
    loss = linear_cross_entropy(hidden, weight, targets)
    a = torch.autograd.grad(loss, hidden, torch.tensor(2.0, device="cuda"), retain_graph=True)[0].clone()
    b = torch.autograd.grad(loss, hidden)[0]
    torch.testing.assert_close(a.float(), 2 * b.float(), rtol=0, atol=0)


@cuda
def test_gradient_against_differences():
    """The loss is smooth: for a step e along d, (L(x + e d) - L(x - e d)) / 2e = <grad, d> + O(e^2) third
    derivatives. Steps are exact in bf16 (a power of two added to entries on a grid of it); the bound is the fp32
    loss's noise over the step plus |d|^3-scaled curvature, sum of |w|^3 terms bounded by the logits' change cubed."""
    hidden, weight, targets, g = _inputs(9, 400, 64)
    step = 2.0 ** -4
    hidden = (hidden.float() / step).round().clamp(-100, 100).mul(step).to(torch.bfloat16)
    direction = torch.randint(-1, 2, hidden.shape, device="cuda", generator=g).to(torch.bfloat16)
    x = hidden.clone().requires_grad_()
    grad = torch.autograd.grad(linear_cross_entropy(x, weight, targets, reduction="sum"), x)[0]
    plus = linear_cross_entropy(hidden + step * direction, weight, targets, reduction="none").double()
    minus = linear_cross_entropy(hidden - step * direction, weight, targets, reduction="none").double()
    change = (step * direction.double()) @ weight.double().t()
    spread = (change.amax(-1) - change.amin(-1))
    # |third derivative of log-sum-exp along a line| <= spread^3; remainder of the central difference is a sixth of it
    bound = spread ** 3 / 6 + 2e-5 + 3 * U * change.abs().amax(-1) * 2
    slope = (grad.double() * step * direction.double()).sum(-1)
    assert ((plus - minus) / 2 - slope).abs().le(bound).all()


@cuda
def test_an_index_outside_the_vocabulary():
    hidden, weight, targets, _ = _inputs(40, 300, 64)
    hidden.requires_grad_()
    weight.requires_grad_()
    targets[7], targets[8] = 300, -5
    loss = linear_cross_entropy(hidden, weight, targets, reduction="none")
    dh, dw = torch.autograd.grad(loss, (hidden, weight), torch.ones_like(loss))
    assert torch.isnan(loss[7:9]).all() and torch.isfinite(loss).sum() == 38
    assert not dh[7:9].any() and torch.isfinite(dh).all() and torch.isfinite(dw).all()
    index = torch.tensor([[3, 2 ** 40]], device="cuda")
    assert torch.isnan(linear_topk_kl(hidden[:1], weight, index, torch.zeros(1, 2, device="cuda")))


@cuda
def test_side_stream():
    hidden, weight, targets, _ = _inputs(64, 3000, 256)
    expected = linear_cross_entropy(hidden, weight, targets, reduction="none")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_cross_entropy(hidden, weight, targets, reduction="none")
        top = top_log_probs(hidden, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, expected)
    assert torch.equal(top[1], top_log_probs(hidden, 5)[1])


def _top(logits, k, temperature=1.0):
    z = logits.double() + 0.0
    index = torch.sort(z, dim=-1, descending=True, stable=True)[1][..., :k]
    return torch.log_softmax(z / temperature, -1).gather(-1, index), index


def _check_top(logits, k, temperature=1.0):
    got, index = top_log_probs(logits, k, temperature)
    expected, order = _top(logits, k, temperature)
    assert index.dtype == torch.int64 and got.dtype == torch.float32
    assert torch.equal(index, order)
    # fp32 logit / temperature and a denominator summed in fp32: a few roundings of the largest magnitude
    scale = logits.double().nan_to_num(0, 0, 0).abs().max().item() / temperature
    torch.testing.assert_close(got.double(), expected, rtol=0, atol=8 * 2.0 ** -24 * (scale + 32))


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (2, 31, 31), (5, 1001, 7), (3, 4097, 1024), (40, 32003, 200),
                                      (1, 248077, 64), (300, 700, 64), (2, 131072, 1000)])
def test_top_log_probs(dtype, rows, V, k):
    g = torch.Generator(device="cuda").manual_seed(rows + V + k)
    logits = (torch.randn(rows, V, device="cuda", generator=g) * 3).to(dtype)
    _check_top(logits, k)
    _check_top(logits, k, 2.5)


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_log_probs_ties_and_orders(dtype):
    V = 20011
    ramp = torch.linspace(-4, 4, V, device="cuda")
    rows = [ramp, ramp.flip(0), torch.zeros(V, device="cuda"), -torch.zeros(V, device="cuda"),
            torch.where(torch.arange(V, device="cuda") % 3 == 0, 0.0, -0.0), (ramp * 3).round(),
            torch.where(torch.arange(V, device="cuda") == V - 1, 5.0, -5.0),
            torch.where(torch.arange(V, device="cuda") < 40, ramp, -math.inf)]
    _check_top(torch.stack(rows).to(dtype), 100)


@cuda
def test_top_log_probs_strides_and_infinities():
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(6, 5003, device="cuda", generator=g).to(torch.bfloat16)
    _check_top(wide[:, 3:4000], 50)
    _check_top(wide[::2, 1:], 50)
    _check_top(wide.t().contiguous().t(), 9)
    _check_top(wide.view(2, 3, 5003), 9)
    odd = torch.randn(3, 999, device="cuda", generator=g)
    odd[0] = -math.inf
    odd[1, 500], odd[2, 7] = math.inf, math.nan
    log_probs, index = top_log_probs(odd, 4)
    assert index[0].tolist() == [0, 1, 2, 3] and index[1, 0] == 500 and index[2, 0] == 7
    assert torch.isnan(log_probs[0]).all() and torch.isnan(log_probs[1, 0]) and torch.isnan(log_probs[2]).all()


@cuda
def test_gpu_refusals():
    hidden, weight, targets, _ = _inputs(4, 300, 64)
    with pytest.raises(TypeError, match="bf16"):
        linear_cross_entropy(hidden.float(), weight, targets)
    with pytest.raises(TypeError, match="bf16"):
        linear_cross_entropy(hidden, weight.float(), targets)
    with pytest.raises(ValueError, match="multiples of 8"):
        linear_cross_entropy(hidden[:, :60], weight[:, :60], targets)
    with pytest.raises(ValueError, match="multiples of 8"):
        linear_cross_entropy(hidden, weight.t().contiguous().t(), targets)
    with pytest.raises(ValueError, match="devices"):
        linear_cross_entropy(hidden, weight, targets.cpu())
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(linear_cross_entropy(hidden.requires_grad_(), weight, targets), hidden, create_graph=True)
    with pytest.raises(ValueError, match="devices"):
        linear_cross_entropy(hidden, weight.cpu(), targets)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        top_log_probs(hidden.half(), 3)


@cuda
@pytest.mark.parametrize("ignored", [0, 500, 32900])
def test_more_rows_than_a_chunk(ignored):
    """32768 rows at a time with gradients, 16384 without; the weight's gradient adds up over the chunks."""
    hidden, weight, targets, g = _inputs(33000, 300, 64)
    targets[torch.randperm(33000, device="cuda", generator=g)[:ignored]] = -100
    _check(hidden, weight, targets[:, None], None, 1.0, False, "sum")
    loss = linear_cross_entropy(hidden, weight, targets, reduction="none")
    expected, _, _ = _oracle(hidden, weight, targets[:, None], None, -100, 1.0, 0)
    torch.testing.assert_close(loss.double(), expected, rtol=1e-5, atol=1e-4)


@cuda
def test_offsets_beyond_32_bits():
    """A weight of 2.2e9 entries and logits of 2.2e9: the first and last rows against 64 bits."""
    V, C, T = 430003, 5120, 40
    g = torch.Generator(device="cuda").manual_seed(8)
    weight = torch.empty(V, C, device="cuda", dtype=torch.bfloat16).normal_(0, 1.4 / math.sqrt(C), generator=g)
    hidden = torch.randn(T, C, device="cuda", generator=g).to(torch.bfloat16)
    targets = torch.randint(V - 2000, V, (T,), device="cuda", generator=g)
    z = torch.cat([hidden.double() @ part.double().t() for part in weight.split(50000)], 1)
    q = torch.softmax(z, -1)
    dz = q.scatter_add(1, targets[:, None], torch.full((T, 1), -1.0, device="cuda", dtype=torch.float64)) / T
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = linear_cross_entropy(h, w, targets)
    dh, dw = torch.autograd.grad(loss, (h, w))
    x = hidden.detach().double()
    err = (C / 16 + 16) * 2.0 ** -23 * x.norm(dim=-1).max().item() * 1.6
    expected = torch.nn.functional.cross_entropy(z, targets)
    torch.testing.assert_close(loss.detach().double(), expected, rtol=1e-5, atol=2 * err)
    last = slice(V - 2000, V)
    tol = 3 * U + 4 * err
    for rows in (slice(0, 64), last):
        _within(dw[rows], dz[:, rows].t() @ x, tol * (dz[:, rows].abs().t() @ x.abs()))
    expected = sum(dz[:, a:a + 50000] @ weight[a:a + 50000].detach().double() for a in range(0, V, 50000))
    bound = sum(dz[:, a:a + 50000].abs() @ weight[a:a + 50000].detach().double().abs() for a in range(0, V, 50000))
    _within(dh, expected, tol * bound)
    del weight, w, dw, z, q, dz
    logits = torch.empty(8700, 248077, device="cuda", dtype=torch.bfloat16).normal_(0, 2, generator=g)
    log_probs, index = top_log_probs(logits, 7)
    for row in (0, 8699):
        expected, order = _top(logits[row:row + 1], 7)
        assert torch.equal(index[row:row + 1], order)
        torch.testing.assert_close(log_probs[row:row + 1].double(), expected, rtol=0, atol=1e-4)


@cuda
def test_calls_in_a_cuda_graph():
    hidden, weight, targets, g = _inputs(96, 3000, 256)
    hidden.requires_grad_()
    weight.requires_grad_()

    def call():
        loss = linear_cross_entropy(hidden, weight, targets)
        return (loss.detach(), *torch.autograd.grad(loss, (hidden, weight)), *top_log_probs(hidden.detach(), 5))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    with torch.no_grad():
        targets.copy_(targets.flip(0))
        hidden.mul_(1.5)
    graph.replay()
    for a, b in zip(out, call()):
        assert torch.equal(a, b)


@cuda
@pytest.mark.parametrize("T", [1, 31, 32, 33, 128, 129])
def test_scores_equal_the_losses_of_a_training_call(T):
    """Without gradients few rows take a path of their own: the same bits per token, whatever masked rows hold, and the
    same sums but for the order of 64-bit additions."""
    hidden, weight, targets, _ = _inputs(T, 1500, 136)
    targets[T // 2:T // 2 + 3] = -100
    hidden[T // 2] = math.nan
    if T > 8:
        hidden[T // 2 + 1] = math.inf
        targets[2], targets[5] = 1500, -7
    for reduction in ("none", "sum", "mean"):
        score = linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        loss = linear_cross_entropy(hidden.clone().requires_grad_(), weight, targets, reduction=reduction).detach()
        tolerance = 0 if reduction == "none" else 1e-6
        torch.testing.assert_close(score, loss, rtol=tolerance, atol=0, equal_nan=True)
    if T > 8:
        targets[2] = targets[5] = 3
    for reduction in ("sum", "mean"):
        score = linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        loss = linear_cross_entropy(hidden.clone().requires_grad_(), weight, targets, reduction=reduction).detach()
        assert torch.isfinite(score)
        torch.testing.assert_close(score, loss, rtol=1e-6, atol=0)
