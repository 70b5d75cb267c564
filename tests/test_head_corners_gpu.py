"""Corners of the vocabulary-head operators on the GPU against 64-bit formulas: students that are sure of their record,
records of the whole vocabulary, logits of any size, masks of the type's lowest value, NaN.

Tolerances are those of test_head_losses_gpu.py (u = 2^-8; a gradient is off by (3 u + 4 dz) times the same product of
absolute values, dz the bound of a logit's error) unless a test derives its own.
"""
import ctypes
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

from rwkv_theseus_b200.losses import linear_cross_entropy, linear_topk_kl, top_log_probs
from test_head_losses_gpu import U, _check, _inputs, _oracle, _record, _within

pytestmark = pytest.mark.gpu
cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA unavailable")


def _sure(T, V, gap, mass, entries=4):
    """Rows whose student is `gap` nats surer of its `entries` recorded tokens than of the rest, where the teacher's
    record holds `mass`. Feature j of the width stands for the j-th group of tokens and is zero for all others."""
    g = torch.Generator(device="cuda").manual_seed(T + V + int(gap))
    weight = torch.randn(V, 64, device="cuda", generator=g) * 0.15
    hidden = torch.randn(T, 64, device="cuda", generator=g)
    weight[:, :8] = 0.0
    hidden[:, :8] = 0.0
    for j in range(8):
        weight[j * entries:(j + 1) * entries, j] = 1.0
    group = torch.randint(0, 8, (T,), device="cuda", generator=g)
    hidden[torch.arange(T, device="cuda"), group] = gap
    index = group[:, None] * entries + torch.arange(entries, device="cuda")
    p = torch.rand(T, entries, device="cuda", generator=g) + 0.2
    return hidden.to(torch.bfloat16), weight.to(torch.bfloat16), index, (p / p.sum(-1, keepdim=True) * mass).log()


@cuda
@pytest.mark.parametrize("T", [5, 100, 150])
@pytest.mark.parametrize("gap", [80.0, 100.0, 300.0])
@pytest.mark.parametrize("mass,entries", [(0.5, 4), (0.9, 1), (0.999999, 4)])
def test_a_student_that_is_sure_of_its_record(T, gap, mass, entries):
    """The rest of the vocabulary has a probability of e^-gap, and is all that pushes mass back to it."""
    hidden, weight, index, log_probs = _sure(T, 1003, gap, mass, entries)
    _check(hidden, weight, index, log_probs, 1.0, True, "mean")
    _check(hidden, weight, index, log_probs, 0.5, True, "none")
    _check(hidden, weight, index, log_probs, 1.0, False, "mean")


@cuda
@pytest.mark.parametrize("T", [5, 100, 150])
@pytest.mark.parametrize("V", [8, 64, 700])
def test_a_record_of_the_whole_vocabulary_without_all_its_mass(T, V):
    """Nothing is left for the rest's class, in the loss and in its gradient."""
    hidden, weight, _, g = _inputs(T, V, 64)
    log_probs, index = _record(hidden, weight, V, 1.0, g)
    _check(hidden, weight, index, log_probs + math.log(0.6), 1.0, True, "mean")
    log_probs[:, 1:3] = -math.inf
    _check(hidden, weight, index, log_probs, 1.0, True, "none")


@cuda
@pytest.mark.parametrize("T", [20, 100, 150])
def test_the_largest_of_very_large_logits(T):
    """Two equal logits share each row, one of them its target; all others are far below. They are exact (one product
    and zeros), so the other one's gradient is 1/2 up to the 16-bit form of its logit (2^-10 octaves, 7e-4) and two
    roundings to bf16."""
    hidden = torch.zeros(T, 64, device="cuda")
    hidden[:, 0] = torch.linspace(8192, 32000, T, device="cuda").to(torch.bfloat16)
    weight = torch.zeros(600, 64, device="cuda")
    weight[5, 0], weight[300, 0], weight[300, 1] = 1.0, 1.0, 1.0
    hidden = hidden.to(torch.bfloat16).requires_grad_()
    weight = weight.to(torch.bfloat16).requires_grad_()
    loss = linear_cross_entropy(hidden, weight, torch.full((T,), 5, device="cuda"), reduction="sum")
    dh, dw = torch.autograd.grad(loss, (hidden, weight))
    half = torch.full((T,), 0.5, device="cuda", dtype=torch.float64)
    torch.testing.assert_close(dh[:, 1].double(), half, rtol=0, atol=0.5 * (7e-4 + 2 * U))
    half = 0.5 * hidden[:, 0].detach().double().sum()
    torch.testing.assert_close(dw[300, 0].double(), half, rtol=7e-4 + 2 * U, atol=0)
    torch.testing.assert_close(dw[5, 0].double(), -half, rtol=7e-4 + 2 * U, atol=0)


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 20011, 248077])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
def test_top_log_probs_of_masks_of_the_lowest_value(dtype, V, temperature):
    """Logits masked by the type's lowest number: most of a row, all but one entry, all of it, and beside the largest.
    Expected in 64 bits, rounded to fp32 (a masked entry may be -inf there); the bound is that of
    test_head_losses_gpu.py for the unmasked logits, and the magnitude's rounding for the masked ones."""
    g = torch.Generator(device="cuda").manual_seed(V)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = torch.randn(6, V, device="cuda", generator=g).mul_(3).to(dtype)
    logits[0, : V // 2] = low
    logits[1, 20:] = low
    logits[2, 1:] = low
    logits[3] = low
    logits[4, 7] = high
    logits[5, ::2], logits[5, 1::2] = low, -math.inf
    got, index = top_log_probs(logits, 30, temperature)
    z = logits.double()
    order = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :30]
    expected = torch.log_softmax(z / temperature, -1).gather(1, order).float()
    assert torch.equal(index, order)
    torch.testing.assert_close(got, expected, rtol=2.0 ** -21, atol=8 * 2.0 ** -24 * (20 / temperature + 32))


@cuda
@pytest.mark.parametrize("T", [20, 150])
def test_a_weight_without_numbers(T):
    """Logits that are NaN have NaN gradients, held or not."""
    hidden, weight, targets, _ = _inputs(T, 700, 64)
    weight[:, 3] = math.nan
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = linear_cross_entropy(hidden, weight, targets)
    dh, dw = torch.autograd.grad(loss, (hidden, weight))
    assert torch.isnan(loss) and torch.isnan(dh).all() and torch.isnan(dw).all()


class _Call(ctypes.Structure):
    """RtHeadLoss of csrc/api.h."""
    _fields_ = [("hidden", ctypes.c_void_p), ("ld_hidden", ctypes.c_long), ("weight", ctypes.c_void_p),
                ("ld_weight", ctypes.c_long), ("index", ctypes.c_void_p), ("log_probs", ctypes.c_void_p),
                ("rows", ctypes.c_long), ("vocab", ctypes.c_long), ("width", ctypes.c_int), ("K", ctypes.c_int),
                ("ignore", ctypes.c_long), ("scale", ctypes.c_float), ("tail", ctypes.c_int),
                ("reduction", ctypes.c_int), ("row_grad", ctypes.c_void_p), ("row_loss", ctypes.c_void_p),
                ("loss", ctypes.c_void_p), ("dhidden", ctypes.c_void_p), ("dweight", ctypes.c_void_p)]


@cuda
@pytest.mark.parametrize("T,grad_h,grad_w", [(5, False, False), (5, True, True), (5, False, True), (150, True, True),
                                             (150, False, True), (33000, False, True)])
def test_a_product_that_gave_up_a_wait_leaves_nan(T, grad_h, grad_w):
    """The status word as such a product leaves it, set before the call: no number comes back that looks like a result.
    Unset, the entry does what the public function does. (No kernel is kept waiting here.)"""
    from rwkv_theseus_b200.ops import native
    lib = ctypes.CDLL(native().__file__)
    floats = lib.rt_head_loss_workspace_floats
    floats.restype, floats.argtypes = ctypes.c_long, [ctypes.c_long] * 2 + [ctypes.c_int] * 4
    run = lib.rt_head_loss_status
    run.argtypes = [ctypes.c_void_p] * 4
    hidden, weight, targets, _ = _inputs(T, 300, 64)
    targets[1] = -100
    live = targets != -100
    rows, loss = torch.empty(T, device="cuda"), torch.empty((), device="cuda")
    dh, dw = torch.empty_like(hidden), torch.empty_like(weight)
    work = torch.empty(floats(T, 300, 64, 1, grad_h, grad_w), device="cuda")
    for fault in (0, 1):
        status = torch.full((1,), fault, device="cuda", dtype=torch.int32)
        call = _Call(hidden.data_ptr(), 64, weight.data_ptr(), 64, targets.data_ptr(), None, T, 300, 64, 1, -100,
                     1.0, 0, 2, None, rows.data_ptr(), loss.data_ptr(), dh.data_ptr() if grad_h else None,
                     dw.data_ptr() if grad_w else None)
        assert run(ctypes.byref(call), work.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert status.item() == fault
        if fault:
            assert torch.isnan(loss) and torch.isnan(rows[live]).all()
            assert not grad_h or torch.isnan(dh[live]).all()
            assert not grad_w or torch.isnan(dw[0, :8]).all()
        else:
            h, w = hidden.clone().requires_grad_(grad_h), weight.clone().requires_grad_(grad_w)
            expected = linear_cross_entropy(h, w, targets)
            assert torch.equal(loss, expected.detach())
            wanted = [(h, dh)] * grad_h + [(w, dw)] * grad_w
            for (_, got), grad in zip(wanted, torch.autograd.grad(expected, [t for t, _ in wanted]) if wanted else ()):
                assert torch.equal(got, grad)


@cuda
def test_top_log_probs_from_two_threads():
    """Records of different lengths at once: a launch's shared memory is not what the other thread last asked for."""
    from rwkv_theseus_b200.ops import native
    run = ctypes.CDLL(native().__file__).rt_top_log_probs
    long, pointer = ctypes.c_long, ctypes.c_void_p
    run.argtypes = [ctypes.c_int, pointer, long, long, long, ctypes.c_int, ctypes.c_float] + [pointer] * 4
    V = 32003
    logits = torch.randn(2, V, device="cuda")
    codes = {}

    def call(k):
        values = torch.empty(2, k, device="cuda")
        index = torch.empty(2, k, device="cuda", dtype=torch.int64)
        stream = torch.cuda.Stream()
        codes[k] = {run(0, logits.data_ptr(), 2, V, V, k, 1.0, values.data_ptr(), index.data_ptr(), None,
                        stream.cuda_stream) for _ in range(3000)}
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=call, args=(k,)) for k in (200, 1024)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert codes == {200: {0}, 1024: {0}}


@cuda
def test_forward_mode_derivatives_are_refused():
    """A tangent is not dropped without a word, whether or not the tensor also wants a gradient."""
    hidden, weight, targets, _ = _inputs(5, 300, 64)
    with forward_ad.dual_level():
        h, w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (hidden, weight))
        learning = forward_ad.make_dual(hidden.clone().requires_grad_(), torch.ones_like(hidden))
        for pair in ((h, weight), (hidden, w), (learning, weight)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                linear_cross_entropy(*pair, targets)
        with pytest.raises(RuntimeError, match="forward-mode"):
            top_log_probs(h, 3)
    assert torch.isfinite(linear_cross_entropy(hidden, weight, targets))


@cuda
@pytest.mark.parametrize("T", [4, 150])
@pytest.mark.parametrize("C", [64, 5120])
def test_logits_without_rounding(T, C):
    """One-hot hidden states: each logit is one product and zeros, so the tensor cores round nothing, and what undoes
    their rounding elsewhere (C / 16 x 2^-26 of a logit) is all of the error but for fp32's: the scale's two roundings
    and the result's (4 x 2^-24 of a logit), and the sum of exponentials (2^-22 each, at most 70 additions of a thread)."""
    g = torch.Generator(device="cuda").manual_seed(C)
    weight = (torch.randn(700, C, device="cuda", generator=g)).to(torch.bfloat16)
    hidden = torch.zeros(T, C, device="cuda", dtype=torch.bfloat16)
    hidden[torch.arange(T, device="cuda"), torch.randint(0, C, (T,), device="cuda", generator=g)] = 10.0
    targets = torch.randint(0, 700, (T,), device="cuda", generator=g)
    z = hidden.double() @ weight.double().t()
    expected = torch.nn.functional.cross_entropy(z, targets, reduction="none")
    got = linear_cross_entropy(hidden, weight, targets, reduction="none").double()
    bound = z.abs().max().item() * (C // 16 * 2.0 ** -26 + 4 * 2.0 ** -24) + 2.0 ** -22 + 70 * 2.0 ** -24
    assert ((got - expected).abs() <= bound).all(), ((got - expected).abs().max().item(), bound)


@cuda
@pytest.mark.parametrize("T", [96, 300])
@pytest.mark.parametrize("K,tail", [(0, False), (8, False), (8, True)])
def test_the_norm_of_the_gradients_errors(T, K, tail):
    """What the logits' gradient, rounded to bf16 once, and a rounded result cost, is what the gradients may be off by:
    the errors' norm against that of the same two roundings in 64 bits, with the 16-bit form of the logits (6.8e-4 of an
    exponential at most, independent of each other) beside it, and a tenth for the sample."""
    hidden, weight, targets, g = _inputs(T, 2000, 256)
    log_probs, index = (None, targets[:, None]) if K == 0 else _record(hidden, weight, K, 1.0, g)
    _, dz, _ = _oracle(hidden, weight, index, log_probs, -100, 1.0, tail)
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    loss = (linear_cross_entropy(h, w, targets, reduction="sum") if K == 0 else
            linear_topk_kl(h, w, index, log_probs, tail=tail, reduction="sum"))
    x, W, rounded = hidden.double(), weight.double(), dz.to(torch.bfloat16).double()
    for got, exact, once, spread in zip(
            torch.autograd.grad(loss, (h, w)), (dz @ W, dz.t() @ x), (rounded @ W, rounded.t() @ x),
            (dz.square() @ W.square(), dz.square().t() @ x.square())):
        allowed = (once.to(torch.bfloat16).double() - exact).norm().square() + 6.8e-4 ** 2 * spread.sum()
        assert (got.double() - exact).norm() <= 1.1 * allowed.sqrt()


@cuda
@pytest.mark.parametrize("T", [300, 1100])
def test_the_weights_gradient_alone(T):
    """What tuning a head asks for, in tiles of rows: with the gradient of the hidden states the same bits."""
    hidden, weight, targets, g = _inputs(T, 1500, 136)
    targets[: T // 4] = -100
    log_probs, index = _record(hidden, weight, 12, 1.0, g)
    for call in (lambda h, w: linear_cross_entropy(h, w, targets),
                 lambda h, w: linear_topk_kl(h, w, index, log_probs)):
        w = weight.clone().requires_grad_()
        alone = torch.autograd.grad(call(hidden, w), w)[0]
        h = hidden.clone().requires_grad_()
        assert torch.equal(alone, torch.autograd.grad(call(h, w), (h, w))[1])
    _, dz, valid = _oracle(hidden, weight, index, log_probs, -100, 1.0, True)
    dz, x = dz / valid.sum(), hidden.double()
    xmax, wmax = (t.float().norm(dim=-1).max().item() for t in (hidden, weight))
    tol = 3 * U + 4 * (136 / 16 + 16) * 2.0 ** -23 * xmax * wmax
    _within(alone, dz.t() @ x, tol * (dz.abs().t() @ x.abs()))


@cuda
@pytest.mark.parametrize("T", [70, 300])
def test_both_losses_in_one_graph(T):
    """A weighted sum of the two, as head tuning forms it: each gradient is rounded once more for its factor, and their
    sum once."""
    hidden, weight, targets, g = _inputs(T, 1500, 136)
    targets[::5] = -100
    log_probs, index = _record(hidden, weight, 12, 2.0, g)
    index[::3] = -1
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    loss = 0.3 * linear_topk_kl(h, w, index, log_probs, 2.0) + 0.7 * linear_cross_entropy(h, w, targets)
    grads = torch.autograd.grad(loss, (h, w))
    x, W = hidden.double(), weight.double()
    xmax, wmax = (t.norm(dim=-1).max().item() for t in (x, W))
    err = (136 / 16 + 16) * 2.0 ** -23 * xmax * wmax
    expected, bound, value = [0, 0], [0, 0], 0
    parts = ((0.3, index, log_probs, 0.5, True), (0.7, targets[:, None], None, 1.0, False))
    for factor, ids, logp, scale, tail in parts:
        rows, dz, valid = _oracle(hidden, weight, ids, logp, -100, scale, tail)
        value += factor * rows.sum() / valid.sum()
        dz = dz * (factor * scale / valid.sum())
        for i, (a, b) in enumerate(((dz, W), (dz.t(), x))):
            expected[i] = expected[i] + a @ b
            bound[i] = bound[i] + (4 * U + 4 * err) * (a.abs() @ b.abs())
    torch.testing.assert_close(loss.detach().double(), value, rtol=1e-5, atol=2 * err + 1e-6)
    for got, e, b in zip(grads, expected, bound):
        _within(got, e, b + U * (e.abs() + b))


@cuda
@pytest.mark.parametrize("T,live", [(40, 30), (300, 255), (33000, 32640)])
@pytest.mark.parametrize("K,reduction", [(0, "mean"), (0, "none"), (4, "mean")])
def test_a_factor_of_all_rows_is_not_rounded(T, live, K, reduction):
    """1 / live is 0.23 to 0.39% off in bf16. It is no part of the logits' gradient, whose rounding (of the rows before
    any factor) is what the gradients' errors in norm may come from, as above."""
    hidden, weight, targets, g = _inputs(T, 300, 64)
    dropped = torch.randperm(T, device="cuda", generator=g)[:T - live]
    temperature = 1.0
    if K == 0:
        targets[dropped] = -100
        log_probs, index = None, targets[:, None]
    else:
        temperature = 0.7
        log_probs, index = _record(hidden, weight, K, temperature, g)
        index[dropped] = -1
    _, dz, _ = _oracle(hidden, weight, index, log_probs, -100, 1.0 / temperature, True)
    factor = 1.0 / temperature / live
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    loss = (linear_cross_entropy(h, w, targets, reduction=reduction) if K == 0 else
            linear_topk_kl(h, w, index, log_probs, temperature))
    if reduction == "none":
        loss = loss.sum() / live
    x, W, rounded = hidden.double(), weight.double(), dz.to(torch.bfloat16).double()
    for got, exact, once, spread in zip(
            torch.autograd.grad(loss, (h, w)), (dz @ W, dz.t() @ x), (rounded @ W, rounded.t() @ x),
            (dz.square() @ W.square(), dz.square().t() @ x.square())):
        exact, once = exact * factor, once * factor
        allowed = (once.to(torch.bfloat16).double() - exact).norm().square() + (6.8e-4 * factor) ** 2 * spread.sum()
        assert (got.double() - exact).norm() <= 1.1 * allowed.sqrt()
