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

from rwkv_theseus_b200.losses import linear_cross_entropy, top_log_probs
from test_head_losses_gpu import U, _check, _inputs, _record

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
