"""Vocabulary-head losses on CPU: the plain definitions against 64-bit formulas and against differences, their masks,
and the refusals of the public functions."""
import math

import pytest
import torch
from torch.nn import functional as F

from rwkv_theseus_b200.losses import linear_cross_entropy, linear_topk_kl, top_log_probs


def _problem(T=7, V=23, C=8, K=4, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    hidden = torch.randn(T, C, generator=g, dtype=torch.float64).to(dtype)
    weight = torch.randn(V, C, generator=g, dtype=torch.float64).to(dtype)
    teacher = torch.randn(T, V, generator=g, dtype=torch.float64)
    targets = torch.randint(0, V, (T,), generator=g)
    return hidden, weight, teacher, targets


def _kl(hidden, weight, indices, log_probs, temperature, tail):
    """Row by row from the definition: KL between the two distributions over the record (and the rest)."""
    log_q = torch.log_softmax(hidden @ weight.t() / temperature, -1)
    rows = []
    for t in range(len(hidden)):
        kept = indices[t] >= 0
        if not kept.any():
            rows.append(log_q.new_zeros(()))
            continue
        inside = indices[t][kept]
        p = log_probs[t][kept].exp()
        loss = (p * (log_probs[t][kept] - log_q[t, inside])).sum()
        outside = [v for v in range(weight.shape[0]) if v not in inside.tolist()]
        if tail and outside and p.sum() < 1:
            rest = 1 - p.sum()
            loss = loss + rest * (rest.log() - log_q[t, outside].logsumexp(0))
        rows.append(loss)
    return torch.stack(rows)


def test_cross_entropy_matches_the_formula():
    hidden, weight, _, targets = _problem()
    targets[2] = -100
    expected = F.cross_entropy(hidden @ weight.t(), targets, reduction="none")
    for reduction, value in (("none", expected), ("sum", expected.sum()), ("mean", expected.sum() / 6)):
        got = linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        torch.testing.assert_close(got, value, rtol=1e-12, atol=1e-12)
    shaped = linear_cross_entropy(hidden.view(1, 7, 8), weight, targets.view(1, 7).int(), reduction="none")
    assert shaped.shape == (1, 7)
    torch.testing.assert_close(shaped[0], expected, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("K", [1, 4, 23])
def test_topk_kl_matches_the_formula(tail, K):
    hidden, weight, teacher, _ = _problem()
    log_probs, indices = top_log_probs(teacher, K, temperature=2.0)
    indices[3, K // 2:] = -1
    indices[5] = -1
    expected = _kl(hidden, weight, indices, log_probs.double(), 2.0, tail)
    got = linear_topk_kl(hidden, weight, indices, log_probs.double(), 2.0, tail, "none")
    # at K = V the record holds all the mass but for its own rounding, which neither form gives to an empty rest
    torch.testing.assert_close(got, expected, rtol=1e-9, atol=1e-9)
    mean = linear_topk_kl(hidden, weight, indices, log_probs.double(), 2.0, tail)
    torch.testing.assert_close(mean, expected.sum() / (indices >= 0).any(-1).sum(), rtol=1e-9, atol=1e-9)


@pytest.mark.parametrize("tail", [False, True])
def test_gradients_match_differences(tail):
    hidden, weight, teacher, targets = _problem()
    targets[0] = -100
    log_probs, indices = top_log_probs(teacher, 4)
    indices[1, 2:] = -1
    indices[6] = -1
    hidden.requires_grad_()
    weight.requires_grad_()
    assert torch.autograd.gradcheck(lambda h, w: linear_cross_entropy(h, w, targets), (hidden, weight))
    assert torch.autograd.gradcheck(lambda h, w: linear_topk_kl(h, w, indices, log_probs, 1.5, tail, "none"),
                                    (hidden, weight))


def test_a_full_record_is_the_full_kl():
    hidden, weight, teacher, _ = _problem()
    log_probs, indices = top_log_probs(teacher, 23)
    log_q, log_p = torch.log_softmax(hidden @ weight.t(), -1), torch.log_softmax(teacher, -1)
    torch.testing.assert_close(linear_topk_kl(hidden, weight, indices, log_probs, tail=False, reduction="sum"),
                               (log_p.exp() * (log_p - log_q)).sum(), rtol=1e-9, atol=1e-9)


def test_rows_without_an_entry_and_entries_without_mass():
    hidden, weight, teacher, targets = _problem()
    assert linear_cross_entropy(hidden, weight, torch.full_like(targets, -1), ignore_index=-1).item() == 0.0
    none = torch.full((7, 3), -1)
    assert linear_topk_kl(hidden, weight, none, torch.zeros(7, 3, dtype=torch.float64)).item() == 0.0
    log_probs, indices = top_log_probs(teacher, 4)
    log_probs[:, 3] = -math.inf  # recorded, but without mass: leaves the rest's class, adds no term
    got = linear_topk_kl(hidden, weight, indices, log_probs, reduction="none")
    torch.testing.assert_close(got, _kl_without_mass(hidden, weight, indices, log_probs), rtol=1e-9, atol=1e-9)


def _kl_without_mass(hidden, weight, indices, log_probs):
    log_q = torch.log_softmax(hidden @ weight.t(), -1)
    p = log_probs.exp()
    loss = (p[:, :3] * (log_probs[:, :3] - log_q.gather(1, indices[:, :3]))).sum(-1)
    rest = 1 - p.sum(-1)
    outside = log_q.scatter(1, indices, -math.inf).logsumexp(-1)
    return loss + rest * (rest.log() - outside)


def test_top_log_probs_takes_equal_logits_by_index():
    logits = torch.tensor([[1.0, 3.0, 3.0, -math.inf, 3.0, 0.0, -0.0], [2.0] * 7])
    log_probs, indices = top_log_probs(logits, 5)
    assert indices.tolist() == [[1, 2, 4, 0, 5], [0, 1, 2, 3, 4]]
    torch.testing.assert_close(log_probs, torch.log_softmax(logits, -1).gather(1, indices))
    assert top_log_probs(logits.view(1, 2, 7), 3, temperature=0.5)[1].shape == (1, 2, 3)


def test_refusals():
    hidden, weight, teacher, targets = _problem()
    log_probs, indices = top_log_probs(teacher, 4)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(hidden, weight, targets, reduction="max")
    with pytest.raises(ValueError, match="hidden"):
        linear_cross_entropy(hidden[:, :5], weight, targets)
    with pytest.raises(ValueError, match="do not match"):
        linear_cross_entropy(hidden, weight, targets[:3])
    with pytest.raises(TypeError, match="int32 or int64"):
        linear_cross_entropy(hidden, weight, targets.float())
    with pytest.raises(ValueError, match="do not match"):
        linear_cross_entropy(hidden, weight, indices)
    with pytest.raises(IndexError):
        linear_cross_entropy(hidden, weight, targets + 23)
    with pytest.raises(IndexError):
        linear_cross_entropy(hidden, weight, torch.full_like(targets, -5))
    with pytest.raises(ValueError, match="log_probs"):
        linear_topk_kl(hidden, weight, indices, log_probs[:, :2])
    with pytest.raises(ValueError, match="1 to 1024"):
        linear_topk_kl(hidden, weight, indices[:, :0], log_probs[:, :0])
    with pytest.raises(TypeError, match="floating"):
        linear_topk_kl(hidden, weight, indices, indices)
    with pytest.raises(ValueError, match="temperature"):
        linear_topk_kl(hidden, weight, indices, log_probs, temperature=0.0)
    with pytest.raises(IndexError):
        linear_topk_kl(hidden, weight, indices + 23, log_probs)
    for k in (0, 24):
        with pytest.raises(ValueError, match="k must be"):
            top_log_probs(teacher, k)
    with pytest.raises(ValueError, match="temperature"):
        top_log_probs(teacher, 2, temperature=-1.0)


def test_c_entries_refuse_before_any_cuda_call():
    """Sizes, counts and alignments out of range return cudaErrorInvalidValue; stand-in addresses are never used."""
    import ctypes
    import glob
    from pathlib import Path
    found = glob.glob(str(Path(__file__).resolve().parents[1] / "rwkv_theseus_b200" / "_C*.so"))
    if not found:
        pytest.skip("extension not built")
    lib = ctypes.CDLL(found[0])
    vp, lg, it, fl = ctypes.c_void_p, ctypes.c_long, ctypes.c_int, ctypes.c_float
    lib.rt_top_log_probs.argtypes = [it, vp, lg, lg, lg, it, fl, vp, vp, vp, vp]
    lib.rt_top_workspace_bytes.argtypes, lib.rt_top_workspace_bytes.restype = [it, lg, lg, it], lg
    lib.rt_head_loss.argtypes = [vp, vp, vp]
    lib.rt_scale_bf16.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(lg), vp, vp]
    good = 0x10000

    def top(rows=4, V=100, k=5, work=good):
        return lib.rt_top_log_probs(1, good, rows, V, V, k, 1.0, good, good, work, None)

    assert top(k=0) == top(k=101) == top(k=1025, V=5000) == top(V=0) == top(rows=-1) == 1
    assert top(rows=0) == 0
    assert top(rows=1, V=1 << 22, work=None) == 1                     # cut into segments, which need their workspace
    assert top(rows=1, V=1 << 24, k=1024) == 1 and lib.rt_top_workspace_bytes(1, 1, 1 << 24, 1024) == -1

    class HeadLoss(ctypes.Structure):
        _fields_ = [("hidden", vp), ("ld_hidden", lg), ("weight", vp), ("ld_weight", lg), ("index", vp),
                    ("log_probs", vp), ("rows", lg), ("vocab", lg), ("width", it), ("K", it), ("ignore", lg),
                    ("scale", fl), ("tail", it), ("reduction", it), ("row_grad", vp), ("row_loss", vp), ("loss", vp),
                    ("dhidden", vp), ("dweight", vp)]

    def head(work=good, **changes):
        call = HeadLoss(hidden=good, ld_hidden=64, weight=good, ld_weight=64, index=good, rows=4, vocab=100, width=64,
                        K=1, ignore=-100, scale=1.0, row_loss=good)
        for name, value in changes.items():
            setattr(call, name, value)
        return lib.rt_head_loss(ctypes.byref(call), work, None)

    assert lib.rt_head_loss(None, good, None) == 1 and head(work=None) == 1 and head(work=good + 8) == 1
    for changes in (dict(rows=-1), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=2 ** 31), dict(width=60),
                    dict(K=0), dict(K=2), dict(K=1025, log_probs=good), dict(ld_hidden=60), dict(ld_weight=60),
                    dict(hidden=None), dict(weight=None), dict(hidden=good + 2), dict(weight=good + 8),
                    dict(dhidden=good + 4), dict(dweight=good + 2)):
        assert head(**changes) == 1, changes
    assert head(rows=0) == 0                                           # no reduction, no weight gradient: nothing to do
    assert lib.rt_scale_bf16((vp * 2)(good + 2, None), (lg * 2)(8, 0), good, None) == 1
    assert lib.rt_scale_bf16((vp * 2)(None, None), (lg * 2)(0, 0), good, None) == 0
