"""The losses' PyTorch path keeps what the functions promise: left-out rows may hold anything, indices
outside the vocabulary are loud, nothing left to count has gradients of 0. On the CPU, and the same
calls on the GPU (where an index out of range must not reach a PyTorch kernel's assertion)."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import linear_cross_entropy, linear_distillation

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NAN = float("nan")


def problem(device, lead=(6,)):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(*lead, 8, generator=gen)
    w = torch.randn(12, 8, generator=gen)
    target = torch.randint(0, 12, lead, generator=gen)
    index = torch.randint(0, 12, (*lead, 3), generator=gen)
    logits = torch.randn(*lead, 3, generator=gen)
    return [t.to(device) for t in (x, w, target, index, logits)]


def run(loss_of, x, w):
    x, w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = loss_of(x, w)
    dx, dw = torch.autograd.grad(loss, [x, w], torch.ones_like(loss))
    return loss.detach(), dx, dw


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("value", [NAN, float("inf")])
def test_left_out_rows_may_hold_anything(value, reduction, device):
    x, w, target, index, logits = problem(device, (2, 3))
    target[0, 1], index[0, 1], logits[1, 2] = -100, -1, float("-inf")
    for out, loss_of in (((0, 1), lambda a, b: linear_cross_entropy(a, b, target, reduction=reduction, impl="torch")),
                         ((0, 1), lambda a, b: linear_distillation(a, b, index, logits, 2.0, reduction, impl="torch")),
                         ((1, 2), lambda a, b: linear_distillation(a, b, index, logits, 2.0, reduction, impl="torch"))):
        want = run(loss_of, x, w)
        y = x.clone()
        y[out] = value
        got = run(loss_of, y, w)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert (got[1][out] == 0).all() and torch.isfinite(got[2]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_counts(reduction, device):
    x, w, target, index, logits = problem(device)
    target[:], index[:] = -100, -1
    for loss_of in (lambda a, b: linear_cross_entropy(a, b, target, reduction=reduction, impl="torch"),
                    lambda a, b: linear_distillation(a, b, index, logits, 2.0, reduction, impl="torch")):
        loss, dx, dw = run(loss_of, x, w)
        assert torch.isnan(loss) if reduction == "mean" else (loss == 0).all()
        assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [12, 1 << 40])
def test_indices_outside_the_vocabulary(bad, device):
    x, w, target, index, logits = problem(device)
    target[2], index[2, 1] = bad, bad
    cases = [lambda a, b: linear_cross_entropy(a, b, target, reduction="none", impl="torch"),
             lambda a, b: linear_distillation(a, b, index, logits, 2.0, "none", impl="torch")]
    if bad == 12:
        below = target.clone()
        below[2] = -5
        cases.append(lambda a, b: linear_cross_entropy(a, b, below, reduction="none", impl="torch"))
    rest = torch.arange(6, device=device) != 2
    for loss_of in cases:
        loss, dx, dw = run(loss_of, x, w)
        assert torch.isnan(loss[2]) and torch.isfinite(loss[rest]).all()
        assert torch.isnan(dx[2]).all() and torch.isfinite(dx[rest]).all() and torch.isnan(dw).all()
    logits[2, 1] = float("-inf")                        # probability 0: counts for nothing
    assert all(torch.isfinite(t).all() for t in run(cases[1], x, w))


def test_flat_targets_beside_a_batch():
    x, w, target, *_ = problem("cpu", (2, 3))
    assert torch.equal(linear_cross_entropy(x, w, target.reshape(-1)), linear_cross_entropy(x, w, target))
