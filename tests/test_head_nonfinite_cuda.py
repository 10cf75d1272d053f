"""Infinities, NaN and indices outside the vocabulary in rows that count: loud there, nowhere else.

On every path of the head's losses: the CUDA cores (2 rows), the tensor cores (40), left-out rows
listed (600). Losses and dx of the other rows are what they are without the bad ones, to the bit
where nothing of theirs is scaled by them; dw, a sum over the rows, is NaN as PyTorch's.
"""
from __future__ import annotations

import pytest
import torch

from mamba_metal import linear_cross_entropy, linear_distillation
from test_head_cuda import BF16, DEV, F32, head_inputs, leaves

pytestmark = pytest.mark.gpu
VOCAB, DIM, K = 300, 72, 5


def problem(rows, dtype, kd):
    x, w, target, gen = head_inputs(rows, VOCAB, DIM, dtype, seed=rows)
    if kd:
        index = torch.randint(0, VOCAB, (rows, K), generator=gen)
        return x, w, index, torch.randn(rows, K, generator=gen)
    return x, w, target, None


def run(x, w, index, logits, reduction):
    xd, wd = leaves(x, w)
    if logits is None:
        loss = linear_cross_entropy(xd, wd, index.to(DEV), reduction=reduction)
    else:
        loss = linear_distillation(xd, wd, index.to(DEV), logits.to(DEV), 2.0, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, [xd, wd], torch.ones_like(loss))
    return loss.detach().cpu(), dx.cpu(), dw.cpu()


def only(bad, clean, got, reduction):
    loss, dx, dw = got
    if reduction == "none":
        assert torch.equal(torch.isnan(loss), bad) and torch.equal(loss[~bad], clean[0][~bad])
    else:
        assert torch.isnan(loss)
    assert torch.isnan(dx[bad]).all() and torch.equal(dx[~bad], clean[1][~bad])
    assert torch.isnan(dw).all()


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("kd", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [2, 40, 600])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_values_of_x(value, rows, dtype, kd, reduction):
    x, w, index, logits = problem(rows, dtype, kd)
    clean = run(x, w, index, logits, reduction)
    bad = torch.arange(rows) % 7 == 1
    x = x.clone()
    x[bad, 5] = value
    only(bad, clean, run(x, w, index, logits, reduction), reduction)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [2, 40, 600])
def test_a_nan_in_w_reaches_every_row(rows, dtype):
    for kd in (False, True):
        x, w, index, logits = problem(rows, dtype, kd)
        w = w.clone()
        w[7, 3] = float("nan")
        loss, dx, dw = run(x, w, index, logits, "none")
        assert torch.isnan(loss).all() and torch.isnan(dx).all() and torch.isnan(dw).all()


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [2, 40, 600])
@pytest.mark.parametrize("at", [VOCAB, 1 << 31, 1 << 40])
def test_list_entries_outside_the_vocabulary(at, rows, dtype, reduction):
    x, w, index, logits = problem(rows, dtype, True)
    bad = torch.arange(rows) % 7 == 1
    out = index.clone()
    out[bad, 2] = at
    loss, dx, dw = run(x, w, out, logits, reduction)
    assert torch.equal(torch.isnan(loss), bad) if reduction == "none" else torch.isnan(loss)
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all() and torch.isnan(dw).all()
    # an entry of probability 0 there counts for nothing
    logits = logits.clone()
    logits[bad, 2] = float("-inf")
    loss, dx, dw = run(x, w, out, logits, reduction)
    assert torch.isfinite(loss).all() and torch.isfinite(dx).all() and torch.isfinite(dw).all()
