"""How near the head's bf16 gradients come to float64, beside their own rounding.

A bf16 gradient cannot be nearer than its last rounding, whose norm R is known from float64's
values. What the kernels may add above 256 rows is dz in scaled fp16: at most
u = 2^-11 of each value, each value's rounding its own, so at most u of the norms of the terms
dz_v w_v (dx) and dz_m x_m (dw) as independent errors, whose squares add up: the terms' norms
are computed below. The float32 sums (2^-24 a step) disappear beside both, as does the
1 % by which rounding the value beside it (not the value) may differ in norm over the tens of
thousands of elements here (their mean square spreads by less than 1 / sqrt(10^4)).
"""
from __future__ import annotations

import math

import pytest
import torch

from mamba_metal import linear_cross_entropy, linear_distillation
from test_head_cuda import BF16, DEV, head_inputs, leaves

pytestmark = pytest.mark.gpu
U16 = 2.0 ** -11


def gradients64(x, w, index, p, r):
    """dx, dw and the norms of their terms in float64, for dz = r (q - p)."""
    x, w = x.double(), w.double()
    dz = torch.softmax(x @ w.t(), 1) * p.sum(1, keepdim=True)
    dz = dz.scatter_add(1, index, -p) * r[:, None]
    sq = dz.pow(2)
    terms = (float((sq.sum(0) * w.pow(2).sum(1)).sum().sqrt()), float((sq.sum(1) * x.pow(2).sum(1)).sum().sqrt()))
    return (dz @ w, dz.t() @ x), terms


def held(got, want, terms):
    for name, g, v, t in zip(("dx", "dw"), got, want, terms):
        own = float((v.to(BF16).double() - v).norm())
        off = float((g.cpu().double() - v).norm())
        assert off <= 1.01 * math.hypot(own, U16 * t), (name, off / float(v.norm()), own / float(v.norm()))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows", [200, 257, 600])
def test_cross_entropy_gradients_are_rounded_once(rows, reduction):
    x, w, target, gen = head_inputs(rows, 3001, 200, BF16, seed=rows)
    r = torch.rand(rows, generator=gen) + 0.01 if reduction == "none" else torch.full((rows,), 1.0 / rows)
    xd, wd = leaves(x, w)
    loss = linear_cross_entropy(xd, wd, target.to(DEV), reduction=reduction)
    got = torch.autograd.grad(loss, [xd, wd], r.to(DEV) if reduction == "none" else None)
    held(got, *gradients64(x, w, target[:, None], torch.ones(rows, 1, dtype=torch.float64), r.double()))


@pytest.mark.parametrize("rows", [257, 600])
def test_distillation_gradients_are_rounded_once(rows):
    x, w, _, gen = head_inputs(rows, 3001, 200, BF16, seed=rows + 1)
    index = torch.stack([torch.randperm(3001, generator=gen)[:32] for _ in range(rows)])
    logits = 2 * torch.randn(rows, 32, generator=gen)
    xd, wd = leaves(x, w)
    got = torch.autograd.grad(linear_distillation(xd, wd, index.to(DEV), logits.to(DEV)), [xd, wd])
    p = torch.softmax(logits.double(), 1)
    held(got, *gradients64(x, w, index, p, torch.full((rows,), 1.0 / rows, dtype=torch.float64)))
