"""A vocabulary row far above the rest: float32 products keep 2^-39 of w's largest element.

w is scaled as a whole for its two fp16 parts (22 bits down to 2^-16 of the largest element, below
that an absolute 2^-39 of it), so one large row takes bits from the others. The bounds of
_head_ref.py count that (FOOT times the largest); bf16 rows stay exact down to 2^-31 of the largest.
x has no part along the large row's only column, so that its logits stay those of the others.
"""
from __future__ import annotations

import pytest
import torch

from _head_ref import sparse
from test_head_cuda import BF16, F32, head_inputs, run_ce

import _head_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [5, 40, 400])
@pytest.mark.parametrize("power", [12, 16, 20])
def test_one_large_row(power, rows, dtype):
    x, w, target, gen = head_inputs(rows, 500, 96, dtype, seed=power + rows)
    x[:, 11] = 0
    w[33] = 0
    w[33, 11] = 2.0 ** power
    target[target == 33] = 34
    loss, grads = run_ce(x, w, target, "mean", torch.tensor(1.0))
    want = _head_ref.solve(x, w, *sparse(1, target=target, ignore=-100), 1.0, "mean", torch.tensor(1.0))
    _head_ref.check("loss", loss, want["loss"], want["e_loss"])
    for name, got in zip(("dx", "dw"), grads):
        _head_ref.check(name, got, want[name], want["e_" + name])
    # column 11 of dx is dz[33] times the large element, which its sum holds to the type
    keep = torch.arange(96) != 11
    if power <= 16:                             # 22 bits still: norms as for any other weight
        tol = 2.0 ** -7 if dtype == BF16 else 2e-5
        _head_ref.check_norm("dx", grads[0].cpu()[:, keep], want["dx"][:, keep], tol)
        _head_ref.check_norm("dw", grads[1], want["dw"], tol)
