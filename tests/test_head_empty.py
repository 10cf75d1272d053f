"""No rows at all: the loss is 0 (a mean NaN, 0 / 0) and both gradients are there, of zeros."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import linear_cross_entropy, linear_distillation
from mamba_metal.head import _no_rows

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def zeros(loss, x, w, reduction):
    assert loss.dtype == torch.float32
    assert loss.shape == ((2, 0) if reduction == "none" else ())
    assert torch.isnan(loss) if reduction == "mean" else (loss == 0).all()
    for grad, of in zip(torch.autograd.grad(loss.sum(), [x, w]), (x, w)):
        assert grad.shape == of.shape and grad.dtype == of.dtype and (grad == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows(dtype, reduction, device):
    x = torch.zeros(2, 0, 8, dtype=dtype, device=device, requires_grad=True)
    w = torch.ones(5, 8, dtype=dtype, device=device, requires_grad=True)
    target = torch.zeros(2, 0, dtype=torch.int64, device=device)
    index, logits = torch.zeros(2, 0, 3, dtype=torch.int64, device=device), torch.zeros(2, 0, 3, device=device)
    zeros(linear_cross_entropy(x, w, target, reduction=reduction), x, w, reduction)
    zeros(linear_distillation(x, w, index, logits, reduction=reduction), x, w, reduction)
    zeros(_no_rows(x, w, (2, 0), reduction), x, w, reduction)       # the kernels' stand-in, here on any device
    # one gradient alone, and none
    alone = linear_cross_entropy(x.detach(), w, target, reduction=reduction)
    assert (torch.autograd.grad(alone.sum(), w)[0] == 0).all()
    with torch.no_grad():
        assert not linear_cross_entropy(x, w, target, reduction=reduction).requires_grad
