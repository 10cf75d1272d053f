"""sample_tokens in PyTorch ops: the steps one by one, ties, masks, refusals."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from mamba_metal import _native, sample_tokens

INF = float("inf")


def draw(z, u, **kw):
    return sample_tokens(torch.tensor([z]), torch.tensor([u]), **kw).item()


def test_the_steps():
    z = [0.0, math.log(2.0), math.log(4.0), math.log(1.0)]            # weights 1, 2, 4, 1
    assert [draw(z, u) for u in (0.0, 0.12, 0.13, 0.37, 0.38, 0.87, 0.88, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [draw(z, u, top_k=2) for u in (0.0, 0.32, 0.34, 0.99)] == [1, 1, 2, 2]
    assert {draw(z, u, top_p=0.45) for u in (0.0, 0.5, 0.99)} == {2}            # 4 of 8 is enough
    assert [draw(z, u, top_p=0.55) for u in (0.0, 0.99)] == [1, 2]
    assert [draw(z, u, top_k=3, top_p=0.99) for u in (0.0, 0.99)] == [0, 2]    # of equal ones the lower index
    assert [draw(z, u, min_p=0.4) for u in (0.0, 0.99)] == [1, 2]
    assert {draw(z, u, min_p=7.0) for u in (0.0, 0.99)} == {2}
    assert {draw(z, u, temperature=0.0) for u in (0.0, 0.99)} == {2}
    assert [draw(z, u, temperature=1e9) for u in (0.24, 0.26, 0.74, 0.76)] == [0, 1, 2, 3]
    token, lp = sample_tokens(torch.tensor([z]), torch.tensor([0.9]), top_k=3, return_logprob=True)
    assert token.item() == 2 and abs(lp.item() - math.log(4 / 7)) < 1e-6


def test_masks_ties_and_rows_without_anything():
    assert draw([-INF, 1.0, -INF], 0.7) == 1 and draw([-INF] * 3, 0.5) == -1 and draw([0.0, float("nan")], 0.5) == -1
    assert [draw([3.0] * 4, u, top_k=2) for u in (0.0, 0.99)] == [0, 1]
    assert [draw([3.0] * 4, u, top_p=0.5) for u in (0.0, 0.99)] == [0, 1]
    assert [draw([0.0, INF, 5.0, INF], u) for u in (0.0, 0.6)] == [1, 3]
    low = torch.finfo(torch.float32).min
    assert draw([low, low, 0.0], 0.999) == 2 and draw([low, low], 0.7) == 1
    assert draw([0.0, 1.0], 1.0) == 1 and draw([0.0, 1.0], -1.0) == 0
    token, lp = sample_tokens(torch.full((1, 2), -INF), torch.tensor([0.5]), return_logprob=True)
    assert token.item() == -1 and math.isnan(lp.item())


def test_settings_of_each_rows_own():
    z = torch.randn(2, 3, 50)
    u = torch.rand(2, 3)
    t, k, p, m = torch.rand(2, 3) + 0.5, torch.tensor([[0, 1, 2], [3, 4, 100]]), torch.rand(2, 3), 0.1 * torch.rand(2, 3)
    got = sample_tokens(z, u, t, k, p, m)
    assert got.shape == (2, 3) and got.dtype == torch.int64
    for i in range(2):
        for j in range(3):
            assert got[i, j] == sample_tokens(z[i, j], u[i, j], float(t[i, j]), int(k[i, j]), float(p[i, j]), float(m[i, j]))


def test_refusals():
    z, u = torch.randn(3, 5), torch.rand(3)
    for kw in (dict(uniform=u[:2]), dict(logits=z[:, :0]), dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.1), dict(min_p=-0.1),
               dict(temperature=float("nan")), dict(top_k=torch.tensor([1, 2])), dict(top_p=torch.rand(3, 1)), dict(impl="nonsense")):
        with pytest.raises(ValueError):
            sample_tokens(**{"logits": z, "uniform": u, **kw})
    for kw in (dict(logits=z.long()), dict(uniform=u.long()), dict(top_k=torch.rand(3)), dict(impl="cuda")):
        with pytest.raises(RuntimeError):
            sample_tokens(**{"logits": z, "uniform": u, **kw})


def test_the_c_interface_refuses_before_a_launch():
    lib = _native.load()
    p, odd = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10004)

    def call(z=p, u=p, k=None, wide=0, token=p, rows=1, vocab=5, dtype=0, ld=5):
        return lib.mms_sample(z, ld, u, None, 1.0, k, wide, 0, None, 1.0, None, 0.0, token, None, rows, vocab, dtype, None)

    assert [call(z=None), call(u=None), call(token=None), call(rows=0), call(vocab=0), call(dtype=3), call(ld=-1),
            call(rows=(1 << 24) + 1)] == [_native.MMS_ERR_INVALID_ARG] * 8
    assert call(token=odd) == call(k=odd, wide=1) == call(z=ctypes.c_void_p(0x10002)) == _native.MMS_ERR_MISALIGNED
