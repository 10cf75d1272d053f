"""What the head's losses and the residual norm allocate does not follow torch.set_default_dtype.

The kernels write float32 whatever the default is: a buffer of another type would be too small
or read as something else. On the CPU a stand-in for the library looks at the buffers (nothing is
launched); on the GPU every result equals the one under the default float32 to the bit.
"""
from __future__ import annotations

import contextlib

import pytest
import torch

from mamba_metal import _native, linear_cross_entropy, linear_distillation, residual_rms_norm

DEFAULTS = [torch.bfloat16, torch.float64]


@contextlib.contextmanager
def default_dtype(dtype):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        yield
    finally:
        torch.set_default_dtype(before)


class NoLaunch:
    """Sizes of 256 bytes; every other entry returns MMS_OK and does nothing."""

    def __getattr__(self, name):
        return lambda *args: 256 if name.endswith("_size") else 0


@pytest.mark.parametrize("default", DEFAULTS)
def test_buffers_are_float32(default, monkeypatch):
    monkeypatch.setattr(_native, "load", NoLaunch)
    monkeypatch.setattr(_native, "_stream", lambda device: 0)
    _native._head_sizes.cache_clear()
    x, w = torch.zeros(5, 8), torch.zeros(9, 8)
    index, logits = torch.zeros(5, 3, dtype=torch.int64), torch.zeros(5, 3)
    try:
        with default_dtype(default):
            made = [_native.linear_ce_fwd(x, w, index[:, 0], -100, r)[0] for r in ("none", "mean", "sum")]
            made += [_native.linear_kd_fwd(x, w, index, logits, 1.0, r)[0] for r in ("none", "mean", "sum")]
            made.append(_native.norm_fwd(x, x, None, w[0], None, None, 1e-6)[2])
    finally:
        _native._head_sizes.cache_clear()
    assert [t.dtype for t in made] == [torch.float32] * 7


@pytest.mark.gpu
def test_the_probe_writes_within_its_buffer():
    with default_dtype(torch.float16):
        assert _native.pipe_rate("ffma", iters=64) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 40, 600])
@pytest.mark.parametrize("default", DEFAULTS)
def test_results_do_not_follow_the_default(default, rows, dtype):
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 72, generator=gen, dtype=torch.float32).to(dtype).cuda()
    w = torch.randn(300, 72, generator=gen, dtype=torch.float32).to(dtype).cuda()
    target = torch.randint(0, 300, (rows,), generator=gen).cuda()
    index = torch.randint(-1, 300, (rows, 4), generator=gen).cuda()
    logits = torch.randn(rows, 4, generator=gen, dtype=torch.float32).cuda()

    def calls():
        out = []
        for reduction in ("none", "mean", "sum"):
            for loss_of in (lambda a, b: linear_cross_entropy(a, b, target, reduction=reduction),
                            lambda a, b: linear_distillation(a, b, index, logits, 2.0, reduction=reduction)):
                a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
                loss = loss_of(a, b)
                out += [loss.detach(), *torch.autograd.grad(loss, [a, b], torch.ones_like(loss))]
                with torch.no_grad():
                    out.append(loss_of(a, b))
        a, b = x.clone().requires_grad_(True), w[0].clone().requires_grad_(True)
        h, u = residual_rms_norm(a, x, b, gate=x, scale=w[1])
        return out + [h.detach(), u.detach(), *torch.autograd.grad([h, u], [a, b], [x, x])]

    want = calls()
    with default_dtype(default):
        got = calls()
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(want, got))
    assert all(t.dtype == torch.float32 for t in got[:24:4])
