"""causal_conv and causal_conv_packed in PyTorch ops: the definition, nn.Conv1d, refusals."""
from __future__ import annotations

import ctypes

import pytest
import torch
import torch.nn.functional as F

from mamba_metal import _native, causal_conv, causal_conv_packed, causal_conv_ref

F64 = torch.float64


@pytest.mark.parametrize("taps", [1, 2, 4, 9])
@pytest.mark.parametrize("length", [1, 3, 20])
@pytest.mark.parametrize("silu", [True, False])
def test_torch_form_is_the_blocks_convolution(length, taps, silu):
    """The block's layers (transposes, padded nn.Conv1d, SiLU) in float64, and their gradients."""
    g = torch.Generator().manual_seed(taps)
    x = torch.randn(2, length, 6, generator=g, dtype=F64, requires_grad=True)
    conv = torch.nn.Conv1d(6, 6, taps, padding=taps - 1, groups=6).double()
    want = conv(x.transpose(1, 2))[:, :, :length].transpose(1, 2)
    want = F.silu(want) if silu else want
    got = causal_conv(x, conv.weight, conv.bias, silu=silu)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    dy = torch.randn(want.shape, generator=g, dtype=F64)
    leaves = [x, conv.weight, conv.bias]
    for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.allclose(a, b, rtol=1e-11, atol=1e-11)


def test_packed_torch_form_is_the_convolution_of_each_sequence():
    g = torch.Generator().manual_seed(0)
    lens, k, d = [5, 0, 1, 2, 9], 4, 3
    x, w, bias = torch.randn(20, d, generator=g, dtype=F64), torch.randn(d, k, generator=g, dtype=F64), torch.randn(d, generator=g, dtype=F64)
    starts = torch.tensor([2] + lens).cumsum(0)
    window = torch.randn(7, d, k - 1, generator=g, dtype=F64)
    before = window.clone()
    slots, out = torch.tensor([1, 1, -1, 3, 9]), torch.tensor([0, 2, 4, 3, -1])
    y = causal_conv_packed(x, w, bias, window, starts, slots, out)
    for s, n in enumerate(lens):
        first = int(starts[s])
        old = before[slots[s]].t() if 0 <= slots[s] < 7 else torch.zeros(k - 1, d, dtype=F64)
        rows = torch.cat([old, x[first:first + n]])
        assert torch.allclose(y[first:first + n], causal_conv_ref(rows[None], w, bias)[0, k - 1:])
        if out[s] >= 0:
            assert torch.equal(window[out[s]], rows[n:].t())
    assert torch.equal(window[[1, 5, 6]], before[[1, 5, 6]]) and (y[:2] == 0).all() and (y[19:] == 0).all()
    # pieces of one sequence, one call after another, are the sequence
    whole = causal_conv(x[None], w, bias)[0]
    window.zero_()
    pieces = [causal_conv_packed(x[a:b], w, bias, window, torch.tensor([0, b - a]), torch.tensor([2]))
              for a, b in ((0, 1), (1, 3), (3, 13), (13, 20))]
    assert torch.allclose(torch.cat(pieces), whole)


def test_refusals():
    x, w, bias = torch.zeros(2, 5, 6), torch.zeros(6, 4), torch.zeros(6)
    for bad in (dict(x=x[0]), dict(w=w[:5]), dict(w=w[:, None, None]), dict(bias=bias[:5]), dict(w=torch.zeros(6, 2, 4))):
        with pytest.raises(ValueError):
            causal_conv(bad.get("x", x), bad.get("w", w), bad.get("bias", bias))
    with pytest.raises(ValueError, match="scan_impl"):
        causal_conv(x, w, bias, impl="nonsense")
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv(x, w, bias, impl="cuda")
    rows, window, starts = x[0], torch.zeros(3, 6, 3), torch.tensor([0, 2, 5])
    for kw in (dict(window=window[:, :, :2]), dict(starts=starts[None]), dict(slots=torch.tensor([0])),
               dict(out_slots=torch.tensor([0, 1, 2])), dict(starts=None), dict(starts=torch.arange(5))):
        with pytest.raises(ValueError):
            causal_conv_packed(rows, w, bias, **{"window": window, "starts": starts, **kw})
    for kw in (dict(starts=starts.float()), dict(slots=torch.tensor([True, False]))):
        with pytest.raises(RuntimeError, match="integers"):
            causal_conv_packed(rows, w, bias, window, **{"starts": starts, **kw})


def test_the_c_interface_refuses_before_a_launch():
    lib = _native.load()
    p, odd = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001)
    fwd = lambda x=p, ldt=6, bt=2, t=5, d=6, k=4, dtype=0: lib.mms_conv_fwd(x, 30, ldt, p, p, p, bt, t, d, k, 1, dtype, None)
    bad = _native.MMS_ERR_INVALID_ARG
    assert [fwd(x=None), fwd(bt=0), fwd(t=0), fwd(d=0), fwd(k=0), fwd(k=9), fwd(dtype=2), fwd(ldt=-1),
            fwd(bt=1 << 20, t=1 << 20), fwd(d=1 << 25)] == [bad] * 10
    assert fwd(x=odd) == _native.MMS_ERR_MISALIGNED
    need = lib.mms_conv_workspace_size(2, 5, 6, 4)
    bwd = lambda ws, nb: lib.mms_conv_bwd(p, 30, 6, p, p, p, p, p, p, ws, nb, 2, 5, 6, 4, 1, 0, None)
    assert need > 0 and bwd(p, need - 1) == bwd(None, need) == _native.MMS_ERR_WORKSPACE
    assert bwd(ctypes.c_void_p(0x10010), need) == _native.MMS_ERR_MISALIGNED
    packed = lambda starts=p, rows=5, count=2, places=3, k=4, wide=0: lib.mms_conv_packed(
        p, 6, p, p, p, places, starts, p, p, wide, p, rows, count, 6, k, 1, 0, None)
    assert [packed(starts=None), packed(rows=0), packed(count=0), packed(places=0), packed(k=9)] == [bad] * 5
    assert packed(starts=ctypes.c_void_p(0x10004), wide=1) == _native.MMS_ERR_MISALIGNED
