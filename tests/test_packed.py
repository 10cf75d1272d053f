"""selective_scan_packed in PyTorch ops: against the scan of each sequence; refusals."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mamba_metal import _native, gated_output, selective_scan, selective_scan_packed, selective_scan_proj, selective_scan_step

F64 = torch.float64


def make(rows, d, n, seed=0, dtype=F64):
    g = torch.Generator().manual_seed(seed)
    x, z = (torch.randn(rows, d, generator=g, dtype=dtype) for _ in range(2))
    dt = torch.nn.functional.softplus(torch.randn(rows, d, generator=g, dtype=dtype) - 2)
    b, c = (torch.randn(rows, n, generator=g, dtype=dtype) for _ in range(2))
    aneg = torch.arange(1, n + 1, dtype=dtype) * (1 + 0.1 * torch.rand(d, n, generator=g, dtype=dtype))
    return x, dt, aneg, b, c, z, 1 + torch.randn(d, generator=g, dtype=dtype)


def test_each_sequence_is_a_scan_from_its_state():
    x, dt, aneg, b, c, z, skip = make(20, 5, 4)
    starts = torch.tensor([1, 8, 8, 9, 19])
    state = torch.randn(6, 5, 4, dtype=F64)
    state[3] = 0
    before = state.clone()
    slots, out = torch.tensor([3, 1, 7, -1]), torch.tensor([0, 4, 5, 2])
    y = selective_scan_packed(x, dt, aneg, b, c, state, starts, slots, out, z, skip)
    # sequences 0 and 3 start from zeros, as the scan does
    for s, (i, j) in ((0, (1, 8)), (3, (9, 19))):
        want, h = selective_scan(x[None, i:j], dt[None, i:j], aneg, b[None, i:j], c[None, i:j], impl="torch", return_state=True)
        assert torch.allclose(y[i:j], gated_output(want, z[None, i:j], skip, impl="torch")[0])
        assert torch.allclose(state[out[s]], h[0])
    assert torch.equal(state[4], before[1])                    # an empty sequence hands its state on
    assert (y[[0, 19]] == 0).all() and torch.equal(state[[1, 3]], before[[1, 3]])
    # single tokens: the decode step
    state = before.clone()
    h = before[:2].clone()
    want = selective_scan_step(x[:2], dt[:2], aneg, b[:2], c[:2], h, impl="torch")
    assert torch.allclose(selective_scan_packed(x[:2], dt[:2], aneg, b[:2], c[:2], state), want)
    assert torch.allclose(state[:2], h) and torch.equal(state[2:], before[2:])


def test_logits_and_raw_a():
    x, dt, aneg, b, c, _, _ = make(9, 5, 4, seed=1)
    state = torch.zeros(1, 5, 4, dtype=F64)
    got = selective_scan_packed(x, dt, aneg, b, c, state, torch.tensor([0, 9]), dt_range=(0.01, 0.2))
    want = selective_scan_proj(x[None], dt[None], aneg, b[None], c[None], 0.01, 0.2, impl="torch")
    assert torch.allclose(got, want[0])


def test_refusals():
    x, dt, aneg, b, c, z, skip = make(6, 5, 4, dtype=torch.float32)
    state, starts = torch.zeros(3, 5, 4), torch.tensor([0, 2, 6])

    def call(**kw):
        a = {"x": x, "dt": dt, "aneg": aneg, "b_in": b, "c_in": c, "state": state, "starts": starts, **kw}
        return selective_scan_packed(**a)

    call()
    for kw in (dict(x=x[None]), dict(dt=dt[:5]), dict(aneg=aneg[:4]), dict(b_in=b[:, :3]), dict(c_in=c[:5]),
               dict(state=state[0]), dict(state=state[:, :4]), dict(z=z[:5]), dict(d_skip=skip[:4]), dict(dt_range=(0.1, 0.1)),
               dict(starts=starts[None]), dict(slots=starts), dict(out_slots=torch.tensor([0])), dict(starts=None),
               dict(starts=torch.arange(7)), dict(impl="nonsense")):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(starts=starts.float()), dict(slots=torch.tensor([0.0, 1.0])), dict(impl="cuda"), dict(impl="metal")):
        with pytest.raises(RuntimeError):
            call(**kw)


def test_the_c_interface_refuses_before_a_launch():
    lib = _native.load()
    p = ctypes.c_void_p(0x10000)

    def call(x=p, aneg=p, b=p, ldb=8, state=p, places=3, starts=p, ws=p, nb=1 << 30, rows=500, count=2, d=6, n=8,
             dtype=0, bc=0, raw=0, lo=0.0, hi=1.0, wide=0):
        return lib.mms_scan_packed(x, 6, p, 6, aneg, b, ldb, p, 8, None, 0, None, raw, lo, hi, state, places, starts, p, p,
                                   wide, p, ws, nb, rows, count, d, n, dtype, bc, None)

    bad, off = _native.MMS_ERR_INVALID_ARG, _native.MMS_ERR_MISALIGNED
    assert call(n=6) == call(n=68) == call(n=0) == _native.MMS_ERR_UNSUPPORTED_N
    assert [call(x=None), call(rows=0), call(count=0), call(places=0), call(d=0), call(dtype=2), call(bc=1), call(raw=1, hi=0.0),
            call(starts=None), call(ldb=-1), call(raw=1, lo=float("nan"))] == [bad] * 11
    odd = ctypes.c_void_p(0x10008)
    assert [call(aneg=odd), call(state=odd), call(ws=odd), call(starts=ctypes.c_void_p(0x10004), wide=1),
            call(starts=None, rows=2, b=odd), call(starts=None, rows=2, ldb=9), call(x=ctypes.c_void_p(0x10002))] == [off] * 7
    need = lib.mms_scan_packed_workspace_size(500, 2, 6, 8)
    assert need > 0 and call(nb=need - 1) == call(ws=None) == _native.MMS_ERR_WORKSPACE
    assert lib.mms_scan_packed_workspace_size(500, 2, 6, 7) == 0
