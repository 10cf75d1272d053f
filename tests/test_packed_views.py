"""What packed calls copy (rows without unit stride) lives until their kernels are launched."""
from __future__ import annotations

import gc
import weakref

import pytest
import torch

from mamba_metal import _native, selective_scan_packed
from mamba_metal.packed import rows_of


@pytest.mark.parametrize("which", ["x", "dt", "b_in", "c_in", "z"])
def test_copies_outlive_the_native_call(monkeypatch, which):
    """Nothing else holds the copy of a transposed view: were it freed before the call, the allocator would
    hand its memory to the output or the workspace, which the kernels write while they read it."""
    rows, d, n = 40, 8, 4
    t = {k: torch.randn(m, rows).t() for k, m in (("x", d), ("dt", d), ("b_in", n), ("c_in", n), ("z", d))}
    copies, alive = [], []

    def copied(key):
        tensor, ld = rows_of(t[key])
        assert tensor is not t[key] and ld == tensor.shape[1]
        copies.append((key, weakref.ref(tensor)))
        return tensor, ld

    class Library:
        def mms_scan_packed_workspace_size(self, *args):
            return 64

        def mms_scan_packed(self, *args):
            gc.collect()
            alive.extend(key for key, ref in copies if ref() is not None)
            return 0

    monkeypatch.setattr(_native, "load", Library)
    monkeypatch.setattr(_native, "_stream", lambda device: 0)
    _native._scan_packed_workspace.cache_clear()
    plain = lambda key: copied(key) if key == which else rows_of(t[key].contiguous())
    try:
        _native.scan_packed(plain("x"), plain("dt"), torch.rand(d, n), plain("b_in"), plain("c_in"), plain("z"), None, None,
                            torch.zeros(1, d, n), torch.tensor([0, rows]), None, None, 1)
    finally:
        _native._scan_packed_workspace.cache_clear()
    assert alive == [which]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starts", [[0, 700, 1000], None])
def test_every_tensor_as_a_transposed_view(starts, dtype):
    """With a gate and several segments (starts), or single tokens: the results of contiguous rows."""
    rows, d, n = 1000, 72, 16
    g = torch.Generator().manual_seed(0)
    t = {k: torch.randn(rows, m, generator=g).to(dtype).cuda() for k, m in (("x", d), ("b_in", n), ("c_in", n), ("z", d))}
    t["dt"] = (0.1 * torch.rand(rows, d, generator=g)).to(dtype).cuda()
    aneg = (1 + torch.rand(d, n, generator=g)).cuda()
    lists = None if starts is None else torch.tensor(starts, device="cuda")

    def call(**other):
        state = torch.zeros(rows if starts is None else 2, d, n, device="cuda")
        y = selective_scan_packed(aneg=aneg, state=state, starts=lists, **{**t, **other})
        return y, state

    want = call()
    views = {k: v.t().contiguous().t() for k, v in t.items()}
    for other in (*({k: v} for k, v in views.items()), views):
        got = call(**other)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), list(other)
