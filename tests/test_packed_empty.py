"""Packed calls without rows hand states on at a cost that grows with the sequences, not with their square."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import causal_conv_packed, selective_scan_packed
from mamba_metal.packed import _nothing_packed

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.uint8])
def test_any_lists(device, dtype):
    """Against one place after another; places outside on either side, slots of the call's own order."""
    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        places, count = int(torch.randint(1, 9, (1,), generator=g)), int(torch.randint(1, 12, (1,), generator=g))
        cache = torch.randn(places, 3, 2, generator=g)
        low = 0 if dtype == torch.uint8 else -2
        src = torch.randint(low, places + 2, (count,), generator=g).to(dtype) if seed % 3 or count > places else None
        dst = torch.randint(low, places + 2, (count,), generator=g).to(dtype)
        for i in range(count):                             # a place that two sequences name is written by one
            if int(dst[i]) in dst[:i].tolist():
                dst[i] = places
        want = cache.clone()
        for i in range(count):
            p = i if src is None else int(src[i])
            if 0 <= int(dst[i]) < places:
                want[int(dst[i])] = cache[p] if 0 <= p < places else 0
        got, x = cache.clone().to(device), torch.zeros(0, 3, device=device)
        assert _nothing_packed(x, got, count, None if src is None else src.to(device), dst.to(device)).shape == (0, 3)
        assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_memory():
    places = 20000
    state, window = torch.ones(places, 4, 4, device="cuda"), torch.ones(places, 4, 3, device="cuda")
    x, bc = torch.zeros(0, 4, device="cuda"), torch.zeros(0, 4, device="cuda")
    w, aneg = torch.ones(4, 4, device="cuda"), torch.ones(4, 4, device="cuda")
    starts = torch.zeros(places + 1, dtype=torch.int32, device="cuda")
    out = torch.arange(places, device="cuda").flip(0)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    selective_scan_packed(x, x, aneg, bc, bc, state, starts, None, out)
    causal_conv_packed(x, w, None, window, starts, None, out)
    # a handful of copies of the cache and of lists (the square of the places would be 400 MB)
    assert torch.cuda.max_memory_allocated() - before < 32 << 20
