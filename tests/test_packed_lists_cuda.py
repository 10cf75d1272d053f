"""Lists of packed sequences that break the rules, on the kernels: wrong rows, no access outside."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import causal_conv_packed, selective_scan_packed

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows,starts", [(32, [32, 0, 32]), (32, [32, 32, 0]), (31, [31, 0, 31]), (40, [40, 8, 0, 33]),
                                         (64, [64, 32, 0, 64]), (64, [33, 0, 64]), (300, [300, 270, 10, 300])])
def test_starts_that_do_not_ascend(rows, starts):
    """Up to one segment of 32 rows (no workspace) and more; what is beside the cache's places stays, and
    a call with good lists after it is right."""
    d, n, places = 8, 4, 3
    g = torch.Generator().manual_seed(rows)
    x, dt, b, c = (torch.rand(rows, m, generator=g).to(DEV) for m in (d, d, n, n))
    aneg, w = torch.rand(d, n, generator=g).to(DEV), torch.rand(d, 4, generator=g).to(DEV)
    state = torch.full((places + 2, d, n), 7.0, device=DEV)
    window = torch.full((places + 2, d, 3), 7.0, device=DEV)
    lists = torch.tensor(starts, device=DEV), torch.tensor([2, -1, 0][:len(starts) - 1], device=DEV)
    y = selective_scan_packed(x, dt, aneg, b, c, state[1:-1], *lists)
    z = causal_conv_packed(x, w, None, window[1:-1], *lists)
    torch.cuda.synchronize()
    assert y.shape == z.shape == (rows, d)
    for cache in (state, window):
        assert (cache[[0, 2, places + 1]] == 7).all()
    good, none = torch.tensor([0, rows], device=DEV), torch.tensor([-1], device=DEV)
    y = selective_scan_packed(x, dt, aneg, b, c, state[1:-1], good, none, torch.tensor([1], device=DEV))
    want, h = torch.zeros(rows, d, device=DEV), torch.zeros(d, n, device=DEV)
    for t in range(rows):
        h = torch.exp(-dt[t, :, None] * aneg) * h + (dt[t] * x[t])[:, None] * b[t]
        want[t] = h @ c[t]
    # positive sums, each step of both off by a few roundings (2^-22 the kernel's decay)
    assert torch.allclose(y, want, rtol=rows * 2.0 ** -20, atol=0)
    assert torch.allclose(state[2], h, rtol=rows * 2.0 ** -20, atol=0)
