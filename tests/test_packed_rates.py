"""Rates so large that a step leaves nothing of a state: the packed scan on every path, short and long."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import selective_scan_packed

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF = float("inf")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 16, 64])
@pytest.mark.parametrize("raw", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 13, 40, 72, 200])
def test_a_huge_rate_keeps_the_last_step_alone(device, dtype, n, raw, rows):
    """Rows that fill no whole tile, single tokens, several segments; an Aneg that is infinite or overflows
    in units of log 2. h_t is dt_t B_t x_t, or, where dt is 0, h_{t-1}; other channels do not notice."""
    d = 6
    g = torch.Generator().manual_seed(rows + n)
    x = torch.randn(rows, d, generator=g).to(dtype)
    dt = torch.randn(rows, d, generator=g).to(dtype) if raw else (0.01 + 0.2 * torch.rand(rows, d, generator=g)).to(dtype)
    b, c = (torch.randn(rows, n, generator=g).to(dtype) for _ in range(2))
    if not raw:
        dt[::5, 1] = 0
        dt[rows // 2:, 2] = 0
    aneg = torch.rand(d, n, generator=g)
    state = torch.randn(2, d, n, generator=g)
    huge = {0: INF, 1: 3e38, 2: INF, 3: 2.5e38}
    used = aneg.clone()
    for ch, v in huge.items():
        used[ch] = v

    def run(rates, starts):
        s = state.clone().to(device)
        y = selective_scan_packed(x.to(device), dt.to(device), rates.to(device), b.to(device), c.to(device), s,
                                  None if starts is None else torch.tensor(starts, device=device),
                                  dt_range=(0.01, 0.2) if raw else None)
        return y.cpu().double(), s.cpu().double()

    for starts in ([0, rows], [0, 0, rows]) + ((None,) if rows <= 2 else ()):
        y, after = run(used, starts)
        y_plain, after_plain = run(aneg, starts)
        assert torch.equal(y[:, 4:], y_plain[:, 4:]) and torch.equal(after[:, 4:], after_plain[:, 4:])
        steps = 0.01 + (0.2 - 0.01) * torch.sigmoid(dt.double()) if raw else dt.double()
        seqs = [(i, i + 1, i) for i in range(rows)] if starts is None else [(starts[i], starts[i + 1], i) for i in range(len(starts) - 1)]
        for first, end, place in seqs:
            for ch in huge:
                h = state[place, ch].double()
                for t in range(first, end):
                    h = (steps[t, ch] * x[t, ch].double()) * b[t].double() if steps[t, ch] != 0 else h
                    terms = h * c[t].double()
                    # dt (of logits: a sigmoid of 16 roundings), dt x, B, C, the sum's n and y's own rounding
                    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
                    bound = (n + 8 + 32 * raw) * 2.0 ** -24 * terms.abs().sum() + half * terms.sum().abs() + 1e-30
                    assert (y[t, ch] - terms.sum()).abs() <= bound * (1 + half), (ch, t)
                assert ((after[place, ch] - h).abs() <= (8 + 32 * raw) * 2.0 ** -24 * h.abs()).all(), ch


@pytest.mark.parametrize("device", DEVICES)
def test_a_rate_that_is_no_number_is_not_taken_for_a_finite_one(device):
    x, bc, aneg = torch.ones(40, 4), torch.ones(40, 4), torch.ones(4, 4)
    aneg[2] = float("nan")
    for rows, starts in ((40, [0, 40]), (1, None)):
        state = torch.zeros(1, 4, 4, device=device)
        y = selective_scan_packed(x[:rows].to(device), x[:rows].to(device), aneg.to(device), bc[:rows].to(device),
                                  bc[:rows].to(device), state, None if starts is None else torch.tensor(starts, device=device))
        assert y[:, 2].isnan().all() and state[0, 2].isnan().all() and torch.isfinite(y[:, [0, 1, 3]]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [9, 40, 700])
def test_what_is_not_finite_stays_so(device, rows):
    """From the row that it enters at, in its channel; infinite or NaN by the path."""
    g = torch.Generator().manual_seed(0)
    x, dt = torch.rand(rows, 4, generator=g), 0.1 * torch.rand(rows, 4, generator=g) + 0.01
    b, c = 0.5 + torch.rand(rows, 4, generator=g), 0.5 + torch.rand(rows, 4, generator=g)
    at = rows // 2
    x[at, 1] = INF
    state = torch.zeros(1, 4, 4)
    state[0, 3, 2] = INF
    s = state.to(device)
    y = selective_scan_packed(x.to(device), dt.to(device), torch.rand(4, 4, generator=g).to(device), b.to(device), c.to(device), s,
                              torch.tensor([0, rows], device=device)).cpu()
    bad = torch.zeros(rows, 4, dtype=torch.bool)
    bad[at:, 1] = True
    bad[:, 3] = True
    assert torch.equal(torch.isfinite(y), ~bad)
    assert not torch.isfinite(s[0, 1]).any() and not torch.isfinite(s[0, 3, 2]) and torch.isfinite(s[0, [0, 2]]).all()
