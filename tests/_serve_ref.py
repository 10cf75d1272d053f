"""Error bounds of the convolution and the packed scan, from their steps, in float64.

U32 = 2^-24 is float32's rounding. The kernels' SiLU takes 2^x from ex2.approx (2^-22 relative)
and 1/x from rcp.approx (2^-23), of an argument that is rounded once: a sigmoid of z is off by at most
(|z| + 16) U32 of itself.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

U32 = 2.0 ** -24


def u(dtype) -> float:
    return 2.0 ** -8 if dtype == torch.bfloat16 else U32


def taps(x, w, bias):
    """(pre, sum of magnitudes) of the convolution of x (B, T, D) with w (D, K) in float64."""
    x, w = x.double(), w.double()
    k = w.shape[1]
    rows = F.pad(x, (0, 0, k - 1, 0))
    pre = sum(w[:, j] * rows[:, j:j + x.shape[1]] for j in range(k))
    size = sum((w[:, j] * rows[:, j:j + x.shape[1]]).abs() for j in range(k))
    return (pre, size) if bias is None else (pre + bias.double(), size + bias.double().abs())


def conv_bound(x, w, bias, silu, dtype):
    """(y, bound)."""
    pre, size = taps(x, w, bias)
    off = (w.shape[1] + 1) * U32 * size
    if not silu:
        return pre, off + u(dtype) * pre.abs()
    y = F.silu(pre)
    off = 1.1 * off + y.abs() * (pre.abs() + 16) * U32          # |silu'| < 1.1
    return y, off + u(dtype) * (y.abs() + off)


def conv_grad_bounds(x, w, bias, dy, silu, dtype, depth):
    """[(dx, bound), (dw, bound), (dbias, bound)]; depth: the longest chain of sums over rows."""
    pre, size = taps(x, w, bias)
    x, wd, dy = x.double(), w.double(), dy.double()
    k = wd.shape[1]
    if silu:
        s = torch.sigmoid(pre)
        slope = s * (1 + pre * (1 - s))
        # |silu''| <= 1/2; the slope's own arithmetic is a few operations on values of at most 1 + |pre|
        off = dy.abs() * (0.5 * (k + 1) * U32 * size + (1 + pre.abs() * s) * (pre.abs() + 24) * U32)
    else:
        slope, off = torch.ones_like(pre), torch.zeros_like(pre)
    ds = dy * slope
    back = lambda g, wk: sum(F.pad(g, (0, 0, 0, k - 1))[:, k - 1 - j:k - 1 - j + g.shape[1]] * wk[:, j] for j in range(k))
    dx = back(ds, wd)
    out = [(dx, back(off, wd.abs()) + (k + 1) * U32 * back(ds.abs(), wd.abs()))]
    rows = F.pad(x, (0, 0, k - 1, 0))
    at = lambda g, r: torch.stack([(g * r[:, j:j + g.shape[1]]).sum((0, 1)) for j in range(k)], 1)
    out.append((at(ds, rows), at(off, rows.abs()) + depth * U32 * at(ds.abs(), rows.abs())))
    out.append((ds.sum((0, 1)), off.sum((0, 1)) + depth * U32 * ds.abs().sum((0, 1))))
    return [(v, o + u(dtype) * (v.abs() + o)) for v, o in out]


def scan_bound(x, dt, aneg, b, c, state, seqs, z, d_skip, dt_range, dtype):
    """(y, bound, state, bound) of the packed scan; seqs: [(first, end, from, to)]. A step's decay is off
    by 2^-22 (ex2) and by its argument's error; a segment's decay, whose argument is a sum over the
    segment's dt, by at most max(a e^-a) < 0.4 roundings a row: 2 U32 a step cover it."""
    x, dt, aneg, b, c = (t.double() for t in (x, dt, aneg, b, c))
    arg_off = torch.full_like(dt, 4 * U32)                       # dt * Aneg * log2 e, three roundings
    if dt_range is not None:
        lo, hi = dt_range
        s = torch.sigmoid(dt)
        arg_off = arg_off + (dt.abs() + 24) * U32 + 8 * U32      # the logit's sigmoid, softplus
        dt, aneg = lo + (hi - lo) * s, F.softplus(aneg)
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    new, new_bound = state.double().clone(), torch.zeros_like(state.double())
    for first, end, src, dst in seqs:
        h = torch.zeros_like(aneg) if src is None else state[src].double()
        e = torch.zeros_like(h)
        for t in range(first, end):
            arg = dt[t, :, None] * aneg
            dA = torch.exp(-arg)
            add = (dt[t] * x[t])[:, None] * b[t]
            kept = dA * h
            e = dA * e + kept.abs() * (2.0 ** -22 + arg * arg_off[t, :, None]) \
                + add.abs() * (4 * U32 + arg_off[t, :, None])
            h = kept + add
            e = e + (kept.abs() + add.abs() + 2 * h.abs()) * U32
            y[t] = h @ c[t]
            bound[t] = e @ c[t].abs() + (aneg.shape[1] + 2) * U32 * (h.abs() @ c[t].abs())
        if dst is not None:
            new[dst], new_bound[dst] = h, e
    if d_skip is not None:
        for first, end, _, _ in seqs:
            y[first:end] += d_skip.double()
            bound[first:end] += U32 * y[first:end].abs()
    if z is not None:
        g = F.silu(z.double())
        bound = bound * g.abs() + (y * g).abs() * (z.double().abs() + 20) * U32
        y = y * g
    return y, bound + u(dtype) * (y.abs() + bound), new, new_bound


def close(got, want, bound, what=""):
    off = (got.detach().cpu().double() - want.cpu()).abs()
    bound = bound.cpu() + 1e-30
    assert got.shape == want.shape and not torch.isnan(off).any(), what
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, (what, worst)
    return worst
