"""The head's losses and their gradients in float64, with rigorous error bounds (test helper).

u(t) is the unit roundoff (half of torch.finfo(t).eps). With g(n) = (n + 16) * 2^-23 the
kernels' sums of n products err by at most g(n) times the sum of the products' magnitudes:
every step of an accumulation, rounded or truncated to 24 bits, loses at most 2^-23 of a
partial sum that those magnitudes bound, and the 16 covers the two fp16 parts of a float32
factor (each factor to 2^-22, the left-out product of the second parts 2^-22: 3 * 2^-22 =
6 * 2^-23) and the scaling by log2(e) / temperature. The fp16 parts follow a scaling of the
largest element to at least 2^14 and end at fp16's last step of 2^-24: half of it is 2^-39 of
the largest element, the absolute term FOOT (for dz, whose scale is 2^14 times 1: 2^-39 of r).
"""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
FOOT = 2.0 ** -39


def u(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def g(n: int) -> float:
    return (n + 16) * 2.0 ** -23


def sparse(case_k, target=None, ignore=None, index=None, logits=None, tau=1.0):
    """(index (M, k) clamped, p (M, k), own (M), counts (M)) of a cross entropy or a distillation:
    loss = counts * tau^2 * (own - sum_j p_j (z / tau - lse))."""
    if target is not None:
        counts = target != ignore
        return (torch.where(counts, target, 0)[:, None], counts.double()[:, None],
                torch.zeros(len(target), dtype=torch.float64), counts)
    valid = index >= 0
    t = torch.where(valid, logits.double() / tau, -math.inf)
    counts = ~(t == -math.inf).all(1)
    t = torch.where(counts[:, None], t, 0.0)
    p = torch.where(valid & counts[:, None], torch.softmax(t, 1), 0.0)
    log_p = torch.log_softmax(t, 1)
    own = torch.where(p > 0, p * log_p, 0.0).sum(1)
    return index.clamp(min=0), p, own, counts


def solve(x, w, index, p, own, counts, tau, reduction, dloss):
    """Row losses, the reduced loss, dx, dw in float64 on the CPU, and a bound on the kernels'
    error in each. x, w: CPU tensors of the kernels' type; rows that do not count are zeroed."""
    dtype = x.dtype
    x, w = torch.where(counts[:, None], x.double(), 0.0), w.double()
    rows, dim = x.shape
    vocab = w.shape[0]
    z = x @ w.t() / tau
    ez = (g(dim) * (x.abs() @ w.abs().t()) / tau).amax(1)            # a bound on any logit of the row
    if dtype == torch.float32:
        ez = ez + FOOT * (w.abs().max() * x.abs().sum(1) + x.abs().amax(1) * w.abs().sum(1).max()) / tau
    lse = torch.logsumexp(z, 1)
    log_q = z.gather(1, index) - lse[:, None]
    row = torch.where(counts, tau ** 2 * (own - (p * log_q).sum(1)), 0.0)
    # lse moves by at most ez; its own sum of vocab + 64 terms, exp2 and log2 at 2^-21 relative;
    # the teacher's softmax and the closing sum: 16 roundings of the terms' magnitudes
    mag = p.sum(1) * lse.abs() + (p * log_q.abs()).sum(1) + own.abs()
    e_lse = ez + math.log(vocab + 2) * 4 * U32 + (vocab ** 0.5 + 64) * 2 * U32 + lse.abs() * 4 * U32
    e_row = torch.where(counts, tau ** 2 * (p.sum(1) * (ez + e_lse) + (32 + p.shape[1]) * U32 * (mag + 8)), 0.0)
    n = counts.sum().double()
    if reduction == "none":
        loss, e_loss, r = row, e_row, dloss.double()
    else:
        over = n if reduction == "mean" else torch.ones_like(n)
        loss = row.sum() / over
        e_loss = (e_row.sum() + (rows / 1024 + 64) * U32 * row.abs().sum()) / over
        r = dloss.double() / over * torch.ones(rows, dtype=torch.float64)
    r = torch.where(counts, r, 0.0) * tau
    q = torch.exp(z - lse[:, None])
    mass = p.sum(1, keepdim=True)
    dz = (q * mass).scatter_add(1, index, -p) * r[:, None]
    # dz: q to within the errors of z and lse; p to its exponential (arguments up to 40, a few
    # roundings) and its sum over lists (k / 32 a lane, five levels); q - p itself rounds at its
    # own size, or at 1 where p is above 1/2; then dz is stored with dtype's roundoff (float32:
    # two parts, 2^-22)
    ep = (64 + p.shape[1] / 32) * U32 * p + 4 * U32 * (p > 0.5)
    ed = r.abs()[:, None] * (q * (2 * (ez + e_lse)[:, None] + 16 * U32) + torch.zeros_like(q).scatter_add(1, index, ep))
    ed = ed + dz.abs() * (u(dtype) if dtype != torch.float32 else 4 * U32)
    if dtype == torch.float32:
        ed = ed + 2 * FOOT * r.abs()[:, None]
    dx, dw = dz @ w, dz.t() @ x
    e_dx = ed @ w.abs() + g(vocab) * (dz.abs() @ w.abs())
    e_dw = ed.t() @ x.abs() + g(rows) * (dz.t().abs() @ x.abs())
    if dtype == torch.float32:
        e_dx = e_dx + FOOT * w.abs().max() * dz.abs().sum(1, keepdim=True)
        e_dw = e_dw + FOOT * (r[:, None] * x).abs().max() * (dz / torch.where(r == 0, 1.0, r)[:, None]).abs().sum(0)[:, None]
    tiny = 1e-36                                                     # float32's range at its foot
    e_dx = e_dx * (1 + u(dtype)) + u(dtype) * dx.abs() + tiny
    e_dw = e_dw * (1 + u(dtype)) + u(dtype) * dw.abs() + tiny
    return dict(row=row, loss=loss, e_loss=e_loss, dx=dx, e_dx=e_dx, dw=dw, e_dw=e_dw)


def check(name, got, want, err):
    """got within err of want, element by element; NaN nowhere."""
    got = got.detach().cpu().double()
    off = (got - want).abs()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    worst = float((off / err.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{name}: {worst:.3g} times the bound"


def check_norm(name, got, want, tol):
    """The 2-norm of the difference within tol of want's: what elementwise bounds are too wide for."""
    got = got.detach().cpu().double()
    rel = float((got - want).norm() / want.norm().clamp(min=1e-300))
    assert rel <= tol, f"{name}: {rel:.3g} > {tol:.3g}"
