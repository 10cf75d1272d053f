"""The head's losses where the vocabulary is cut into pieces, forward and backward.

A piece is bounded by w's staged rows (512 MB: wide rows, float32 or unaligned bf16), and in the
forward by the parts of the log-sum-exp, in the backward by dz. Targets and list entries lie on
both sides of every border that 2 to 10 equal pieces of whole tiles can have. Compared with
float64 on the GPU, element by element within _head_ref's bounds where the logits are few enough.
"""
from __future__ import annotations

import math

import pytest
import torch

from _head_ref import solve, sparse
from mamba_metal import _native, linear_cross_entropy, linear_distillation

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
TILE = 256


def inputs(rows, vocab, dim, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    w = torch.randn(vocab, dim, generator=gen, device="cuda") * (2.0 / math.sqrt(dim))
    target = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    edges = []
    for pieces in range(2, 11):
        size = -(-(-(-vocab // pieces)) // TILE) * TILE
        edges += [e + d for e in range(size, vocab, size) for d in (-1, 0)]
    edges = torch.tensor(edges + [0, vocab - 1], device="cuda")
    n = min(rows // 2, len(edges))
    target[:n] = edges[torch.randperm(len(edges), generator=gen, device="cuda")[:n]]
    x = torch.randn(rows, dim, generator=gen, device="cuda") + 2 * torch.rand(rows, 1, generator=gen, device="cuda") * w[target]
    return x.to(dtype), w.to(dtype), target, edges, gen


def lists(rows, vocab, k, edges, gen):
    """k entries a row, in no order, some empty, one of them twice, half from the borders."""
    index = torch.randint(0, vocab, (rows, k), generator=gen, device="cuda")
    index[:, : k // 2] = edges[torch.randint(0, len(edges), (rows, k // 2), generator=gen, device="cuda")]
    index[:, 1] = -1
    index[:, k - 1] = index[:, 0]
    return index, 2 * torch.randn(rows, k, generator=gen, device="cuda")


def cut(rows, vocab, dim, k, dtype):
    """Whether the forward (few rows, which the CUDA cores take: the backward) asks for less than w's staged copy."""
    whole = vocab * ((dim + 7) // 8 * 8) * (4 if dtype == F32 else 2)
    backward = rows <= (8 if dtype == F32 else 2)
    return _native.load().mms_head_workspace_size(rows, vocab, dim, k, int(dtype == BF16), dim, dim, backward) < whole


def held(x, w, parts, tau, reduction, dloss, loss, grads):
    with torch.device("cuda"):
        want = solve(x, w, *parts, tau, reduction, dloss)
        for name, got in (("loss", loss.detach()), ("dx", grads[0]), ("dw", grads[1])):
            off = (got.double() - want[name]).abs()
            worst = float((off / want["e_" + name].clamp(min=1e-300)).max())
            assert torch.isfinite(got).all() and worst <= 1.0, f"{name}: {worst:.3g} times the bound"
            del off


# rows: on the CUDA cores (3, 2), with the loss in the last launch (16), above it, with left-out rows (600)
STAGED = [(16, 140000, 1024, F32), (40, 140000, 1024, F32), (600, 70001, 2050, F32), (3, 140000, 1024, F32),
          (24, 140000, 2047, BF16), (600, 140000, 2047, BF16), (2, 140000, 2047, BF16)]


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,vocab,dim,dtype", STAGED)
def test_cross_entropy(rows, vocab, dim, dtype, reduction):
    x, w, target, edges, gen = inputs(rows, vocab, dim, dtype)
    assert cut(rows, vocab, dim, 0, dtype)
    if rows > 3:
        target[2::5] = -100
        x[2::5] = float("nan")
    dloss = torch.randn(rows, generator=gen, device="cuda") if reduction == "none" else torch.tensor(1.3, device="cuda")
    xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xd, wd, target, reduction=reduction)
    grads = torch.autograd.grad(loss, [xd, wd], dloss.reshape(loss.shape))
    with torch.device("cuda"):
        parts = sparse(1, target=target, ignore=-100)
    held(x, w, parts, 1.0, reduction, dloss, loss, grads)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(xd, wd, target, reduction=reduction), loss)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,vocab,dim,dtype", STAGED)
def test_distillation(rows, vocab, dim, dtype, reduction):
    x, w, _, edges, gen = inputs(rows, vocab, dim, dtype)
    k = 40
    assert cut(rows, vocab, dim, k, dtype)
    index, logits = lists(rows, vocab, k, edges, gen)
    if rows > 3:
        index[1::4] = -1
        x[1::4] = float("nan")
    dloss = torch.randn(rows, generator=gen, device="cuda") if reduction == "none" else torch.tensor(0.8, device="cuda")
    xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_distillation(xd, wd, index, logits, 2.0, reduction=reduction)
    grads = torch.autograd.grad(loss, [xd, wd], dloss.reshape(loss.shape))
    with torch.device("cuda"):
        parts = sparse(k, index=index, logits=logits, tau=2.0)
    held(x, w, parts, 2.0, reduction, dloss, loss, grads)


@pytest.mark.parametrize("rows,vocab", [(8192, 300000), (1 << 20, 3000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_rows(dtype, rows, vocab):
    """300000 entries: parts of the log-sum-exp for 8192 rows exceed 512 MB above 262143, dz above
    32768 (float32 16384). A million rows: dz exceeds 2 GB above 1024 entries (float32 512). Losses
    as _head_ref bounds a row's (logits of 16 products: below 2e-6 of 1 plus the loss), gradients
    by their norms: float32 2e-5 as in test_head_cuda.py, bf16 the result's own rounding and 2^-11."""
    dim, k = 16, 6
    x, w, target, edges, gen = inputs(rows, vocab, dim, dtype)
    target[::7] = -100
    index, logits = lists(rows, vocab, k, edges, gen)
    index[::9] = -1
    for kd in (False, True):
        xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        if kd:
            loss = linear_distillation(xd, wd, index, logits, 2.0, reduction="none")
        else:
            loss = linear_cross_entropy(xd, wd, target, reduction="none")
        dx, dw = torch.autograd.grad(loss.sum(), [xd, wd])
        tau = 2.0 if kd else 1.0
        want_dx, want_dw = torch.empty(rows, dim, dtype=torch.float64, device="cuda"), 0
        step = (1 << 30) // vocab
        for a in range(0, rows, step):
            s = slice(a, a + step)
            with torch.device("cuda"):
                at, p, own, counts = sparse(k, index=index[s], logits=logits[s], tau=tau) if kd \
                    else sparse(1, target=target[s], ignore=-100)
            z = x[s].double() @ w.double().t() / tau
            lse = torch.logsumexp(z, 1)
            row = torch.where(counts, tau ** 2 * (own - (p * (z.gather(1, at) - lse[:, None])).sum(1)), 0.0)
            assert ((loss[s].detach().double() - row).abs() <= 2e-6 * (1 + row.abs()) * tau ** 2).all()
            z = torch.exp(z - lse[:, None]) * p.sum(1, keepdim=True)
            z = z.scatter_add(1, at, -p) * (counts * tau)[:, None]
            want_dx[s] = z @ w.double()
            want_dw = want_dw + z.t() @ x[s].double()
            del z
        for name, got, want in (("dx", dx, want_dx), ("dw", dw, want_dw)):
            own = float((want.to(BF16).double() - want).norm()) if dtype == BF16 else 0.0
            tol = math.hypot(1.01 * own, 2.0 ** -11 * float(want.norm())) if dtype == BF16 else 2e-5 * float(want.norm())
            assert float((got.double() - want).norm()) <= tol, name
        del want_dx, want_dw, dx, dw
