"""bf16 gradients over long sums: many rows (dw), a large vocabulary (dx).

The tensor core adds 16 products at a time with truncation to 24 bits, so a long sum drifts
towards zero: each addition loses less than 2^-23 of the sum so far. The kernels cut sums into parts of at
most 2048 products (128 additions: 2^-16) and round the parts' sums to nearest. What is looked at
is the mean, over the N > 4 10^5 elements of a gradient, of got - bf16(want) towards or from zero, over
|want|: the drift stays in it. The sums are coherent and their values spread over binades, so that
the results round either way: dz's own roundings (2^-11 of each of 10^5 and more values, in
each sum its own) move a result by 2^-11 / sqrt(10^5) = 2^-19, and what flips with that goes down by
another sqrt(N). The exponentials err by 2^-21, their mean too. 2^-18 is left for all of it.
dz's logits z are themselves one such part where x has up to 2048 columns: below by up to 2^-16 z
where all products are positive, and so is log q (the forward's log-sum-exp comes in finer parts).
The first test has z = 2 to 12 and adds the mean of 2^-16 z as dw's terms weigh it; in the second
the products have both signs, and z's sums stay below 1.
The sizes give more tiles than the GPU has pairs of SMs, so that there are sums that
are not split among them; without parts their drift is up to 2^-9 (dw) and 2^-10 (dx).
"""
from __future__ import annotations

import pytest
import torch

from mamba_metal import linear_cross_entropy

pytestmark = pytest.mark.gpu
BOUND = 2.0 ** -16 + 2.0 ** -18


def spread(gen, *shape):
    """Between 1 and 4, uniform in the logarithm."""
    return 4 ** torch.rand(*shape, generator=gen, device="cuda")


def drift_of(got, want):
    return abs(float(((got.double() - want.bfloat16().double()) / want).mean()))


def test_a_quarter_million_rows():
    rows, vocab, dim = 1 << 18, 4096, 2048
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = (0.1 * spread(gen, dim) * (torch.rand(rows, dim, generator=gen, device="cuda") + 0.5)).bfloat16()
    w = (0.01 * spread(gen, vocab, 1) * torch.rand(vocab, dim, generator=gen, device="cuda")).bfloat16()
    target = torch.zeros(rows, dtype=torch.int64, device="cuda")
    wd = w.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(linear_cross_entropy(x, wd, target), wd)
    want, by_z = (torch.zeros(vocab, dim, dtype=torch.float64, device="cuda") for _ in range(2))
    for xs in x.split(1 << 15):
        z = xs.double() @ w.double().t()
        q = torch.softmax(z, 1) / rows
        by_z += (q * z).t() @ xs.double()
        q[:, 0] -= 1.0 / rows
        want += q.t() @ xs.double()
    assert drift_of(got, want) <= BOUND + 2.0 ** -16 * float((by_z / want.abs()).mean())


@pytest.mark.parametrize("rows,vocab,dim", [(1024, 1 << 17, 8192), (200, 1 << 19, 2048)])
def test_many_entries(rows, vocab, dim):
    """One plane of dz, and two, whose sums are split among the pairs and still longer than a part."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = (0.01 * torch.randn(rows, dim, generator=gen, device="cuda")).bfloat16()
    w = (0.1 * spread(gen, dim) * (torch.rand(vocab, dim, generator=gen, device="cuda") + 0.5)).bfloat16()
    w[7] = 0.001                                    # the target's share of dx: next to nothing
    target = torch.full((rows,), 7, device="cuda")
    xd = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(linear_cross_entropy(xd, w, target, reduction="sum"), xd)
    z = torch.cat([x.double() @ ws.double().t() for ws in w.split(1 << 14)], 1)
    dz = torch.softmax(z, 1)
    dz[:, 7] -= 1
    want = sum(d @ ws.double() for d, ws in zip(dz.split(1 << 14, 1), w.split(1 << 14)))
    assert drift_of(got, want) <= BOUND
