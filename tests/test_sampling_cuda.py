"""The sampling kernel against sample_tokens_ref: the same tokens, log-probabilities to float32.

The kernel's weights are float64 rounded to whole numbers of 2^-44 of the largest, at most 2^-45
off, and their sums are exact; a draw or a cut would have to lie within the sums' error (V 2^-45 at
most, 2^-45 sqrt(V) as a rule) of a border to differ. The log-probability is the logarithm of a
float64 quotient rounded once, and the reference's too: two roundings of its value and the kept
weights' error, V 2^-45 of a sum of at least 1, apart at most.
"""
from __future__ import annotations

import pytest
import torch

from mamba_metal import sample_tokens, sample_tokens_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def check(z, u, t=1.0, k=0, p=1.0, m=0.0):
    on = lambda v: v.to(DEV) if torch.is_tensor(v) else v
    token, lp = sample_tokens(on(z), on(u), on(t), on(k), on(p), on(m), return_logprob=True)
    want, wlp = (v.cpu() for v in sample_tokens_ref(on(z), on(u), on(t), on(k), on(p), on(m)))
    assert torch.equal(token.cpu(), want), (token.cpu() != want).nonzero()[:5]
    lp = lp.cpu()
    assert torch.equal(lp.isnan(), wlp.isnan())
    good = ~wlp.isnan()
    assert ((lp - wlp).abs()[good] <= 2 * 2.0 ** -24 * wlp[good].abs() + z.shape[-1] * 2.0 ** -45).all()
    assert torch.equal(sample_tokens(on(z), on(u), on(t), on(k), on(p), on(m)).cpu(), want)
    return token


def logits(rows, vocab, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = spread * torch.randn(rows, vocab, generator=g)
    return z.to(dtype), torch.rand(rows, generator=g), g


WIDE = [(1, 300000), (2, 131072), (3, 131073)]
SIZES = [(1, 1), (3, 2), (2, 31), (5, 33), (1, 511), (4, 4097), (1, 32768), (40, 5003), (80, 20001), (150, 9001), (300, 1000), (2, 131072)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_each_cut_matches(rows, vocab, dtype):
    z, u, g = logits(rows, vocab, dtype, rows + vocab)
    for kw in (dict(), dict(t=0.7), dict(t=0.0), dict(k=1), dict(k=2), dict(k=40), dict(k=max(1, vocab // 2)), dict(k=vocab),
               dict(k=vocab + 5), dict(p=0.5), dict(p=0.9), dict(p=0.999), dict(p=0.0), dict(p=1e-9), dict(m=0.05), dict(m=1.0),
               dict(k=50, p=0.9, m=0.01, t=1.3), dict(p=0.95, t=5.0), dict(t=100.0, p=0.7), dict(t=0.05, p=0.99)):
        check(z, u, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", WIDE)
def test_flat_and_wide_rows_do_not_overflow(rows, vocab, dtype):
    """All weights the largest there is, at and above the sizes where sums need more bits."""
    flat, u, g = logits(rows, vocab, dtype, vocab)
    for z in (torch.zeros_like(flat), flat, torch.where(flat > 4, 0.0, -3.0).to(dtype)):
        for kw in (dict(), dict(p=0.5), dict(p=0.999), dict(k=vocab // 2, p=0.7), dict(k=70000)):
            check(z, u, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_settings_of_each_rows_own(rows, vocab, dtype):
    z, u, g = logits(rows, vocab, dtype, 7 * rows + vocab, spread=3.0)
    t = 1.5 * torch.rand(rows, generator=g)
    t[::7] = 0.0
    k = torch.tensor([0, 1, 7, 300, 3000, vocab])[torch.randint(0, 6, (rows,), generator=g)]
    p = torch.rand(rows, generator=g) * 1.1
    m = 0.2 * torch.rand(rows, generator=g) * (torch.rand(rows, generator=g) < 0.5)
    check(z, u, t, k, p, m)
    check(z, u, t, k.int(), p.double(), m)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks_ties_and_borders(dtype):
    low = torch.finfo(dtype).min
    for vocab in (5, 3000, 40000):
        for rows in (1, 200):
            z, u, g = logits(rows, vocab, dtype, vocab + rows)
            gone = torch.rand(rows, vocab, generator=g) < 0.7
            for fill in (-INF, low, -1e4):
                w = z.masked_fill(gone, fill)
                for kw in (dict(), dict(k=40), dict(p=0.9), dict(k=vocab - 1, p=0.99), dict(t=3.0, m=0.01), dict(t=float(2 ** 100), p=0.5)):
                    check(w, u, **kw)
            flat = torch.full_like(z, 3.0)
            steps = (torch.arange(vocab) % 3).to(dtype).expand(rows, vocab).contiguous()
            signed = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0).to(dtype).expand(rows, vocab).contiguous()
            for w in (flat, steps, -steps, signed, torch.where(gone, flat, -INF)):
                for kw in (dict(), dict(k=3), dict(k=vocab // 2 + 1), dict(p=0.5), dict(p=0.3), dict(k=vocab // 2 + 1, p=0.7), dict(m=0.5)):
                    check(w, u, **kw)
            one = torch.full_like(z, -INF)
            one[:, vocab // 2] = -5.0
            check(one, u, p=0.5)
            assert (check(torch.full_like(z, -INF), u) == -1).all()
            for bad in (float("nan"), INF):
                w = z.clone()
                w[0, vocab - 1] = bad
                for kw in (dict(), dict(k=5), dict(p=0.4), dict(k=2, p=0.9, m=0.1), dict(t=0.0)):
                    check(w, u, **kw)
            w = z.clone()
            w[:, 1:4] = INF
            for kw in (dict(), dict(k=2), dict(k=vocab - 1, p=0.5), dict(p=0.99), dict(m=0.9)):
                check(w, u, **kw)
            for edge in (torch.zeros(rows), torch.ones(rows), torch.full((rows,), -1.0), torch.full((rows,), 1 - 2.0 ** -24),
                         torch.full((rows,), float("nan"))):
                check(z, edge, p=0.9)
                check(z, edge)


def test_huge_spreads_need_many_rounds():
    """Values over float32's whole range in one row, most of them in a bin's width of one another."""
    g = torch.Generator().manual_seed(3)
    z = torch.randn(6, 20000, generator=g)
    z[0] = torch.sign(z[0]) * 10.0 ** (38 * torch.rand(20000, generator=g) ** 0.5)
    z[1] = 1e-30 * z[1]
    z[2] = 1e38 * torch.tanh(z[2])
    z[3, 0] = 3e38
    z[4] = 1.0 + 2.0 ** -20 * torch.randint(0, 9, (20000,), generator=g)
    z[5, ::2] = -3e38
    u = torch.rand(6, generator=g)
    for t in (1.0, 1e37, 1e-30, 1e-38):
        for kw in (dict(), dict(k=5000), dict(k=15000, p=0.3), dict(p=0.8), dict(p=0.2)):
            check(z, u, t=t, **kw)


def test_strided_rows_other_shapes_and_unaligned_bases():
    z, u, _ = logits(12, 5000, F32, 1)
    want = check(z, u, p=0.9, k=100)
    wide = torch.full((12, 5100), float("nan"), device=DEV)
    for off in (0, 1, 2, 3, 77):
        wide[:, off:off + 5000] = z.to(DEV)
        assert torch.equal(sample_tokens(wide[:, off:off + 5000], u.to(DEV), top_p=0.9, top_k=100), want)
    assert torch.equal(sample_tokens(z.t().contiguous().to(DEV).t(), u.to(DEV), top_p=0.9, top_k=100), want)
    assert torch.equal(sample_tokens(z.to(DEV).view(3, 4, 5000), u.to(DEV).view(3, 4), top_p=0.9, top_k=100), want.view(3, 4))
    assert torch.equal(sample_tokens(z[3].to(DEV), u[3].to(DEV), top_p=0.9, top_k=100), want[3])
    assert sample_tokens(z[:0].to(DEV), u[:0].to(DEV)).shape == (0,)
    one = z[:1].to(DEV).expand(12, 5000)
    assert torch.equal(sample_tokens(one, u.to(DEV), top_p=0.9), sample_tokens(one.contiguous(), u.to(DEV), top_p=0.9))


def test_draws_follow_the_distribution():
    z = torch.tensor([0.0, 1.0, 2.0, -INF, 0.5])
    n = 100000
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    token = sample_tokens(z.to(DEV).expand(n, 5), u.float().to(DEV))
    share = torch.bincount(token.cpu(), minlength=5) / n
    # u is an even grid, rounded by at most 2^-25: one grid step at each of two ends
    assert (share - torch.softmax(z.double(), 0)).abs().max() <= 2 / n + 2.0 ** -24


def test_streams_graphs_and_refusals():
    z, u, _ = logits(64, 30000, BF16, 4)
    z, u = z.to(DEV), u.to(DEV)
    want = sample_tokens(z, u, top_p=0.9, top_k=3000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(z, u, top_p=0.9, top_k=3000)
    graph.replay()
    assert torch.equal(out, want)
    z.neg_()
    graph.replay()
    assert torch.equal(out, sample_tokens(z, u, top_p=0.9, top_k=3000)) and not torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [sample_tokens(z, u, top_p=0.9, top_k=3000) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, out) for g in got)
    for kw in (dict(logits=z.half()), dict(logits=z.double()), dict(uniform=u.cpu()), dict(temperature=u.cpu()), dict(top_k=u)):
        with pytest.raises(RuntimeError):
            sample_tokens(**{"logits": z, "uniform": u, **kw})
