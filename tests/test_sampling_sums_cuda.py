"""Sampling where few of a row's entries are kept and the draw queues them a warp's worth at a time."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import sample_tokens, sample_tokens_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(1, 65536), (3, 140000), (200, 30000)])
def test_every_kept_entry_counts_once(rows, vocab):
    """More entries kept than are ever sorted, in runs of every length among the 32 lanes' entries. The
    log-probability takes the sum of all of them: one lost, or one taken twice, moves it by 3e-6 at least."""
    g = torch.Generator().manual_seed(vocab)
    keep = torch.rand(rows, vocab, generator=g) < 0.3 * torch.rand(rows, vocab // 500 + 1, generator=g).repeat_interleave(500, 1)[:, :vocab]
    # (float32 values that differ by little, so that each kept weight is between 1 / e and 1)
    z = torch.where(keep, torch.rand(rows, vocab, generator=g), torch.full((), -1.0)).cuda()
    u = torch.rand(rows, generator=g).cuda()
    k = keep.sum(1).cuda()
    assert int(k.min()) > 2100 and int(k.max()) < 100000
    for kw in (dict(top_k=k), dict(top_k=k, min_p=0.5), dict(top_k=k - 3, top_p=0.97)):
        token, lp = sample_tokens(z, u, return_logprob=True, **kw)
        want, wlp = sample_tokens_ref(z, u, **kw)
        assert torch.equal(token, want)
        # two roundings of the logarithm to float32, weights' of at most vocab 2^-45 of a sum of at least 1
        assert ((lp - wlp).abs() <= 2 * 2.0 ** -24 * wlp.abs() + vocab * 2.0 ** -45).all()
