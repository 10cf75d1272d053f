"""Sampling beside infinite logits and from settings that are no numbers."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import sample_tokens, sample_tokens_ref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF, BIG = float("inf"), torch.finfo(torch.float32).max


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [4, 3000, 40000])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=2), dict(top_k=3, top_p=0.9), dict(top_k=1), dict(top_p=0.6), dict(min_p=0.5),
                                dict(top_k=2000), dict(top_k=2, min_p=1.0), dict(temperature=INF, top_k=2), dict(temperature=0.0)])
def test_the_largest_finite_logit_weighs_nothing_beside_an_infinite_one(device, vocab, kw):
    z = torch.zeros(3, vocab, device=device)
    z[0, :2] = torch.tensor([INF, BIG])
    z[1, 1:4] = torch.tensor([BIG, BIG, INF])
    z[2, :2] = torch.tensor([BIG, 1.0])                    # no infinite one: it is the largest
    u = torch.tensor([0.9, 0.1, 0.0], device=device)
    token, lp = sample_tokens(z, u, return_logprob=True, **kw)
    assert token[:2].tolist() == [0, 3] and (lp[:2] == 0).all()
    want, wlp = sample_tokens_ref(z, u, **kw)
    assert torch.equal(token, want) and torch.allclose(lp, wlp, rtol=2.0 ** -22, atol=vocab * 2.0 ** -45)
