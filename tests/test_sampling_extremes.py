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


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 5000])
def test_a_setting_that_is_no_number_draws_nothing(device, dtype, vocab):
    g = torch.Generator().manual_seed(0)
    z, u = torch.randn(4, vocab, generator=g).to(dtype).to(device), torch.rand(4, generator=g).to(device)
    for own in ("temperature", "top_p", "min_p"):
        for kw in (dict(), dict(top_k=3), dict(top_k=1), dict(top_k=vocab // 2)):
            values = torch.tensor([0.5, float("nan"), 0.2, 0.9], device=device)
            token, lp = sample_tokens(z, u, return_logprob=True, **{**kw, own: values})
            want, wlp = sample_tokens_ref(z, u, **{**kw, own: values})
            assert token[1] == want[1] == -1 and lp[1].isnan() and wlp[1].isnan(), own
            keep = [0, 2, 3]
            assert torch.equal(token[keep], want[keep]) and (token[keep] >= 0).all() and torch.isfinite(lp[keep]).all()
