"""Derivatives around the fused convolution that are there, or refused, but not dropped."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import MambaConfig, TinyMamba

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["conv.weight", "conv.bias"])
def test_one_parameter_of_the_convolution_trained_through_a_cached_step(name):
    """All else frozen: what enters the first block's convolution has no graph of its own."""
    idx = torch.randint(0, 50, (2, 6), generator=torch.Generator().manual_seed(0)).cuda()
    grads = []
    for fuse_conv in (False, True):
        torch.manual_seed(1)
        m = TinyMamba(MambaConfig(vocab_size=50, d_model=16, n_layers=1, d_ff=32, d_state=8, fuse_conv=fuse_conv)).cuda()
        for key, p in m.named_parameters():
            p.requires_grad_(key.endswith(name))
        cache = {}
        with torch.no_grad():
            m(idx[:, :5], cache=cache)
        logits = m(idx[:, 5:], cache=cache)[0]
        assert logits.requires_grad
        logits.square().sum().backward()
        grads.append(dict(m.named_parameters())[f"blocks.0.{name}"].grad)
    assert grads[1].abs().max() > 0 and torch.allclose(*grads, rtol=1e-5, atol=1e-6)
