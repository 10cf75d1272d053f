"""Derivatives around the fused convolution that are there, or refused, but not dropped."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from mamba_metal import MambaConfig, TinyMamba, causal_conv

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


def test_a_forward_mode_tangent_is_refused():
    """Whichever tensor carries it, with gradients on or off; without one, within a level, nothing changes."""
    g = torch.Generator().manual_seed(0)
    t = dict(x=torch.randn(2, 9, 8, generator=g).cuda(), weight=torch.randn(8, 4, generator=g).cuda(),
             bias=torch.randn(8, generator=g).cuda())
    want = causal_conv(**t)
    with forward_ad.dual_level():
        assert torch.equal(causal_conv(**t), want)
        for key, v in t.items():
            dual = {**t, key: forward_ad.make_dual(v, torch.ones_like(v))}
            with pytest.raises(NotImplementedError):
                causal_conv(**dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                causal_conv(**dual)
            # (the PyTorch form has it)
            assert forward_ad.unpack_dual(causal_conv(**dual, impl="torch")).tangent is not None
