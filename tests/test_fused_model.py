"""TinyMamba with the residual norm and the head's losses fused (MambaConfig.fuse_norm, fuse_loss).

The fused model is the plain one within rounding: on the CPU (where the fused calls run PyTorch
ops) and on the GPU (kernels), for the loss, every parameter's gradient, the recurrent cache and
the distillation loss. float32 throughout; a parameter's gradient passes some 30 products of up
to 700 terms, 2^-24 each and independent: 1e-4 of its norm leaves a factor of 30.
"""
from __future__ import annotations

import pytest
import torch

from _inputs import SEED
from mamba_metal import MambaConfig, TinyMamba, linear_distillation_ref

VOCAB = 700
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def models(device, **over):
    kw = dict(vocab_size=VOCAB, d_model=64, n_layers=2, d_ff=128, max_seq_len=64, d_state=8, d_conv=4)
    kw.update(over)
    torch.manual_seed(SEED)
    plain = TinyMamba(MambaConfig(**kw)).to(device)
    fused = TinyMamba(MambaConfig(**kw, fuse_norm=True, fuse_loss=True)).to(device)
    fused.load_state_dict(plain.state_dict())
    g = torch.Generator().manual_seed(3)
    idx = torch.randint(0, VOCAB, (3, 41), generator=g).to(device)
    return plain, fused, idx


def grads_of(model, loss):
    model.zero_grad(set_to_none=True)
    loss.backward()
    return {k: p.grad for k, p in model.named_parameters()}


def same_grads(a, b):
    assert a.keys() == b.keys()
    for k in a:
        assert float((a[k] - b[k]).norm()) <= 1e-4 * float(b[k].norm()), k


@pytest.mark.parametrize("device", DEVICES)
def test_loss_and_gradients(device):
    plain, fused, idx = models(device)
    targets = idx[:, 1:].clone()
    targets[0, :5] = -100
    logits, want = plain(idx[:, :-1], targets)
    none, got = fused(idx[:, :-1], targets)
    assert logits is not None and none is None
    assert abs(got.item() - want.item()) <= 1e-5 * want.item()
    same_grads(grads_of(fused, got), grads_of(plain, want))


@pytest.mark.parametrize("device", DEVICES)
def test_logits_and_recurrent_cache(device):
    plain, fused, idx = models(device)
    with torch.no_grad():
        assert torch.allclose(fused(idx)[0], plain(idx)[0], atol=1e-5)
        cache: dict = {}
        fused(idx[:, :30], cache=cache)
        steps = [fused(idx[:, t:t + 1], cache=cache)[0][:, -1] for t in range(30, 36)]
        full = plain(idx[:, :36])[0][:, 30:]
    for t, s in enumerate(steps):
        assert torch.allclose(s, full[:, t], atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_distillation_through_the_model(device):
    plain, fused, idx = models(device)
    g = torch.Generator().manual_seed(5)
    index = torch.randint(-1, VOCAB, (3, 40, 6), generator=g).to(device)
    logits = torch.randn(3, 40, 6, generator=g).to(device)
    got = fused.distill_loss(idx[:, :-1], index, logits, temperature=2.0)
    want = linear_distillation_ref(plain.hidden(idx[:, :-1]), plain.head.weight, index, logits, 2.0)
    assert abs(got.item() - want.item()) <= 1e-5 * want.item()
    same_grads(grads_of(fused, got), grads_of(plain, want))


def test_a_model_without_blocks():
    _, fused, idx = models("cpu", n_layers=0)
    assert fused(idx, idx)[1].ndim == 0


@pytest.mark.gpu
def test_a_captured_training_step():
    """Both losses' steps in one graph, replayed on other tokens: the eager step's values."""
    _, fused, idx = models("cuda")
    g = torch.Generator().manual_seed(7)
    index = torch.randint(-1, VOCAB, (3, 40, 6), generator=g).cuda()
    logits = torch.randn(3, 40, 6, generator=g).cuda()
    other = torch.randint(0, VOCAB, (3, 41), generator=g).cuda()
    tokens = idx.clone()
    tokens_in, targets = tokens[:, :-1], tokens[:, 1:]

    def step():
        loss = fused(tokens_in, targets)[1] + fused.distill_loss(tokens_in, index, logits, 2.0)
        return loss.detach(), grads_of(fused, loss)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        tokens.copy_(other)
        want, want_grads = step()
        tokens.copy_(idx)
    torch.cuda.current_stream().wait_stream(side)
    fused.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    tokens.copy_(other)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    same_grads(grads, want_grads)
