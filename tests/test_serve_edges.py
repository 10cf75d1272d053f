"""Corners of the packed calls and of sampling: nothing to do, one tap, infinite temperatures, default types."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import (MambaConfig, TinyMamba, causal_conv, causal_conv_packed, causal_conv_packed_ref,
                         sample_tokens, selective_scan_packed)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_temperature_draws_evenly_from_what_is_not_masked(device):
    z = torch.tensor([[3.0, -float("inf"), -50.0, 0.0]] * 4, device=device)
    u = torch.tensor([0.0, 0.3, 0.34, 0.9], device=device)
    token, logprob = sample_tokens(z, u, temperature=float("inf"), return_logprob=True)
    assert token.tolist() == [0, 0, 2, 3]
    # log(1 / 3) from exact counts: a logarithm and two roundings to float32
    assert torch.allclose(logprob, torch.full_like(logprob, 1 / 3).log(), rtol=2.0 ** -21, atol=0)


@pytest.mark.parametrize("device", DEVICES)
def test_a_top_k_beyond_any_row_keeps_all(device):
    z = torch.linspace(-1, 1, 9, device=device).expand(5, 9)
    u = torch.linspace(0, 0.99, 5, device=device)
    assert torch.equal(sample_tokens(z, u, top_k=2 ** 64 + 1), sample_tokens(z, u))
    with pytest.raises(TypeError):
        sample_tokens(z, u, top_k=2.5)


@pytest.mark.parametrize("device", DEVICES)
def test_calls_without_rows_hand_states_on(device):
    """An empty sequence's state goes on; one that starts from nothing leaves zeros, whatever the cache holds."""
    starts = torch.zeros(4, dtype=torch.int32, device=device)
    src, dst = torch.tensor([-1, 1, 3], device=device), torch.tensor([2, 0, -1], device=device)
    cache = torch.arange(4 * 8 * 4, dtype=torch.float32, device=device).view(4, 8, 4)
    cache[0], cache[3] = float("nan"), float("inf")
    want = cache.clone()
    want[2], want[0] = 0.0, cache[1]
    x, bc, aneg = (torch.zeros(n, m, device=device) for n, m in ((0, 8), (0, 4), (8, 4)))
    state = cache.clone()
    assert selective_scan_packed(x, x, aneg, bc, bc, state, starts, src, dst).shape == (0, 8)
    assert torch.equal(state.nan_to_num(7.0), want.nan_to_num(7.0))
    window = cache.clone()[:, :, :3].contiguous()
    assert causal_conv_packed(x, torch.zeros(8, 4, device=device), None, window, starts, src, dst).shape == (0, 8)
    assert torch.equal(window.nan_to_num(7.0), want[:, :, :3].nan_to_num(7.0))


@pytest.mark.parametrize("device", DEVICES)
def test_one_tap_needs_no_window(device):
    x, w, window = torch.randn(5, 8, device=device), torch.randn(8, 1, device=device), torch.empty(2, 8, 0, device=device)
    starts = torch.tensor([0, 2, 5], device=device)
    want = causal_conv_packed_ref(x.double(), w.double(), None, window.double(), starts)
    for got in (causal_conv_packed(x, w, None, window, starts), causal_conv(x[None], w)[0],
                causal_conv_packed(x, w, None, torch.empty(5, 8, 0, device=device))):
        # a product, then a SiLU (ex2 and a reciprocal, an argument rounded once)
        assert ((got - want).abs() <= want.abs() * ((x * w[:, 0]).abs() + 18) * 2.0 ** -24 * 1.2).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d_conv", [1, 2, 8])
def test_decoding_with_fused_convolution_of_any_taps(device, d_conv):
    torch.manual_seed(0)
    m = TinyMamba(MambaConfig(vocab_size=60, d_model=24, n_layers=2, d_ff=48, d_state=8, d_conv=d_conv,
                              fuse_conv=True)).to(device)
    idx = torch.randint(0, 60, (2, 12), device=device)
    cache = m.new_cache(2)
    with torch.no_grad():
        want = m(idx)[0][:, -1]
        starts = torch.tensor([0, 11, 22], device=device)
        m.serve(idx[:, :11].reshape(-1), cache, starts)
        assert torch.allclose(m.serve(idx[:, 11], cache), want, rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
def test_default_types_do_not_leak_into_the_calls():
    g = torch.Generator().manual_seed(0)
    x, w, dy = (torch.randn(s, generator=g).cuda() for s in ((2, 9, 8), (8, 4), (2, 9, 8)))
    bc, aneg, z = (torch.rand(s, generator=g).cuda() for s in ((9, 4), (8, 4), (9, 50)))
    starts, none = torch.tensor([0, 4, 9], device="cuda"), torch.tensor([-1, -1], device="cuda")

    def calls():
        wg = w.clone().requires_grad_()
        y = causal_conv(x, wg)
        y.backward(dy)
        state = torch.zeros(2, 8, 4, device="cuda", dtype=torch.float32)
        window = torch.zeros(2, 8, 3, device="cuda", dtype=torch.float32)
        return [y.detach(), wg.grad, causal_conv_packed(x[0], w, None, window, starts), window,
                selective_scan_packed(x[0], bc[:, :1].expand(9, 8), aneg, bc, bc, state, starts, none, torch.arange(2, device="cuda")), state,
                *sample_tokens(z, bc[:, 0], 0.7, 20, 0.9, return_logprob=True)]

    want = calls()
    torch.set_default_dtype(torch.float64)
    try:
        got = calls()
    finally:
        torch.set_default_dtype(torch.float32)
    for a, b in zip(want, got):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.gpu
def test_graphs_that_share_a_pool_and_calls_on_two_streams():
    """Long prompts (with a workspace) captured twice into one pool and replayed in turn, and run on two streams."""
    g = torch.Generator().manual_seed(0)
    d, n, rows = 256, 16, 2000
    x, dt = torch.randn(2, rows, d, generator=g).cuda(), (0.1 * torch.rand(2, rows, d, generator=g)).cuda()
    b, c = torch.randn(2, rows, n, generator=g).cuda(), torch.randn(2, rows, n, generator=g).cuda()
    aneg = (1 + torch.rand(d, n, generator=g)).cuda()
    starts = torch.tensor([0, 700, rows], device="cuda")
    states = [torch.zeros(2, d, n, device="cuda") for _ in range(2)]

    def call(i):
        return selective_scan_packed(x[i], dt[i], aneg, b[i], c[i], states[i], starts)

    want = [call(i) for i in range(2)]
    ends = [s.clone() for s in states]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(call(i))
        graphs.append(graph)
    for i in (0, 1, 1, 0):
        states[i].zero_()
        graphs[i].replay()
        assert torch.equal(outs[i], want[i]) and torch.equal(states[i], ends[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in states:
        s.zero_()
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i]) and torch.equal(states[i], ends[i])
