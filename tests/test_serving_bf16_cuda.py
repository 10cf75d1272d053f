"""TinyMamba in bf16 served by the kernels: every call that its blocks make, on the rows, windows and states
that they have there, against float64 within the bounds of tests/_serve_ref.py."""
from __future__ import annotations

import pytest
import torch

import mamba_metal.model as model_module
from _serve_ref import close, conv_bound, scan_bound
from mamba_metal import MambaConfig, TinyMamba, sample_tokens, sample_tokens_ref
from mamba_metal.packed import places_of

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
LENS = (5, 1, 70, 3)


def model(**kw):
    torch.manual_seed(0)
    m = TinyMamba(MambaConfig(**{**dict(vocab_size=60, d_model=24, n_layers=2, d_ff=48, d_state=8), **kw}))
    with torch.no_grad():
        for b in m.blocks:
            b.conv.bias.normal_()
            b.D_skip.normal_()
    return m.to(BF16).cuda()


def sequences(x, cache, starts, slots, out_slots):
    return places_of(x.shape[0], *(None if v is None else v.cpu() for v in (starts, slots, out_slots)), cache.shape[0])


@pytest.fixture
def calls(monkeypatch):
    """Checks each packed call of the model; the list of what it checked."""
    seen = []
    conv, scan = model_module.causal_conv_packed, model_module.selective_scan_packed

    def checked_conv(x, weight, bias, window, starts=None, slots=None, out_slots=None, impl="auto"):
        assert x.dtype == window.dtype == weight.dtype == BF16 and x.stride(0) == 2 * x.shape[1]     # a half of in_proj's
        old, k = window.clone(), weight.shape[-1]
        y = conv(x, weight, bias, window, starts, slots, out_slots, impl=impl)
        left = old.clone()
        for first, end, src, dst in sequences(x, window, starts, slots, out_slots):
            rows = torch.cat([torch.zeros(k - 1, x.shape[1], dtype=BF16, device="cuda") if src is None else old[src].t(), x[first:end]])
            want, bound = conv_bound(rows[None].cpu(), weight.squeeze(1).cpu(), bias.cpu(), True, BF16)
            close(y[first:end], want[0, k - 1:], bound[0, k - 1:], "convolution")
            if dst is not None:
                left[dst] = rows[rows.shape[0] - (k - 1):].t()
        assert torch.equal(window, left)
        seen.append(("conv", x.shape[0]))
        return y

    def checked_scan(x, dt, aneg, b_in, c_in, state, starts=None, slots=None, out_slots=None, z=None, d_skip=None, dt_range=None,
                     impl="auto"):
        assert x.dtype == dt.dtype == b_in.dtype == z.dtype == BF16 and state.dtype == torch.float32
        old = state.clone()
        y = scan(x, dt, aneg, b_in, c_in, state, starts, slots, out_slots, z=z, d_skip=d_skip, dt_range=dt_range, impl=impl)
        on_host = [t.cpu() for t in (x, dt, aneg, b_in, c_in, old)]
        seqs = sequences(x, state, starts, slots, out_slots)
        wy, by, ws, bs = scan_bound(*on_host, seqs, z.cpu(), d_skip.cpu(), dt_range, BF16)
        for first, end, _, _ in seqs:
            close(y[first:end], wy[first:end], by[first:end], "scan")
        close(state, ws, bs, "state")
        seen.append(("scan", x.shape[0]))
        return y

    monkeypatch.setattr(model_module, "causal_conv_packed", checked_conv)
    monkeypatch.setattr(model_module, "selective_scan_packed", checked_scan)
    return seen


@pytest.mark.parametrize("kw", [dict(), dict(fuse_norm=True), dict(d_conv=2, d_state=20, d_inner=33), dict(d_state=64)])
def test_serve(kw, calls):
    """Prompts in places out of order, pieces and single tokens among them, then a token each, two from one place."""
    m = model(**kw)
    g = torch.Generator().manual_seed(1)
    ps = [torch.randint(0, 60, (n,), generator=g).cuda() for n in LENS]
    cache = m.new_cache(6)
    slots, none = torch.tensor([4, 0, 5, 2], device="cuda"), torch.full((4,), -1, device="cuda")
    starts = torch.tensor([0, *LENS], device="cuda").cumsum(0)
    for logits in (m.serve(torch.cat(ps), cache, starts, none, slots),
                   m.serve(torch.cat(ps), cache, starts.int(), slots),
                   m.serve(torch.arange(4, device="cuda"), cache, None, slots[[0, 1, 2, 2]], torch.tensor([4, 0, 1, 3], device="cuda"))):
        assert logits.shape == (4, 60) and logits.dtype == BF16 and torch.isfinite(logits).all()
        u = torch.rand(4, generator=g).cuda()
        for settings in (dict(), dict(top_k=5, temperature=0.7), dict(top_p=0.8)):
            assert torch.equal(sample_tokens(logits, u, **settings), sample_tokens_ref(logits, u, **settings)[0])
    assert calls == [("conv", 79), ("scan", 79)] * 4 + [("conv", 4), ("scan", 4)] * 2


def test_generate_is_serving_step_by_step(calls):
    m = model(fuse_norm=True)
    g = torch.Generator().manual_seed(2)
    ps = [torch.randint(0, 60, (n,), generator=g).cuda() for n in LENS]
    u = torch.rand(5, 4, generator=g).cuda()
    out = m.generate(ps, 5, temperature=0.9, top_k=30, uniform=u)
    cache, idx = m.new_cache(4), torch.cat(ps)
    for i in range(5):
        logits = m.serve(idx, cache, torch.tensor([0, *LENS], device="cuda").cumsum(0) if i == 0 else None)
        idx = sample_tokens(logits, u[i], 0.9, 30)
        assert torch.equal(idx, out[:, i])
    assert len(calls) == 2 * 2 * 2 * 5
