"""TinyMamba.serve with starts that break the rules: wrong rows, no access outside (a gather outside the
rows would end the process's CUDA context)."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import MambaConfig, TinyMamba, causal_conv_packed, selective_scan_packed

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def model(device):
    torch.manual_seed(0)
    return TinyMamba(MambaConfig(vocab_size=30, d_model=16, n_layers=2, d_ff=32, d_state=8)).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("starts", [[0, 3, 900], [0, 1 << 40, 5], [4, 2, 5], [-7, 2, 5], [0, 0, 5], [0, 2, -9]])
def test_bad_starts_give_some_rows(device, starts):
    m = model(device)
    idx = torch.arange(5, device=device)
    cache = m.new_cache(3)
    logits = m.serve(idx, cache, torch.tensor(starts, device=device), torch.tensor([0, 2], device=device))
    assert logits.shape == (2, 30) and torch.isfinite(logits).all()
    for block in cache["blocks"]:
        assert (block["h"][1] == 0).all() and (block["conv"][1] == 0).all()
    # and good ones after them
    good = m.serve(idx, m.new_cache(1), torch.tensor([0, 5], device=device))
    with torch.no_grad():
        assert torch.allclose(good, m(idx[None])[0][0, -1:], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("device", DEVICES)
def test_no_tokens(device):
    m = model(device)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    with pytest.raises(ValueError, match="idx is empty"):
        m.serve(none, m.new_cache(2), torch.tensor([0, 0, 0], device=device))
    assert m.serve(none, m.new_cache(2)).shape == (0, 30)
    assert m.serve(none, m.new_cache(2), torch.tensor([0], device=device)).shape == (0, 30)


def test_the_torch_forms_clamp_starts_as_the_kernels_do():
    x, w, bc, aneg = torch.rand(6, 4), torch.rand(4, 3), torch.rand(6, 4), torch.rand(4, 4)
    for starts, same in (([0, 3, 99], [0, 3, 6]), ([-4, 2, 6], [0, 2, 6]), ([2, 9, 50], [2, 6, 6])):
        got, want = [], []
        for lists, out in ((starts, got), (same, want)):
            window, state = torch.ones(2, 4, 2), torch.ones(2, 4, 4)
            out += [causal_conv_packed(x, w, None, window, torch.tensor(lists)), window,
                    selective_scan_packed(x, x, aneg, bc, bc, state, torch.tensor(lists)), state]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
