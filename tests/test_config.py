"""MambaConfig: options added later stand behind the older ones, and what the fused ones pass by."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import MambaConfig, TinyMamba


def test_positional_arguments_keep_their_places():
    cfg = MambaConfig(100, 64, 2, 128, 64, 8, 4, None, 0, 8, "torch", False, False, 0.002, 0.2, 1e-5)
    assert (cfg.scan_impl, cfg.fuse_proj, cfg.fuse_gate) == ("torch", False, False)
    assert (cfg.dt_min, cfg.dt_max, cfg.norm_eps) == (0.002, 0.2, 1e-5)
    assert (cfg.fuse_norm, cfg.fuse_loss) == (False, False)


@pytest.mark.parametrize("fuse", [False, True])
def test_which_modules_run(fuse):
    """With the flags off every module's forward runs; with them on what the config says does not."""
    model = TinyMamba(MambaConfig(50, 16, 2, 32, 32, 4, 4, fuse_norm=fuse, fuse_loss=fuse))
    ran = set()
    for name, module in model.named_modules():
        module.register_forward_hook(lambda m, a, out, name=name: ran.add(name))
    idx = torch.zeros(1, 5, dtype=torch.int64)
    model(idx, idx)
    passed_by = {"blocks.0", "blocks.1", "blocks.1.norm", "ln_f", "head"}
    assert (passed_by & ran == set()) if fuse else passed_by <= ran
    assert {"tok", "blocks.0.norm", "blocks.1.in_proj", "blocks.1.out_proj"} <= ran
