"""MambaConfig by position: options added later stand behind the older ones."""
from __future__ import annotations

from mamba_metal import MambaConfig


def test_positional_arguments_keep_their_places():
    cfg = MambaConfig(100, 64, 2, 128, 64, 8, 4, None, 0, 8, "torch", False, False, 0.002, 0.2, 1e-5)
    assert (cfg.scan_impl, cfg.fuse_proj, cfg.fuse_gate) == ("torch", False, False)
    assert (cfg.dt_min, cfg.dt_max, cfg.norm_eps) == (0.002, 0.2, 1e-5)
    assert (cfg.fuse_norm, cfg.fuse_loss) == (False, False)
