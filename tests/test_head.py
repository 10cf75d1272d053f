"""The head's losses and the residual norm on the CPU: formulas, dispatch, refusals, C ABI checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mamba_metal import (_native, linear_cross_entropy, linear_distillation, residual_rms_norm)


def _head(rows=5, vocab=11, dim=6, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=gen, dtype=torch.float64)
    w = torch.randn(vocab, dim, generator=gen, dtype=torch.float64)
    return x, w, torch.randint(0, vocab, (rows,), generator=gen), gen


def test_cross_entropy_is_its_formula():
    x, w, target, _ = _head()
    target[2] = -100
    z = x @ w.t()
    rows = torch.logsumexp(z, 1) - z.gather(1, target.clamp(min=0)[:, None])[:, 0]
    rows[2] = 0
    assert torch.allclose(linear_cross_entropy(x, w, target, reduction="none"), rows)
    assert torch.allclose(linear_cross_entropy(x, w, target), rows.sum() / 4)
    assert torch.allclose(linear_cross_entropy(x, w, target, reduction="sum"), rows.sum())


def test_distillation_is_its_formula_and_reduces_to_cross_entropy():
    x, w, target, gen = _head()
    index = torch.tensor([[0, 3, 3], [1, -1, 2], [-1, -1, -1], [4, 5, 6], [7, 8, -1]])
    logits = torch.randn(5, 3, generator=gen, dtype=torch.float64)
    logits[3] = float("-inf")
    tau = 2.0
    log_q = torch.log_softmax(x @ w.t() / tau, 1)
    rows = torch.zeros(5, dtype=torch.float64)
    for m in (0, 1, 4):
        at = [j for j in range(3) if index[m, j] >= 0]
        p = torch.softmax(logits[m, at] / tau, 0)
        rows[m] = tau ** 2 * sum(p[i] * (p[i].log() - log_q[m, index[m, j]]) for i, j in enumerate(at))
    assert torch.allclose(linear_distillation(x, w, index, logits, tau, reduction="none"), rows)
    assert torch.allclose(linear_distillation(x, w, index, logits, tau), rows.sum() / 3)
    one = linear_distillation(x, w, target[:, None], torch.zeros(5, 1, dtype=torch.float64))
    assert torch.allclose(one, linear_cross_entropy(x, w, target))


def test_norm_is_its_formula():
    gen = torch.Generator().manual_seed(1)
    x, y, gate = (torch.randn(3, 4, 7, generator=gen, dtype=torch.float64) for _ in range(3))
    w, post, scale = (torch.randn(7, generator=gen, dtype=torch.float64) for _ in range(3))
    eps = 1e-3
    a = y * gate / (1 + torch.exp(-gate))
    b = post * a / torch.sqrt((a * a).mean(-1, keepdim=True) + eps)
    h = x + scale * b
    got_h, got_u = residual_rms_norm(x, y, w, post, gate, scale, eps)
    assert torch.allclose(got_h, h)
    assert torch.allclose(got_u, w * h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps))
    got_h, got_u = residual_rms_norm(x, y, w)
    assert torch.equal(got_h, x + y)


def test_ref_gradients_against_differences():
    x, w, target, gen = _head()
    logits = torch.randn(5, 2, generator=gen, dtype=torch.float64)
    index = torch.tensor([[0, 0], [1, -1], [2, 3], [-1, -1], [9, 10]])
    x.requires_grad_(True)
    w.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda a, b: linear_cross_entropy(a, b, target), (x, w))
    assert torch.autograd.gradcheck(lambda a, b: linear_distillation(a, b, index, logits, 2.0), (x, w))
    v = [torch.randn(5, 6, generator=gen, dtype=torch.float64).requires_grad_(True) for _ in range(2)]
    s = [torch.randn(6, generator=gen, dtype=torch.float64).requires_grad_(True) for _ in range(3)]
    assert torch.autograd.gradcheck(lambda *t: residual_rms_norm(x, t[0], t[2], t[3], t[1], t[4]), (*v, *s))


def test_dispatch_and_refusals_off_cuda():
    x, w, target, _ = _head()
    x, w = x.float(), w.float()
    index, logits = target[:, None], torch.zeros(5, 1)
    vec = torch.ones(6)
    calls = [lambda **k: linear_cross_entropy(x, w, target, **k),
             lambda **k: linear_distillation(x, w, index, logits, **k),
             lambda **k: residual_rms_norm(x, x, vec, **k)]
    for call in calls:
        call(impl="auto"), call(impl="torch")
        for impl in ("cuda", "metal"):
            with pytest.raises(RuntimeError, match="CUDA"):
                call(impl=impl)
        with pytest.raises(ValueError, match="scan_impl"):
            call(impl="nope")
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, target, reduction="median")
    with pytest.raises(ValueError, match="reduction"):
        linear_distillation(x, w, index, logits, reduction="median")
    for tau in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            linear_distillation(x, w, index, logits, temperature=tau)
    with pytest.raises(ValueError, match="shapes"):
        linear_distillation(x, w, index, logits[:, :0])
    with pytest.raises(ValueError, match="entries"):
        linear_distillation(x, w, index[:, :0], logits[:, :0])
    with pytest.raises(ValueError, match="entries"):
        linear_distillation(x, w, index.expand(5, 1025), logits.expand(5, 1025))
    with pytest.raises(ValueError, match="shapes"):
        residual_rms_norm(x, x[:2], vec)
    with pytest.raises(ValueError, match="shapes"):
        residual_rms_norm(x, x, vec[:5])
    with pytest.raises(ValueError, match="eps"):
        residual_rms_norm(x, x, vec, eps=-1.0)


def _p(v):
    return ctypes.c_void_p(v)


def test_c_entries_check_before_any_launch():
    """Fake pointers: every call here is refused before a launch."""
    lib = _native.load()
    bad, mis, ws_err = (_native.MMS_ERR_INVALID_ARG, _native.MMS_ERR_MISALIGNED, _native.MMS_ERR_WORKSPACE)
    ok = _p(0x10000)

    def ce_fwd(x=ok, ldx=16, w=ok, ldw=16, t=ok, red=1, loss=ok, kept=ok, ws=_p(0x20000), nb=1 << 40,
               m=4, v=8, d=16, ty=0):
        return lib.mms_linear_ce_fwd(x, ldx, w, ldw, t, -100, red, loss, kept, ws, nb, m, v, d, ty, None)

    assert ce_fwd(m=0) == bad and ce_fwd(v=0) == bad and ce_fwd(d=0) == bad
    assert ce_fwd(ldx=15) == bad and ce_fwd(ldw=15) == bad and ce_fwd(ty=2) == bad
    assert ce_fwd(red=3) == bad and ce_fwd(red=-1) == bad and ce_fwd(m=(1 << 24) + 1) == bad
    assert ce_fwd(v=(1 << 30) + 1) == bad and ce_fwd(d=(1 << 20) + 1, ldx=1 << 21, ldw=1 << 21) == bad
    assert ce_fwd(x=None) == bad and ce_fwd(t=None) == bad
    assert ce_fwd(loss=None) == bad and ce_fwd(kept=None) == bad
    assert ce_fwd(x=_p(0x10008)) == mis and ce_fwd(t=_p(0x10004)) == mis and ce_fwd(kept=_p(0x10008)) == mis
    need = lib.mms_head_workspace_size(4, 8, 16, 0, 0, 16, 16, 0)
    assert need > 0 and ce_fwd(nb=need - 1) == ws_err and ce_fwd(ws=None) == ws_err
    assert ce_fwd(ws=_p(0x20010)) == mis
    assert lib.mms_head_workspace_size(0, 8, 16, 0, 0, 16, 16, 0) == 0
    assert lib.mms_head_workspace_size(4, 8, 16, 1025, 0, 16, 16, 0) == 0
    assert lib.mms_head_kept_size(4, 0) > 0 and lib.mms_head_kept_size(4, 9) > lib.mms_head_kept_size(4, 1)
    assert lib.mms_head_kept_size(0, 0) == 0 and lib.mms_head_kept_size(4, 1025) == 0

    def kd_fwd(k=2, tau=1.0, logits=ok, nb=0):
        return lib.mms_linear_kd_fwd(ok, 16, ok, 16, ok, logits, k, tau, 1, ok, ok, _p(0x20000), nb, 4, 8, 16,
                                     1, None)

    assert kd_fwd() == ws_err and kd_fwd(k=0) == bad and kd_fwd(k=1025) == bad
    assert kd_fwd(tau=0.0) == bad and kd_fwd(tau=float("nan")) == bad and kd_fwd(logits=None) == bad

    def bwd(dl=ok, kept=ok, dx=ok, nb=0):
        return lib.mms_linear_ce_bwd(ok, 16, ok, 16, ok, -100, 1, dl, kept, dx, ok, _p(0x20000), nb, 4, 8, 16, 1,
                                     None)

    assert bwd() == ws_err and bwd(dl=None) == bad and bwd(kept=None) == bad and bwd(dx=_p(0x10008)) == mis
    assert lib.mms_linear_kd_bwd(ok, 16, ok, 16, ok, 2, 1.0, 1, None, ok, ok, ok, _p(0x20000), 0, 4, 8, 16, 1,
                                 None) == bad

    def norm(x=ok, gate=None, ldg=16, m=4, d=16, ty=0, stat=ok, eps=1e-6):
        return lib.mms_norm_fwd(x, ok, gate, ldg, ok, None, None, eps, ok, ok, stat, m, d, ty, None)

    assert norm(m=0) == bad and norm(d=0) == bad and norm(ty=5) == bad and norm(x=None) == bad
    assert norm(gate=ok, ldg=15) == bad and norm(eps=-1.0) == bad
    assert norm(eps=float("nan")) == bad and norm(m=(1 << 30) + 1) == bad and norm(d=(1 << 30) + 1) == bad
    assert norm(x=_p(0x10002)) == mis and norm(x=_p(0x10001), ty=1) == mis

    def norm_bwd(dx=ok, dy=_p(0x30000), post=None, nb=0):
        return lib.mms_norm_bwd(ok, ok, None, 16, ok, post, None, ok, ok, ok, dx, dy, None, ok, ok, None,
                                _p(0x20000), nb, 4, 16, 0, None)

    assert norm_bwd() == ws_err and norm_bwd(dx=None) == bad
    assert norm_bwd(dy=ok, post=ok) == bad and norm_bwd(dy=ok) == ws_err
