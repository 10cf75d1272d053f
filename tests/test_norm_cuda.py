"""residual_rms_norm on the GPU (mms_norm_fwd, mms_norm_bwd) against float64 autograd.

Bounds: an output element is a few dozen float32 operations on quantities no larger than the
scale given beside it, and is rounded once: at most (64 + dim / 64) 2^-24 of that scale (a row's
sums run over at most dim / 32 terms a lane and five levels of lanes) plus u(dtype) of the value.
A sum over rows adds (rows + 64) 2^-24 of the sum of magnitudes.
"""
from __future__ import annotations

import pytest
import torch

from _head_ref import U32, u
from mamba_metal import _native, residual_rms_norm, residual_rms_norm_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("x", "y", "weight", "post", "gate", "scale")


def norm_inputs(rows, dim, dtype, post, gate, scale, seed=0, strided=True):
    gen = torch.Generator().manual_seed(seed)
    t = dict(x=2 * torch.randn(rows, dim, generator=gen), y=torch.randn(rows, dim, generator=gen),
             weight=1 + 0.2 * torch.randn(dim, generator=gen), post=None, gate=None, scale=None)
    if post:
        t["post"] = 1 + 0.2 * torch.randn(dim, generator=gen)
    if gate:
        t["gate"] = 2 * torch.randn(rows, dim, generator=gen)
    if scale:
        t["scale"] = 0.5 + 0.2 * torch.randn(dim, generator=gen)
    t = {n: None if v is None else v.to(dtype) for n, v in t.items()}
    return t, torch.randn(rows, dim, generator=gen).to(dtype), torch.randn(rows, dim, generator=gen).to(dtype)


def on_device(t, strided=True):
    out = {}
    for n, v in t.items():
        if v is not None:
            if n == "gate" and strided:
                full = torch.full((v.shape[0], 2 * v.shape[1]), float("nan"), dtype=v.dtype, device=DEV)
                full[:, v.shape[1]:] = v.to(DEV)
                v = full[:, v.shape[1]:]
            v = v.to(DEV).detach().requires_grad_(True)
        out[n] = v
    return out


def run(t, dh, du, eps=1e-6, impl="auto"):
    h, uu = residual_rms_norm(t["x"], t["y"], t["weight"], t["post"], t["gate"], t["scale"], eps, impl=impl)
    names = [n for n in NAMES if t[n] is not None]
    grads = torch.autograd.grad([h, uu], [t[n] for n in names], [dh, du])
    return dict(h=h, u=uu, **{"d" + n: gr for n, gr in zip(names, grads)})


def want64(t, dh, du, eps=1e-6):
    t = {n: None if v is None else v.double().requires_grad_(True) for n, v in t.items()}
    return run(t, dh.double(), du.double(), eps, impl="torch")


def compare(t, dh, du, got, eps=1e-6):
    want = want64(t, dh, du, eps)
    rows, dim = t["x"].shape
    dtype = t["x"].dtype
    few = (64 + dim / 64) * U32
    for name, w in want.items():
        w, g = w.detach(), got[name].detach().cpu().double()
        assert got[name].dtype == dtype and g.shape == w.shape, name
        if w.dim() == 2:
            # a row's elements come from quantities within the row: its largest output and inputs
            scale = w.abs().amax(1, keepdim=True) + 1
            if name in ("dx", "dy", "dgate"):
                scale = scale + dh.double().abs().amax(1, keepdim=True)
            bound = few * 8 * scale + u(dtype) * w.abs()
        else:
            bound = (rows + 64) * U32 * 8 * (rows ** 0.5 + 8) * max(1.0, float(w.abs().max()) / rows ** 0.5) \
                + u(dtype) * w.abs()
        off = (g - w).abs()
        assert torch.isfinite(g).all() and (off <= bound).all(), (name, float((off / bound).max()))


FLAGS = [(False, False, False), (True, False, False), (False, True, True), (True, True, True), (False, False, True),
         (False, True, False)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("post,gate,scale", FLAGS)
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 640), (7, 33), (3, 4), (40, 1433), (300, 640), (65, 2048), (5, 9000)])
def test_norm_matches_float64(rows, dim, post, gate, scale, dtype):
    t, dh, du = norm_inputs(rows, dim, dtype, post, gate, scale, seed=rows + dim)
    if dim == 1:                                  # a norm of one element: sign only, gradients cancel
        t["x"] += 4
    compare(t, dh, du, run(on_device(t), dh.to(DEV), du.to(DEV)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_rows_and_wide_rows(dtype):
    for rows, dim in ((5000, 72), (2, 40000)):
        t, dh, du = norm_inputs(rows, dim, dtype, True, True, True, seed=rows)
        compare(t, dh, du, run(on_device(t), dh.to(DEV), du.to(DEV)))


def test_rows_of_zeros_and_of_large_values():
    t, dh, du = norm_inputs(6, 96, F32, True, False, False, seed=1)
    t["x"][1], t["y"][1] = 0, 0
    t["x"][2] *= 1e15
    got = run(on_device(t), dh.to(DEV), du.to(DEV))
    assert (got["u"][1] == 0).all() and (got["h"][1] == 0).all()
    assert all(torch.isfinite(v).all() for v in got.values())
    want = want64(t, dh, du)
    assert torch.allclose(got["u"].cpu().double(), want["u"], rtol=1e-5, atol=1e-5)
    # rows do not mix: a NaN row leaves the others as they were
    t["x"][4] = float("nan")
    again = run(on_device(t), dh.to(DEV), du.to(DEV))
    keep = torch.arange(6) != 4
    for n in ("h", "u", "dx", "dy"):
        assert torch.equal(again[n][keep], got[n][keep]) and torch.isnan(again[n][4]).all()


def test_layouts_and_unaligned_bases():
    t, dh, du = norm_inputs(33, 72, BF16, True, True, True, seed=2)
    base = run(on_device(t), dh.to(DEV), du.to(DEV))
    d = on_device(t, strided=False)
    buf = torch.empty(33 * 72 + 1, dtype=BF16, device=DEV)
    for n in ("x", "y", "gate"):                                       # bases 2 bytes off
        b = buf.clone()
        b[1:] = t[n].to(DEV).reshape(-1)
        d[n] = b[1:].view(33, 72).detach().requires_grad_(True)
    got = run(d, dh.to(DEV), du.to(DEV))
    for n in base:
        assert torch.equal(base[n], got[n]) or torch.allclose(base[n].float(), got[n].float(), rtol=2 ** -7, atol=1e-6), n
    # leading dimensions, transposed x, expanded upstream gradients
    x3 = t["x"].to(DEV).reshape(3, 11, 72).transpose(0, 1).requires_grad_(True)
    y3 = t["y"].to(DEV).reshape(3, 11, 72).transpose(0, 1).requires_grad_(True)
    h, uu = residual_rms_norm(x3, y3, t["weight"].to(DEV))
    assert h.shape == x3.shape
    (h.sum() + uu.sum()).backward()
    hr, ur = residual_rms_norm_ref(x3.detach().double(), y3.detach().double(), t["weight"].to(DEV).double())
    assert torch.allclose(h.double(), hr, rtol=2 ** -8, atol=0)
    assert x3.grad.shape == x3.shape and torch.equal(x3.grad, y3.grad)


def test_one_output_alone_and_the_same_tensor_twice():
    t, dh, du = norm_inputs(20, 64, F32, False, False, False, seed=3)
    d = on_device(t)
    h, uu = residual_rms_norm(d["x"], d["y"], d["weight"])
    gx, gy = torch.autograd.grad(uu, [d["x"], d["y"]], du.to(DEV), retain_graph=True)
    zero = torch.zeros_like(dh)
    ref = want64(t, zero, du)
    assert torch.allclose(gx.cpu().double(), ref["dx"], rtol=1e-5, atol=1e-6) and torch.equal(gx, gy)
    x = d["x"]
    h, uu = residual_rms_norm(x, x, d["weight"])                       # h = 2 x
    (g2,) = torch.autograd.grad([h, uu], x, [dh.to(DEV), du.to(DEV)])
    x64 = t["x"].double().requires_grad_(True)
    h64, u64 = residual_rms_norm(x64, x64, t["weight"].double(), impl="torch")
    (w2,) = torch.autograd.grad([h64, u64], x64, [dh.double(), du.double()])
    assert torch.allclose(g2.cpu().double(), w2, rtol=1e-5, atol=1e-5)


def test_gradient_against_differences():
    """Central differences of the kernel's sum(h dh + u du) along a direction, h^2 / 6 of a third
    derivative below 60 a row element here, and the sums' roundings over h."""
    t, dh, du = norm_inputs(8, 48, F32, True, True, True, seed=4)
    d = on_device(t)
    got = run(d, dh.to(DEV), du.to(DEV))
    gen = torch.Generator().manual_seed(5)
    h = 2.0 ** -7
    for n in NAMES:
        v = torch.randn(t[n].shape, generator=gen)
        v = v / v.norm()

        def f(s):
            q = {k: None if a is None else a.detach() for k, a in d.items()}
            q[n] = q[n] + s * v.to(DEV)
            a, b = residual_rms_norm(q["x"], q["y"], q["weight"], q["post"], q["gate"], q["scale"])
            return float((a.double() * dh.to(DEV).double()).sum() + (b.double() * du.to(DEV).double()).sum())

        slope = float((got["d" + n].cpu().double() * v.double()).sum())
        bound = h * h / 6 * 60 + 2 * 64 * U32 * 8 * 48 / h / 8
        assert abs((f(h) - f(-h)) / (2 * h) - slope) <= bound, n


def test_deterministic_streams_and_graphs():
    t, dh, du = norm_inputs(700, 640, F32, True, True, True, seed=6)
    d = on_device(t)
    dh, du = dh.to(DEV), du.to(DEV)
    a = {n: v.detach() for n, v in run(d, dh, du).items()}
    d = on_device(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(d, dh, du)
        side.synchronize()
    assert all(torch.equal(a[n], b[n]) for n in a)
    del b
    d = on_device(t)                    # leaves that no eager graph has met
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = {n: v.detach() for n, v in run(d, dh, du).items()}
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a[n], c[n]) for n in a)


def test_two_streams_at_once():
    """Workspaces and statistics of calls that run at the same time are their own."""
    jobs = []
    for i in range(3):
        t, dh, du = norm_inputs(900 + i, 1024, BF16, True, True, True, seed=20 + i)
        dh, du = dh.to(DEV), du.to(DEV)
        want = {n: v.detach() for n, v in run(on_device(t), dh, du).items()}
        jobs.append((t, dh, du, want, torch.cuda.Stream()))
    ready = [on_device(t) for t, *_ in jobs]
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(4):
        for (_, dh, du, _, stream), d, g in zip(jobs, ready, got):
            with torch.cuda.stream(stream):
                g.append({n: v.detach() for n, v in run(d, dh, du).items()})
    torch.cuda.synchronize()
    for (_, _, _, want, _), g in zip(jobs, got):
        assert all(torch.equal(want[n], one[n]) for one in g for n in want)


def test_gpu_refusals_and_empty_rows():
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    with pytest.raises(RuntimeError, match="alike"):
        residual_rms_norm(x, x, w.bfloat16())
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        residual_rms_norm(x.half(), x.half(), w.half())
    with pytest.raises(RuntimeError, match="same CUDA"):
        residual_rms_norm(x, x, w.cpu())
    h, uu = residual_rms_norm(x[:0], x[:0], w)
    assert h.shape == (0, 8) and uu.shape == (0, 8)
    with pytest.raises(ValueError, match="up to"):      # a view: refused before anything is copied
        long = x[:1, :1].expand((1 << 30) + 1, 1)
        residual_rms_norm(long, long, w[:1])
    assert _native.device_status() == _native.MMS_OK
