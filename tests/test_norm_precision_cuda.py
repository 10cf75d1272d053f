"""residual_rms_norm's gradients over the rows, held to the float32 of their sums.

dweight, dpost and dscale are sums over the rows of products whose magnitudes M are taken from
float64: dh' = dh + r2 (t - n mean(t n)) counts with |dh| + r2 (|t| + |n| mean|t n|). Each product errs
by at most (64 + dim / 64) 2^-24 of M (some dozens of operations, sums over a row as in test_norm_cuda.py),
and a sum passes a row's additions in a CTA (at most rows / 148 of them, one CTA a SM or more), those
over the CTAs (at most 8 a SM, 32 threads a column) and the threads (5, and slack to 10), 2^-24 of
sum(M) each. Then one rounding to the type. Every output and gradient is also held as a whole: the
roundings of a few dozen operations, each its own, are 2e-6 of the norm of a float32 result at
most (33 times 2^-24), and a bf16 one has its last rounding, 2^-8 at most, besides.
"""
from __future__ import annotations

import pytest
import torch

from _head_ref import U32, check_norm, u
from test_norm_cuda import BF16, DEV, F32, FLAGS, norm_inputs, on_device, run, want64

pytestmark = pytest.mark.gpu


def magnitudes(t, dh, du, eps=1e-6):
    """sum over the rows of M for dweight, and for the sums that dpost and dscale share."""
    t = {n: None if v is None else v.double() for n, v in t.items()}
    a = t["y"] if t["gate"] is None else t["y"] * t["gate"] * torch.sigmoid(t["gate"])
    v = a if t["post"] is None else a * torch.rsqrt(a.pow(2).mean(-1, keepdim=True) + eps)
    post, scale = (torch.ones_like(t["weight"]) if t[n] is None else t[n] for n in ("post", "scale"))
    h = t["x"] + post * scale * v
    r2 = torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    n, tw = h * r2, du.double() * t["weight"]
    # h itself is a sum: its error counts with the magnitudes of both parts
    big_n = (t["x"].abs() + (post * scale * v).abs()) * r2
    d = dh.double().abs() + r2 * (tw.abs() + big_n * (tw * n).abs().mean(-1, keepdim=True))
    sums = (d * v.abs()).sum(0)
    return {"dweight": (du.double().abs() * big_n).sum(0), "dpost": sums * scale.abs(), "dscale": sums * post.abs()}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("post,gate,scale", FLAGS)
@pytest.mark.parametrize("rows,dim", [(1, 640), (300, 640), (777, 1433), (5000, 72), (4100, 33), (9, 9000)])
def test_gradients_hold_the_bits_of_their_sums(rows, dim, post, gate, scale, dtype):
    t, dh, du = norm_inputs(rows, dim, dtype, post, gate, scale, seed=rows + dim)
    got, want = run(on_device(t), dh.to(DEV), du.to(DEV)), want64(t, dh, du)
    size = magnitudes(t, dh, du)
    steps = 64 + dim / 64 + -(-rows // 148) + 148 * 8 / 32 + 10
    for name, w in want.items():
        w, g = w.detach(), got[name].detach().cpu().double()
        check_norm(name, g, w, 2e-6 + (u(dtype) if dtype == BF16 else 0.0))
        if name in size:
            off, bound = (g - w).abs(), steps * U32 * size[name] + u(dtype) * w.abs()
            assert (off <= bound).all(), (name, float((off / bound).max()))
