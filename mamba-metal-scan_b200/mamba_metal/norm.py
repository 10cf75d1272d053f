"""The residual sum after a block fused with the norms around it (sm_100a).

    h, u = residual_rms_norm(x, y, weight, post_weight, gate, scale)

        a = y * silu(gate)                          (no gate: a = y)
        b = post_weight * a / sqrt(mean(a^2) + eps) (no post_weight: b = a)
        h = x + scale * b                           (no scale: h = x + b)
        u = weight * h / sqrt(mean(h^2) + eps)

x is the residual stream, y a block's output, h the stream after the block
and u the next block's input. The reference runs the sum and its RMSNorm as
separate PyTorch ops (mamba_metal/model.py:85-95, 256); here each direction
is one pass over the rows (csrc/mms_norm.cu).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from mamba_metal import _native
from mamba_metal.scan import _IMPLS

MAX_SIZE = 1 << 30    # rows, and columns, of the kernels (MMS_NORM_MAX)


def residual_rms_norm_ref(x, y, weight, post_weight=None, gate=None, scale=None, eps: float = 1e-6):
    """residual_rms_norm in PyTorch ops: float32 arithmetic (float64 for float64), results in x's type."""
    dtype = x.dtype
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    x, y, weight, post_weight, gate, scale = (None if t is None else t.to(wide) for t in
                                              (x, y, weight, post_weight, gate, scale))
    if gate is not None:
        y = y * F.silu(gate)
    if post_weight is not None:
        y = post_weight * y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps)
    h = x + (y if scale is None else scale * y)
    u = weight * h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    return h.to(dtype), u.to(dtype)


class ResidualRMSNormCUDA(torch.autograd.Function):
    """residual_rms_norm on (M, D) rows, one kernel each way (mms_norm_fwd / mms_norm_bwd)."""

    @staticmethod
    def forward(ctx, x, y, weight, post, gate, scale, eps):
        with _native.on_device(x.device):
            h, u, stat = _native.norm_fwd(x, y, gate, weight, post, scale, eps)
        ctx.save_for_backward(x, y, weight, post, gate, scale, stat)
        return h, u

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, du):
        x, y, weight, post, gate, scale, stat = ctx.saved_tensors
        with _native.on_device(x.device):
            dx, dy, dgate, dweight, dpost, dscale = _native.norm_bwd(
                x, y, gate, weight, post, scale, stat, dh.contiguous(), du.contiguous())
        return dx, dy, dweight, dpost, dgate, dscale, None


def _strided_rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, D) with unit column stride and one row stride >= D: a view where t's layout allows."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[0] == 1 or t.shape[1] == 1 or t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
        if t.stride() != (t.shape[1], 1):
            t = t.as_strided(t.shape, (t.shape[1], 1))
    return t


def residual_rms_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor,
                      post_weight: torch.Tensor = None, gate: torch.Tensor = None,
                      scale: torch.Tensor = None, eps: float = 1e-6, impl: str = "auto"):
    """(h, u): the residual stream after a block, and its norm (see the module docstring).

    x, y, gate (..., D), weight, post_weight, scale (D,); all float32 or all
    bfloat16 on the CUDA kernels ('auto' on CUDA tensors, 'cuda', 'metal'),
    with float32 arithmetic and u computed from h before its rounding.
    Elsewhere, or with 'torch', PyTorch ops. gate may be a view with a row
    stride. Differentiable once, with respect to every tensor.
    """
    if impl not in _IMPLS:
        raise ValueError(f"unknown scan_impl {impl!r}; want 'auto', 'cuda', 'metal' or 'torch'")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative; got {eps}")
    rows = [t for t in (x, y, gate) if t is not None]
    vectors = [t for t in (weight, post_weight, scale) if t is not None]
    shape = x.shape
    if x.dim() < 1 or any(t.shape != shape for t in rows) or any(t.shape != shape[-1:] for t in vectors):
        raise ValueError("bad shapes: x, y, gate " + ", ".join(str(tuple(t.shape)) for t in rows)
                         + "; weight, post_weight, scale "
                         + ", ".join(str(tuple(t.shape)) for t in vectors))
    if impl == "torch" or (impl == "auto" and not x.is_cuda):
        return residual_rms_norm_ref(x, y, weight, post_weight, gate, scale, eps)
    tensors = rows + vectors
    device, dtype = x.device, x.dtype
    if not x.is_cuda or any(t.device != device for t in tensors):
        raise RuntimeError(f"scan_impl={impl!r} needs every tensor on the same CUDA device; saw "
                           + ", ".join(str(t.device) for t in tensors))
    if dtype not in (torch.float32, torch.bfloat16) or any(t.dtype != dtype for t in tensors):
        raise RuntimeError("residual_rms_norm takes float32 or bfloat16, all tensors alike; got "
                           + ", ".join(str(t.dtype) for t in tensors))
    if x.shape[-1] > MAX_SIZE or x.numel() > MAX_SIZE * x.shape[-1]:
        raise ValueError(f"residual_rms_norm takes up to {MAX_SIZE} rows and columns; got {tuple(x.shape)}")
    if x.numel() == 0:
        return residual_rms_norm_ref(x, y, weight, post_weight, gate, scale, eps)
    d = shape[-1]
    flat = x.dim() == 2                     # no views, so no autograd nodes, where none are needed
    args = (x.contiguous() if flat else x.reshape(-1, d).contiguous(),
            y.contiguous() if flat else y.reshape(-1, d).contiguous(), weight.contiguous(),
            None if post_weight is None else post_weight.contiguous(),
            None if gate is None else _strided_rows(gate), None if scale is None else scale.contiguous())
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        h, u = ResidualRMSNormCUDA.apply(*args, eps)
    else:
        x, y, weight, post_weight, gate, scale = args
        with _native.on_device(device):
            h, u, _ = _native.norm_fwd(x, y, gate, weight, post_weight, scale, eps, keep=False)
    return (h, u) if flat else (h.view(shape), u.view(shape))
