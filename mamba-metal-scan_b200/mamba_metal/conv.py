"""The block's short causal convolution with its SiLU on NVIDIA B200 (sm_100a).

    causal_conv(x, weight, bias)                     (B, T, D), forward and backward
    causal_conv_packed(x, weight, bias, window, ..)  packed prompts and single tokens, inference

    pre[t, d] = bias[d] + sum_k weight[d, k] x[t - K + 1 + k, d],   y = silu(pre), or pre

Channels stay innermost and x may be a view with strides, such as the half of in_proj's
output that the block convolves; the reference transposes to channels first, runs
nn.Conv1d and SiLU and transposes back (mamba_metal/model.py:175-177, 214-219). Kernels in
csrc/mms_conv.cu, dispatch as in `mamba_metal.scan`: 'auto' runs them on CUDA tensors and
PyTorch ops elsewhere, 'cuda' / 'metal' force them, 'torch' forces PyTorch ops.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from mamba_metal import _native
from mamba_metal.packed import (_FLOATS, _nothing_packed, check_lists, dispatch, int_list, places_of, rows_of,
                                same_device)

MAX_TAPS = 8          # the kernels' (MMS_CONV_MAX_K)


def _taps(weight, d: int):
    """weight as (D, K); nn.Conv1d's (D, 1, K) too."""
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight.squeeze(1)
    if weight.dim() != 2 or weight.shape[0] != d or weight.shape[1] < 1:
        raise ValueError(f"weight must be ({d}, taps) or ({d}, 1, taps); got {tuple(weight.shape)}")
    return weight


def _tangent(t) -> bool:
    """Whether t carries a forward-mode derivative (a kernel would drop it; the autograd function refuses)."""
    return unpack_dual(t).tangent is not None


def _wide(x):
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def causal_conv_ref(x, weight, bias=None, silu: bool = True):
    """causal_conv in PyTorch ops: float32 arithmetic (float64 for float64), the result in x's type."""
    w = _taps(weight, x.shape[-1]).to(_wide(x))
    k = w.shape[1]
    rows = F.pad(x.to(_wide(x)), (0, 0, k - 1, 0))
    y = sum(w[:, j] * rows[:, j:j + x.shape[1]] for j in range(k))
    if bias is not None:
        y = y + bias.to(_wide(x))
    return (F.silu(y) if silu else y).to(x.dtype)


class CausalConvCUDA(torch.autograd.Function):
    """causal_conv on x (B, T, D), weight (D, K), bias (D) or None (mms_conv_fwd / mms_conv_bwd)."""

    @staticmethod
    def forward(ctx, x, weight, bias, silu):
        with _native.on_device(x.device):
            y = _native.conv_fwd(x, weight, bias, silu)
        ctx.save_for_backward(x, weight, bias)
        ctx.silu = silu
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        with _native.on_device(x.device):
            return (*_native.conv_bwd(x, weight, bias, dy.contiguous(), ctx.silu), None)


def _check_kernel(what, x, weight, bias, window=None):
    same_device(what, x, (weight, bias, window))
    dtype = x.dtype
    if dtype not in _FLOATS or weight.dtype != dtype or (bias is not None and bias.dtype != dtype) \
            or (window is not None and window.dtype != dtype):
        raise RuntimeError(f"{what} takes float32 or bfloat16, all tensors alike; got "
                           + ", ".join(str(t.dtype) for t in (x, weight, bias, window) if t is not None))
    if weight.shape[1] > MAX_TAPS:
        raise ValueError(f"{what} takes up to {MAX_TAPS} taps on CUDA; got {weight.shape[1]} "
                         "(impl='torch' takes any number)")
    d = x.shape[-1]
    if x.numel() > _native.SERVE_MAX * max(1, d) or d > _native.SERVE_MAX_DIM:
        raise ValueError(f"{what} takes up to {_native.SERVE_MAX} rows and {_native.SERVE_MAX_DIM} channels; "
                         f"got {tuple(x.shape)}")


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor = None, silu: bool = True,
                impl: str = "auto"):
    """Depthwise causal convolution over dim 1 of x (B, T, D), with SiLU unless silu is False.

    weight (D, K) or nn.Conv1d's (D, 1, K), bias (D,) or None; y (B, T, D) contiguous. Before a
    sequence's first row stand zeros. All float32 or all bfloat16 on the CUDA kernels
    (float32 arithmetic, K up to 8). Differentiable once, with respect to every tensor, in
    reverse mode; on the kernels a forward-mode tangent is refused.
    """
    if x.dim() != 3:
        raise ValueError(f"x must be (batch, time, channels); got {tuple(x.shape)}")
    weight = _taps(weight, x.shape[2])
    if bias is not None and bias.shape != (x.shape[2],):
        raise ValueError(f"bias must be ({x.shape[2]},); got {tuple(bias.shape)}")
    if not dispatch(impl, x):
        return causal_conv_ref(x, weight, bias, silu)
    _check_kernel("causal_conv", x, weight, bias)
    if x.numel() == 0:
        return causal_conv_ref(x, weight, bias, silu)
    if x.stride(2) != 1 and x.shape[2] > 1:
        x = x.contiguous()
    weight = weight if weight.is_contiguous() else weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                     or (bias is not None and bias.requires_grad))) \
            or _tangent(x) or _tangent(weight) or (bias is not None and _tangent(bias)):
        return CausalConvCUDA.apply(x, weight, bias, bool(silu))
    with _native.on_device(x.device):
        return _native.conv_fwd(x, weight, bias, silu)


@torch.no_grad()
def causal_conv_packed_ref(x, weight, bias, window, starts=None, slots=None, out_slots=None, silu: bool = True):
    """causal_conv_packed in PyTorch ops (any device and float type; reads the lists on the host)."""
    w = _taps(weight, x.shape[-1])
    k = w.shape[1]
    y, left = torch.zeros_like(x), []
    for first, end, src, dst in places_of(x.shape[0], starts, slots, out_slots, window.shape[0]):
        old = x.new_zeros(k - 1, x.shape[1]) if src is None else window[src].t()
        rows = torch.cat([old, x[first:end]])
        if end > first:
            y[first:end] = causal_conv_ref(rows[None], w, bias, silu)[0, k - 1:]
        if dst is not None:
            left.append((dst, rows[end - first:].t()))
    for dst, rows in left:
        window[dst] = rows
    return y


def causal_conv_packed(x: torch.Tensor, weight: torch.Tensor, bias, window: torch.Tensor,
                       starts: torch.Tensor = None, slots: torch.Tensor = None,
                       out_slots: torch.Tensor = None, silu: bool = True, impl: str = "auto"):
    """The convolution over packed sequences that go on from `window`; updates it, returns y (L, D).

    x (L, D) rows (strided views too), window (places, D, K - 1) in x's type, contiguous: the
    K - 1 inputs before each sequence's next row, oldest first, as in TinyMamba's cache; the
    lists as in `mamba_metal.packed`. Not differentiable.
    """
    if x.dim() != 2:
        raise ValueError(f"x must be (rows, channels); got {tuple(x.shape)}")
    weight = _taps(weight, x.shape[1])
    k = weight.shape[1]
    if bias is not None and bias.shape != (x.shape[1],):
        raise ValueError(f"bias must be ({x.shape[1]},); got {tuple(bias.shape)}")
    if window.dim() != 3 or window.shape[1:] != (x.shape[1], k - 1):
        raise ValueError(f"window must be (places, {x.shape[1]}, {k - 1}); got {tuple(window.shape)}")
    count = check_lists(x.shape[0], window.shape[0], starts, slots, out_slots, x)
    if not dispatch(impl, x):
        return causal_conv_packed_ref(x, weight, bias, window, starts, slots, out_slots, silu)
    _check_kernel("causal_conv_packed", x, weight, bias, window)
    if not window.is_contiguous():
        raise ValueError(f"window must be contiguous (it is updated in place); got strides {window.stride()}")
    if window.shape[0] > _native.SERVE_MAX or count > _native.SERVE_MAX:
        raise ValueError(f"causal_conv_packed takes up to {_native.SERVE_MAX} sequences and places")
    if x.numel() == 0 or count == 0 or window.shape[0] == 0:
        return _nothing_packed(x, window, count, slots, out_slots)
    weight = weight if weight.is_contiguous() else weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    with _native.on_device(x.device):
        return _native.conv_packed(rows_of(x), weight, bias, window, int_list(starts), int_list(slots),
                                   int_list(out_slots), count, silu)
