"""Losses of a language model's head without its logits, on NVIDIA B200 (sm_100a).

    linear_cross_entropy(x, weight, target)       softmax cross entropy of x W^T
    linear_distillation(x, weight, index, logits) KL divergence from a teacher's top k

x (..., D) are the model's last hidden states, weight (V, D) is the head. The
(rows, V) logits never exist as a whole: the forward keeps one log-sum-exp a
row, the backward computes the logits again in pieces of the vocabulary (see
csrc/mms_head.cu). The reference model computes them and calls PyTorch's cross
entropy (mamba_metal/model.py:293-297).

Dispatch as in `mamba_metal.scan`: 'auto' runs the CUDA kernels on CUDA
tensors and PyTorch ops elsewhere, 'cuda' / 'metal' force the kernels, 'torch'
forces PyTorch ops. The kernels take float32 or bfloat16 (x and weight alike)
and give a float32 loss; gradients have x's and weight's type, and with bf16 come
from probabilities held to 2^-11 of each (to 2^-17 up to 256 rows). float32
products keep 22 bits of w's elements down to 2^-16 of its largest, below that an
absolute 2^-39 of it.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from mamba_metal import _native
from mamba_metal.scan import _IMPLS

MAX_K = 1024          # entries a row of linear_distillation's teacher lists (MMS_HEAD_MAX_K)
# the kernels' largest sizes (MMS_HEAD_MAX_ROWS, _VOCAB, _DIM)
MAX_ROWS, MAX_VOCAB, MAX_DIM = 1 << 24, 1 << 30, 1 << 20


def _reduce(rows, counts, reduction: str):
    if reduction == "none":
        return rows
    return rows.sum() / counts.sum() if reduction == "mean" else rows.sum()


def _logits(x, weight, counts):
    """x W^T, float32 at least, with zeros for the rows that do not count, whatever x holds there."""
    z = F.linear(torch.where(counts[..., None], x, torch.zeros((), dtype=x.dtype, device=x.device)), weight)
    return z.float() if x.dtype in (torch.bfloat16, torch.float16) else z


def _loud(values, bad):
    """values, NaN with NaN gradients where bad."""
    return values * torch.where(bad, float("nan"), 1.0).to(values.dtype)


def linear_cross_entropy_ref(x, weight, target, ignore_index: int = -100, reduction: str = "mean"):
    """linear_cross_entropy in PyTorch ops, with the logits (any device and float type)."""
    vocab, index = weight.shape[0], target.reshape(-1).long()
    counts = index != ignore_index
    rows = F.cross_entropy(_logits(x.reshape(-1, x.shape[-1]), weight, counts), index.clamp(0, vocab - 1), reduction="none")
    rows = torch.where(counts, _loud(rows, counts & ((index < 0) | (index >= vocab))), torch.zeros_like(rows))
    return _reduce(rows.reshape(target.shape), counts, reduction)


def linear_distillation_ref(x, weight, teacher_index, teacher_logits, temperature: float = 1.0,
                            reduction: str = "mean"):
    """linear_distillation in PyTorch ops, with the logits (any device and float type)."""
    index, vocab = teacher_index.long(), weight.shape[0]
    valid = index >= 0
    dtype = x.dtype if x.dtype == torch.float64 else torch.float32
    t = (teacher_logits.to(dtype) / temperature).masked_fill(~valid, float("-inf"))
    some = ~(t == float("-inf")).all(-1)
    logits = _logits(x, weight, some)
    # a row without entries gets a finite stand-in, then probability 0 everywhere
    log_p = torch.log_softmax(t.masked_fill(~some[..., None], 0.0), -1)
    p = torch.where(some[..., None] & valid, log_p.exp(), torch.zeros_like(log_p))
    log_q = torch.log_softmax(logits / temperature, -1).gather(-1, index.clamp(0, vocab - 1))
    terms = torch.where(p == 0, torch.zeros_like(p), p * (log_p - _loud(log_q, (p != 0) & (index >= vocab))))
    rows = torch.where(some, temperature ** 2 * terms.sum(-1), torch.zeros_like(terms[..., 0]))
    return _reduce(rows, some, reduction)


# ------------------------------------------------------------------- the kernels

def _rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, D) with unit column stride, a row stride >= D and a 16-byte aligned base: a view
    of t where its layout allows, else a copy."""
    d = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, d)
    if t.stride() != (d, 1):                    # not plainly contiguous
        if t.shape[0] == 1 or d == 1 or t.stride(1) != 1 or t.stride(0) < d:
            t = t.contiguous()
            if t.stride() != (d, 1):            # sizes of one: strides are free, the kernels' are not
                t = t.as_strided(t.shape, (d, 1))
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


_INDEX_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _check_head(what, x, weight, index, other=None):
    device, dtype = x.device, x.dtype
    if not x.is_cuda or weight.device != device or index.device != device \
            or (other is not None and other.device != device):
        raise RuntimeError(f"{what} runs the CUDA kernels and needs every input on the same CUDA "
                           "device; saw " + ", ".join(str(t.device) for t in (x, weight, index, other)
                                                      if t is not None))
    if dtype not in (torch.float32, torch.bfloat16) or weight.dtype != dtype:
        raise RuntimeError(f"{what} takes float32 or bfloat16, x and weight alike; got {dtype}, "
                           f"{weight.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError(f"bad shapes: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    d = x.shape[-1]
    if x.numel() > MAX_ROWS * d or weight.shape[0] > MAX_VOCAB or d > MAX_DIM:
        raise ValueError(f"{what} takes up to {MAX_ROWS} rows, {MAX_VOCAB} entries of the vocabulary "
                         f"and {MAX_DIM} columns; got x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if index.dtype not in _INDEX_TYPES:
        raise RuntimeError(f"{what} takes integer indices; got {index.dtype}")


def _check_reduction(reduction):
    if reduction not in _native.REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r}; want 'mean', 'sum' or 'none'")


def _flat(t, *shape):
    """t.reshape(shape), without a view where the shape is that already."""
    return t if t.dim() == len(shape) else t.reshape(shape)


def _as(t, dtype):
    """t contiguous and of this type; t itself where it is that already."""
    t = t if t.dtype == dtype else t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _no_rows(x, weight, shape, reduction):
    """The loss of no rows (0 / 0 for a mean), part of x's and weight's graph."""
    nothing = weight[:0].float().sum()
    if reduction == "none":
        return x.float().sum(-1).reshape(shape) + nothing
    s = x.float().sum() + nothing
    return s / 0.0 if reduction == "mean" else s


class LinearCrossEntropyCUDA(torch.autograd.Function):
    """linear_cross_entropy on x (M, D), weight (V, D), target (M), forward and backward."""

    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        with _native.on_device(x.device):
            loss, kept = _native.linear_ce_fwd(x, weight, target, ignore_index, reduction)
        ctx.save_for_backward(x, weight, target, kept)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, weight, target, kept = ctx.saved_tensors
        with _native.on_device(x.device):
            dx, dw = _native.linear_ce_bwd(x, weight, target, ctx.ignore_index, ctx.reduction,
                                           _as(dloss, torch.float32), kept,
                                           *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None


class LinearDistillationCUDA(torch.autograd.Function):
    """linear_distillation on x (M, D), weight (V, D), index and logits (M, k)."""

    @staticmethod
    def forward(ctx, x, weight, index, logits, temperature, reduction):
        with _native.on_device(x.device):
            loss, kept = _native.linear_kd_fwd(x, weight, index, logits, temperature, reduction)
        ctx.save_for_backward(x, weight, index, kept)
        ctx.temperature, ctx.reduction = temperature, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, weight, index, kept = ctx.saved_tensors
        with _native.on_device(x.device):
            dx, dw = _native.linear_kd_bwd(x, weight, index, ctx.temperature, ctx.reduction,
                                           _as(dloss, torch.float32), kept,
                                           *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None, None


def _dispatch(impl: str, x) -> bool:
    """Whether the kernels run."""
    if impl not in _IMPLS:
        raise ValueError(f"unknown scan_impl {impl!r}; want 'auto', 'cuda', 'metal' or 'torch'")
    if impl in ("cuda", "metal") and not x.is_cuda:
        raise RuntimeError(f"scan_impl={impl!r} needs CUDA tensors; got device {x.device.type!r}")
    return impl != "torch" and x.is_cuda


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100, reduction: str = "mean", impl: str = "auto"):
    """Softmax cross entropy of the logits x W^T, without keeping them.

    x (..., D), weight (V, D), target (...) integers. Rows whose target is
    ignore_index have loss and gradient 0, whatever x holds there, and do not
    count in the mean (which is NaN if no row counts, with gradients 0). A target outside
    [0, V) that is not ignore_index gives a NaN loss and NaN gradients.
    reduction 'mean', 'sum' or 'none' (target's shape); the loss is float32.
    Differentiable once, with respect to x and weight.
    """
    _check_reduction(reduction)
    if not _dispatch(impl, x):
        return linear_cross_entropy_ref(x, weight, target, ignore_index, reduction)
    _check_head("linear_cross_entropy", x, weight, target)
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target {tuple(target.shape)} does not match x {tuple(x.shape)}")
    if target.numel() == 0:
        return _no_rows(x, weight, target.shape, reduction)
    x2, w2 = _rows(x), _rows(weight)
    t = _as(_flat(target, -1), torch.int64)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        loss = LinearCrossEntropyCUDA.apply(x2, w2, t, int(ignore_index), reduction)
    else:
        with _native.on_device(x.device):
            loss, _ = _native.linear_ce_fwd(x2, w2, t, int(ignore_index), reduction, keep=False)
    return _flat(loss, *target.shape) if reduction == "none" else loss


def linear_distillation(x: torch.Tensor, weight: torch.Tensor, teacher_index: torch.Tensor,
                        teacher_logits: torch.Tensor, temperature: float = 1.0,
                        reduction: str = "mean", impl: str = "auto"):
    """KL divergence from a teacher's top k logits to softmax(x W^T / temperature).

        p = softmax(teacher_logits / temperature) over the entries with index >= 0
        loss = temperature^2 sum_j p_j (log p_j - log q[teacher_index_j])

    with q over the whole vocabulary, without keeping the student's logits.
    teacher_index (..., k) integers, teacher_logits (..., k) floats (used as
    float32; not differentiated), k <= 1024. Entries with a negative index
    are empty, whatever their logit; rows without an entry (or with only
    logits of -inf) have loss and gradient 0 and do not count in the mean. An
    index may occur twice; one >= V gives a NaN loss and NaN gradients.
    Differentiable once, with respect to x and weight.
    """
    _check_reduction(reduction)
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite; got {temperature}")
    if teacher_index.dim() < 1 or teacher_logits.shape != teacher_index.shape \
            or teacher_index.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"bad shapes: x {tuple(x.shape)}, teacher_index {tuple(teacher_index.shape)}, "
                         f"teacher_logits {tuple(teacher_logits.shape)}")
    k = teacher_index.shape[-1]
    if not 1 <= k <= MAX_K:
        raise ValueError(f"linear_distillation takes 1 to {MAX_K} entries a row; got {k}")
    if not _dispatch(impl, x):
        return linear_distillation_ref(x, weight, teacher_index, teacher_logits.detach(),
                                       temperature, reduction)
    _check_head("linear_distillation", x, weight, teacher_index, teacher_logits)
    if not teacher_logits.is_floating_point():
        raise RuntimeError(f"teacher_logits must be floating point; got {teacher_logits.dtype}")
    lead = x.shape[:-1]
    if teacher_index.numel() == 0:
        return _no_rows(x, weight, lead, reduction)
    x2, w2 = _rows(x), _rows(weight)
    index = _as(_flat(teacher_index, -1, k), torch.int64)
    logits = _as(_flat(teacher_logits.detach(), -1, k), torch.float32)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        loss = LinearDistillationCUDA.apply(x2, w2, index, logits, temperature, reduction)
    else:
        with _native.on_device(x.device):
            loss, _ = _native.linear_kd_fwd(x2, w2, index, logits, temperature, reduction, keep=False)
    return _flat(loss, *lead) if reduction == "none" else loss
