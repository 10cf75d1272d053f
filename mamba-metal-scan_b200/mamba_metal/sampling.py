"""Drawing tokens from logits on NVIDIA B200 (sm_100a).

    token = sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)

The random numbers are the caller's, one a row, so a draw can be repeated and tested. The
model's head gives the logits (`TinyMamba.generate` uses it); the reference stops at them
(mamba_metal/model.py:282-297). Kernel in csrc/mms_sample.cu, dispatch as in
`mamba_metal.scan`.
"""
from __future__ import annotations

import operator

import torch

from mamba_metal import _native
from mamba_metal.packed import _FLOATS, dispatch


def _setting(name, value, lead, device, dtype):
    """(tensor or None, number): a setting of each row's own, or one for all."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.shape != lead:
        raise ValueError(f"{name} must be a number or {tuple(lead)}; got {tuple(value.shape)}")
    if value.device != device:
        raise RuntimeError(f"{name} must be on {device}; got {value.device}")
    if dtype is None:                        # whole numbers
        if value.is_floating_point() or value.is_complex() or value.dtype == torch.bool:
            raise RuntimeError(f"{name} must hold integers; got {value.dtype}")
        if value.dtype != torch.int32 and value.dtype != torch.int64:
            value = value.to(torch.int64)
    elif value.dtype != dtype:
        value = value.to(dtype)
    return value if value.is_contiguous() else value.contiguous(), 0


def sample_tokens_ref(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of sample_tokens in PyTorch ops, in float64 (any device and float type)."""
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    logits = logits.reshape(-1, vocab)
    rows, device = logits.shape[0], logits.device

    def column(v, dtype):
        if isinstance(v, torch.Tensor):
            return v.reshape(-1, 1).to(dtype)
        return torch.full((rows, 1), v, dtype=dtype, device=device)

    t, k = column(temperature, torch.float32).double(), column(top_k, torch.int64)
    p, m = column(top_p, torch.float32).double(), column(min_p, torch.float32).double().clamp(max=1.0)
    u = column(uniform, torch.float32).double()
    u = torch.where(u > 0, u, torch.zeros_like(u)).clamp(max=1.0 - 2.0 ** -24)
    z, index = torch.sort(logits, dim=1, descending=True, stable=True)
    z = z.double()
    top = z[:, :1]
    bad = logits.isnan().any(1) | ~(top[:, 0] > -float("inf")) | t[:, 0].isnan() | p[:, 0].isnan() | m[:, 0].isnan()
    greedy = (t <= 0) | (k == 1) | (p <= 0)
    w = torch.where(top.isinf(), (z == top).double(), torch.exp((z - top) / torch.where(greedy, 1.0, t)))
    w = torch.where(z == -float("inf"), 0.0, w)              # (at an infinite temperature too)
    place = torch.arange(vocab, device=device)
    w = torch.where((place < torch.where(k > 0, k, vocab)) & ~(greedy & (place > 0)), w, 0.0)
    ahead = torch.cumsum(w, 1) - w
    w = torch.where((p >= 1) | (place == 0) | (ahead < p * w.sum(1, keepdim=True)), w, 0.0)
    w = torch.where(w >= m, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)
    upto = torch.cumsum(w, 1)
    hit = (upto > u * upto[:, -1:]) & (w > 0)
    last = vocab - 1 - (w > 0).int().flip(1).argmax(1)
    token = torch.where(hit.any(1), hit.int().argmax(1), last)
    logprob = torch.log(w.gather(1, token[:, None])[:, 0] / upto[:, -1])
    token = torch.where(bad, -1, token)
    logprob = torch.where(bad, float("nan"), logprob).float()
    return token.reshape(lead), logprob.reshape(lead)


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, return_logprob: bool = False, impl: str = "auto"):
    """A token index (int64, -1 for none) from each row of logits (..., V); see the steps below.

        w_i = exp((z_i - max z) / temperature)
        keep the top_k largest logits (0: all), equal ones by lowest index;
        of those the shortest run, largest first, whose weight is at least top_p of theirs;
        of those the ones with w_i >= min_p;
        the first index whose kept weights up to it pass uniform * the kept weights' sum.

    uniform (...,) in [0, 1); temperature, top_k, top_p, min_p: one number, or a tensor (...,)
    with one a row. temperature 0 takes the largest logit. logits of -inf are never drawn; a
    row without any above it, or with a NaN among its logits or settings, gives -1. With
    return_logprob also the log of the token's share of the kept weights (float32, NaN beside -1).
    logits float32 or bfloat16 on the CUDA kernel, rows may be strided. Weights are float64, in the
    kernel rounded to whole numbers of 2^-44 of the largest (2^-(62 - log2 V) above 2^18 entries)
    and summed exactly.
    Not differentiable.
    """
    if logits.dim() < 1 or logits.shape[-1] < 1 or uniform.shape != logits.shape[:-1]:
        raise ValueError(f"bad shapes: logits {tuple(logits.shape)}, uniform {tuple(uniform.shape)}")
    if not logits.is_floating_point() or not uniform.is_floating_point():
        raise RuntimeError(f"logits and uniform must be floating point; got {logits.dtype}, {uniform.dtype}")
    for name, v, low in (("temperature", temperature, 0.0), ("top_k", top_k, 0), ("top_p", top_p, 0.0),
                         ("min_p", min_p, 0.0)):
        if not isinstance(v, torch.Tensor) and not v >= low:
            raise ValueError(f"{name} must not be negative; got {v}")
    if not isinstance(top_k, torch.Tensor):
        top_k = min(operator.index(top_k), logits.shape[-1])
    lead, vocab, device = logits.shape[:-1], logits.shape[-1], logits.device
    if not dispatch(impl, logits):
        for name, v in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            _setting(name, v, lead, device, None if name == "top_k" else torch.float32)
        with torch.no_grad():
            out = sample_tokens_ref(logits, uniform, temperature, top_k, top_p, min_p)
        return out if return_logprob else out[0]
    if logits.dtype not in _FLOATS:
        raise RuntimeError(f"sample_tokens takes float32 or bfloat16 logits; got {logits.dtype}")
    if uniform.device != device:
        raise RuntimeError(f"uniform must be on {device}; got {uniform.device}")
    rows = uniform.numel()
    if vocab > _native.SERVE_MAX or rows > 1 << 24:
        raise ValueError(f"sample_tokens takes up to {1 << 24} rows and {_native.SERVE_MAX} logits a row; "
                         f"got {tuple(logits.shape)}")
    with _native.on_device(device):
        t, t1 = _setting("temperature", temperature, lead, device, torch.float32)
        k, k1 = _setting("top_k", top_k, lead, device, None)
        p, p1 = _setting("top_p", top_p, lead, device, torch.float32)
        m, m1 = _setting("min_p", min_p, lead, device, torch.float32)
        if rows == 0:
            out = torch.empty(lead, dtype=torch.int64, device=device), torch.empty(lead, dtype=torch.float32, device=device)
            return out if return_logprob else out[0]
        z = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
        ld = vocab if rows == 1 else z.stride(0)
        if z.stride(1) != 1 and vocab > 1:
            z, ld = z.contiguous(), vocab
        u = uniform if uniform.dtype == torch.float32 else uniform.float()
        u = u if u.is_contiguous() else u.contiguous()
        token, logprob = _native.sample(z, ld, u, t, t1, k, k1, p, p1, m, m1, return_logprob)
        if len(lead) != 1:
            token = token.view(lead)
            logprob = None if logprob is None else logprob.view(lead)
    return (token, logprob) if return_logprob else token
