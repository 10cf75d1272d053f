"""TinyMamba: the small Mamba language model around the selective scan.

API-compatible with the reference package's `mamba_metal.model`
(Anamaya1729/mamba-metal-scan, mamba_metal/model.py): the same config fields,
module names and parameter shapes (so state_dicts load either way), the same
block arithmetic, and the same `scan_impl` switch. Only the scan itself is
native by default; everything else is ordinary PyTorch. `fuse_norm` runs the
residual sum after each block and the next norm as one kernel each way
(`residual_rms_norm`), `fuse_loss` the head and its cross entropy without the
logits (`linear_cross_entropy`); `TinyMamba.distill_loss` trains on a
teacher's top k logits through the same head (`linear_distillation`).
`fuse_conv` runs the convolution and its SiLU as one kernel each way
(`causal_conv`). `TinyMamba.serve` takes prompts of unequal lengths and single
tokens packed behind one another, with the blocks' states in a cache of places
(`causal_conv_packed`, `selective_scan_packed`), and `TinyMamba.generate` draws from
its logits (`sample_tokens`).

Block (reference model.py:161-256):
    x -> RMSNorm -> in_proj -> (x, z)
    x -> causal depthwise conv -> SiLU
    dt = dt_min + (dt_max - dt_min) * sigmoid(dt_proj(x)),  B = B_proj(x),
    C = C_proj(x),  Aneg = softplus(A)
    y = selective_scan(x, dt, Aneg, B, C) + D_skip
    out = residual + out_proj(y * SiLU(z))

`scan_impl` 'auto' runs the CUDA kernels on CUDA tensors and the associative
`parallel_scan` elsewhere; 'cuda'/'metal' force the kernels; 'torch' forces
the PyTorch recurrence. d_inner defaults to the largest multiple of 8 whose
block costs no more parameters than a transformer block of the same
d_model/d_ff (reference model.py:58-82).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from mamba_metal.conv import causal_conv, causal_conv_packed
from mamba_metal.head import linear_cross_entropy, linear_distillation
from mamba_metal.norm import residual_rms_norm
from mamba_metal.packed import selective_scan_packed
from mamba_metal.sampling import sample_tokens
from mamba_metal.scan import (SSM_CHUNK, gated_output, selective_scan, selective_scan_proj,
                              selective_scan_step, selective_scan_step_ref)


@dataclass
class MambaConfig:
    vocab_size: int
    d_model: int = 384
    n_layers: int = 10
    d_ff: int = 1536          # sizes d_inner through the transformer parameter budget
    max_seq_len: int = 512
    d_state: int = 16
    d_conv: int = 4
    d_inner: Optional[int] = None
    scan_chunk: int = 0       # time slice of the parallel_scan fallback; 0 = one pass
    ssm_chunk: int = SSM_CHUNK  # checkpoint stride of the CUDA scan (memory vs recompute)
    scan_impl: str = "auto"   # 'auto' | 'cuda' | 'metal' | 'torch'
    fuse_proj: bool = True    # CUDA scan computes dt and softplus(A) itself (selective_scan_proj)
    fuse_gate: bool = True    # (y + D_skip) * silu(z) as one CUDA kernel each way (gated_output)
    dt_min: float = 0.001
    dt_max: float = 0.1
    norm_eps: float = 1e-6
    # The three below call the operators with the modules' parameters, not the modules: with fuse_norm
    # the blocks', their norms' and ln_f's forward (the first norm's aside), with fuse_loss and in
    # distill_loss the head's, with fuse_conv and in serve the blocks' conv's does not run, nor do hooks and
    # wrappers on them (sharding or checkpointing by module); in serve the blocks' own does not either.
    fuse_norm: bool = False   # residual sum + next norm as one CUDA kernel each way (residual_rms_norm)
    fuse_loss: bool = False   # with targets: no logits, forward returns (None, loss) (linear_cross_entropy)
    fuse_conv: bool = False   # convolution + SiLU as one CUDA kernel each way, up to 8 taps (causal_conv)


def transformer_block_params(d_model: int, d_ff: int) -> int:
    """Parameters of a pre-norm transformer block: attention (4 d^2), MLP, two norms."""
    attention = 4 * d_model * d_model
    mlp = 2 * d_model * d_ff
    norms = 2 * d_model
    return attention + mlp + norms


def mamba_block_params(d_model: int, d_inner: int, d_state: int, d_conv: int) -> int:
    """Parameters of one MambaBlock as built below."""
    in_proj = 2 * d_model * d_inner
    conv = d_inner * d_conv + d_inner
    dt_proj = d_inner * d_inner + d_inner
    ssm = 3 * d_inner * d_state            # A, B_proj, C_proj
    skip = d_inner
    out_proj = d_inner * d_model
    norm = d_model
    return in_proj + conv + dt_proj + ssm + skip + out_proj + norm


def d_inner_for_budget(target: int, d_model: int, d_state: int, d_conv: int) -> int:
    """Largest multiple of 8 (at least 8) whose MambaBlock fits in `target` parameters.

    mamba_block_params is d_inner^2 + c*d_inner + d_model with
    c = 3*d_model + d_conv + 3 + 3*d_state; take the positive root and round down.
    """
    c = 3 * d_model + d_conv + 3 + 3 * d_state
    disc = c * c + 4 * (target - d_model)
    root = (math.sqrt(disc) - c) / 2.0
    return max(8, 8 * int(root // 8))


class RMSNorm(nn.Module):
    def __init__(self, d: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d))
        self.eps = eps

    def forward(self, x):
        dtype = x.dtype
        xf = x.float()
        xf = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)
        return (self.weight * xf).to(dtype)


# ------------------------------------------------------------------ the scans

def scan_recurrence(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """h_t = a_t * h_{t-1} + b_t over dim 1, one step at a time (h_{-1} = 0)."""
    h = torch.zeros_like(b[:, 0])
    hs = []
    for t in range(a.shape[1]):
        h = a[:, t] * h + b[:, t]
        hs.append(h)
    return torch.stack(hs, dim=1)


def _doubling_scan(a: torch.Tensor, b: torch.Tensor):
    """Inclusive scan of the affine maps h -> a*h + b over dim 1 in log2(T) rounds.

    Returns (A, H): A[t] = a_0*...*a_t and H[t] = the state after step t from
    a zero start. Round r combines every element with the one 2^r earlier;
    positions before the start see the identity map (a=1, b=0).
    """
    A, H = a, b
    T = a.shape[1]
    shift = 1
    while shift < T:
        A_prev = F.pad(A[:, :-shift], (0, 0) * (a.dim() - 2) + (shift, 0), value=1.0)
        H_prev = F.pad(H[:, :-shift], (0, 0) * (a.dim() - 2) + (shift, 0), value=0.0)
        H = A * H_prev + H
        A = A * A_prev
        shift *= 2
    return A, H


def parallel_scan(a: torch.Tensor, b: torch.Tensor, chunk: int = 0) -> torch.Tensor:
    """Same result as scan_recurrence, computed with a log-depth associative scan.

    chunk > 0 scans `chunk` steps at a time and folds in the state carried
    from the previous slice (h += A * carry), which bounds the memory of the
    intermediates without changing the result (reference model.py:139-156).
    """
    T = a.shape[1]
    if not chunk or T <= chunk:
        return _doubling_scan(a, b)[1]
    out, carry = [], None
    for s in range(0, T, chunk):
        A, H = _doubling_scan(a[:, s:s + chunk], b[:, s:s + chunk])
        if carry is not None:
            H = H + A * carry.unsqueeze(1)
        carry = H[:, -1]
        out.append(H)
    return torch.cat(out, dim=1)


# ------------------------------------------------------------------- the block

class MambaBlock(nn.Module):
    """Gated causal conv + diagonal selective SSM inside one residual."""

    def __init__(self, cfg: MambaConfig, d_inner: int):
        super().__init__()
        dm, ds, kc = cfg.d_model, cfg.d_state, cfg.d_conv
        self.d_inner = d_inner
        self.scan_chunk = cfg.scan_chunk
        self.ssm_chunk = cfg.ssm_chunk
        self.scan_impl = cfg.scan_impl
        self.fuse_proj = cfg.fuse_proj
        self.fuse_gate = cfg.fuse_gate
        self.fuse_conv = cfg.fuse_conv
        self.dt_min, self.dt_max = cfg.dt_min, cfg.dt_max
        self.norm = RMSNorm(dm, cfg.norm_eps)
        self.in_proj = nn.Linear(dm, 2 * d_inner, bias=False)
        # padding kc-1 on both sides; keeping the first T outputs makes it causal
        self.conv = nn.Conv1d(d_inner, d_inner, kernel_size=kc, padding=kc - 1,
                              groups=d_inner, bias=True)
        self.dt_proj = nn.Linear(d_inner, d_inner, bias=True)
        self.A = nn.Parameter(torch.arange(1, ds + 1, dtype=torch.float32).repeat(d_inner, 1))
        self.B_proj = nn.Linear(d_inner, ds, bias=False)
        self.C_proj = nn.Linear(d_inner, ds, bias=False)
        self.D_skip = nn.Parameter(torch.ones(d_inner))
        self.out_proj = nn.Linear(d_inner, dm, bias=False)

    def _proj(self, x):
        """(dt, B, C, Aneg) from the post-conv, post-SiLU activations."""
        dt = self.dt_min + (self.dt_max - self.dt_min) * torch.sigmoid(self.dt_proj(x))
        return dt, self.B_proj(x), self.C_proj(x), F.softplus(self.A)

    def _ssm(self, x):
        """(a, b, C) of the recurrence h_t = a_t*h_{t-1} + b_t, materialised."""
        dt, B_t, C_t, Aneg = self._proj(x)
        a = torch.exp(-dt.unsqueeze(-1) * Aneg)
        b = dt.unsqueeze(-1) * B_t.unsqueeze(2) * x.unsqueeze(-1)
        return a, b, C_t

    def _scan(self, x, return_state=False):
        """y_t = sum_n C_tn h_tn; the fused scan when scan_impl allows it."""
        if self.fuse_proj and x.is_cuda and self.scan_impl != "torch":
            # dt and Aneg computed inside the kernels from dt_proj(x) and A
            return selective_scan_proj(x, self.dt_proj(x), self.A, self.B_proj(x), self.C_proj(x),
                                       self.dt_min, self.dt_max, impl=self.scan_impl,
                                       chunk=self.ssm_chunk, return_state=return_state)
        dt, B_t, C_t, Aneg = self._proj(x)
        r = selective_scan(x, dt, Aneg, B_t, C_t, impl=self.scan_impl, chunk=self.ssm_chunk,
                           return_state=return_state)
        if r is not None:
            return r
        a = torch.exp(-dt.unsqueeze(-1) * Aneg)
        b = dt.unsqueeze(-1) * B_t.unsqueeze(2) * x.unsqueeze(-1)
        h = parallel_scan(a, b, chunk=self.scan_chunk)
        y = (h * C_t.unsqueeze(2)).sum(-1)
        return (y, h[:, -1]) if return_state else y

    def _step(self, x, dt, Aneg, B_t, C_t, cache):
        """One token of the recurrence on cache["h"]; y (B, d_inner).

        Without autograd, on CUDA, the fused decode kernel updates the cached
        state in place (it owns that buffer: the scan's returned state is a
        detached checkpoint). With autograd, or off-CUDA, the step is the
        reference's differentiable PyTorch ops and the cache gets a new tensor.
        """
        h = cache["h"]
        needs_grad = torch.is_grad_enabled() and any(
            t.requires_grad for t in (x, dt, Aneg, B_t, C_t, h))
        if x.is_cuda and self.scan_impl != "torch" and not needs_grad:
            if not cache.get("h_owned"):
                h = h.clone(memory_format=torch.contiguous_format)
                cache["h"], cache["h_owned"] = h, True
            return selective_scan_step(x, dt, Aneg, B_t, C_t, h, impl=self.scan_impl)
        y, cache["h"] = selective_scan_step_ref(x, dt, Aneg, B_t, C_t, h)
        cache["h_owned"] = False
        return y

    def forward(self, x, cache=None):
        return x + self.mix(self.norm(x), cache)

    def mix(self, x, cache=None):
        """The block between its norm and the residual sum."""
        x, z = self.in_proj(x).chunk(2, dim=-1)
        kc = self.conv.kernel_size[0]
        fuse_conv = self.fuse_conv and x.is_cuda and self.scan_impl != "torch"
        if cache is not None and cache.get("h") is not None and x.shape[1] == 1:
            # one-token recurrent step against the cached conv window and state
            if fuse_conv and not (torch.is_grad_enabled()
                                  and any(t.requires_grad for t in (x, *self.conv.parameters(), cache["conv"]))):
                if not cache.get("conv_owned"):
                    cache["conv"] = cache["conv"][:, :, :kc - 1].clone(memory_format=torch.contiguous_format)
                    cache["conv_owned"] = True
                x = causal_conv_packed(x[:, 0], self.conv.weight, self.conv.bias, cache["conv"],
                                       impl=self.scan_impl).unsqueeze(1)
            else:
                window = torch.cat([cache["conv"], x.transpose(1, 2)], dim=2)   # (B, d_inner, kc)
                x = F.silu(self.conv(window)[:, :, kc - 1:kc]).transpose(1, 2)
                cache["conv"], cache["conv_owned"] = window[:, :, 1:], False
            dt, B_t, C_t, Aneg = self._proj(x)
            y = self._step(x[:, 0], dt[:, 0], Aneg, B_t[:, 0], C_t[:, 0], cache).unsqueeze(1)
        else:
            xc = x.transpose(1, 2)
            if fuse_conv:
                x = causal_conv(x, self.conv.weight, self.conv.bias, impl=self.scan_impl)
            else:
                x = F.silu(self.conv(xc)[:, :, :xc.shape[2]]).transpose(1, 2)
            if cache is not None:
                tail = xc[:, :, -(kc - 1):]
                if tail.shape[2] < kc - 1:
                    tail = F.pad(tail, (kc - 1 - tail.shape[2], 0))
                cache["conv"], cache["conv_owned"] = tail, False
            # the last checkpoint of the scan is h[:, -1]: the cache costs nothing
            y, h_last = self._scan(x, return_state=True)
            if cache is not None:
                cache["h"], cache["h_owned"] = h_last, False
        if self.fuse_gate and y.is_cuda and self.scan_impl != "torch":
            return self.out_proj(gated_output(y, z, self.D_skip, impl=self.scan_impl))
        y = y + self.D_skip
        return self.out_proj(y * F.silu(z))


    def serve(self, x, cache, starts=None, slots=None, out_slots=None):
        """mix on packed rows x (L, d_model) that go on from the states in cache, without gradients."""
        x, z = self.in_proj(x).chunk(2, dim=-1)
        lists = dict(starts=starts, slots=slots, out_slots=out_slots, impl=self.scan_impl)
        x = causal_conv_packed(x, self.conv.weight, self.conv.bias, cache["conv"], **lists)
        y = selective_scan_packed(x, self.dt_proj(x), self.A, self.B_proj(x), self.C_proj(x), cache["h"], z=z,
                                  d_skip=self.D_skip, dt_range=(self.dt_min, self.dt_max), **lists)
        return self.out_proj(y)


class TinyMamba(nn.Module):
    """A Mamba language model sized to a transformer's parameter budget."""

    def __init__(self, cfg: MambaConfig):
        super().__init__()
        self.cfg = cfg
        d_inner = cfg.d_inner
        if d_inner is None:
            d_inner = d_inner_for_budget(transformer_block_params(cfg.d_model, cfg.d_ff),
                                         cfg.d_model, cfg.d_state, cfg.d_conv)
        self.d_inner = d_inner
        self.tok = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.blocks = nn.ModuleList(MambaBlock(cfg, d_inner) for _ in range(cfg.n_layers))
        self.ln_f = RMSNorm(cfg.d_model, cfg.norm_eps)
        self.head = nn.Linear(cfg.d_model, cfg.vocab_size, bias=False)
        self.head.weight = self.tok.weight          # tied
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)

    def hidden(self, idx, cache=None):
        """The head's input: the last block's residual stream after ln_f, (B, T, d_model)."""
        if cache is not None and "blocks" not in cache:
            cache["blocks"] = [{} for _ in self.blocks]
        per_block = cache["blocks"] if cache is not None else [None] * len(self.blocks)
        x = self.tok(idx)
        if self.cfg.fuse_norm and len(self.blocks):
            norms = [b.norm for b in self.blocks] + [self.ln_f]
            u = norms[0](x)
            for block, bc, norm in zip(self.blocks, per_block, norms[1:]):
                x, u = residual_rms_norm(x, block.mix(u, bc), norm.weight, eps=norm.eps,
                                         impl=self.cfg.scan_impl)
            return u
        for block, bc in zip(self.blocks, per_block):
            x = block(x, bc)
        return self.ln_f(x)

    def forward(self, idx, targets=None, cache=None):
        x = self.hidden(idx, cache)
        if targets is not None and self.cfg.fuse_loss:
            return None, linear_cross_entropy(x, self.head.weight, targets, ignore_index=-100,
                                              impl=self.cfg.scan_impl)
        logits = self.head(x)
        loss = None
        if targets is not None:
            loss = F.cross_entropy(logits.reshape(-1, logits.size(-1)), targets.reshape(-1),
                                   ignore_index=-100)
        return logits, loss

    def distill_loss(self, idx, teacher_index, teacher_logits, temperature: float = 1.0,
                     reduction: str = "mean"):
        """KL divergence of the model's next-token distribution from a teacher's top k logits.

        teacher_index, teacher_logits (B, T, k): see `linear_distillation`.
        """
        return linear_distillation(self.hidden(idx), self.head.weight, teacher_index, teacher_logits,
                                   temperature, reduction, impl=self.cfg.scan_impl)

    # ------------------------------------------------------------------- serving

    def new_cache(self, places: int):
        """States of `places` answers for `serve`, all zeros: what a sequence starts from."""
        w = self.head.weight
        kc, ds = self.cfg.d_conv, self.cfg.d_state
        return {"blocks": [{"conv": w.new_zeros(places, self.d_inner, kc - 1),
                            "h": w.new_zeros(places, self.d_inner, ds, dtype=torch.float32)} for _ in self.blocks]}

    @torch.no_grad()
    def serve(self, idx, cache, starts=None, slots=None, out_slots=None):
        """Logits (S, vocab) behind the last token of each of S packed sequences.

        idx (L,): the tokens of prompts, pieces of prompts and single tokens behind one
        another, each sequence of at least one; cache from `new_cache`, updated in place; starts,
        slots, out_slots as in `mamba_metal.packed` (without starts: one token a sequence). A
        sequence whose slot is outside the cache starts anew. An empty one's logits are some
        other row's.
        """
        if starts is not None and starts.dim() == 1 and starts.shape[0] > 1 and idx.shape[0] == 0:
            raise ValueError(f"serve needs a token of each of {starts.shape[0] - 1} sequences; idx is empty")
        x = self.tok(idx)
        norms = [b.norm for b in self.blocks] + [self.ln_f]
        u = norms[0](x)
        for block, bc, norm in zip(self.blocks, cache["blocks"], norms[1:]):
            y = block.serve(u, bc, starts, slots, out_slots)
            if self.cfg.fuse_norm:
                x, u = residual_rms_norm(x, y, norm.weight, eps=norm.eps, impl=self.cfg.scan_impl)
            else:
                x = x + y
                u = norm(x)
        if starts is not None:
            # (a gather outside the rows would be a device assertion, which ends the process's CUDA calls)
            u = u[(starts[1:].long() - 1).clamp(0, max(0, u.shape[0] - 1))]
        return self.head(u)

    @torch.no_grad()
    def generate(self, prompts, max_new_tokens: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 uniform=None, generator=None):
        """max_new_tokens tokens for each prompt, (S, max_new_tokens), drawn by `sample_tokens`.

        prompts: S 1-D integer tensors of at least one token (of any lengths), or a 2-D tensor.
        temperature, top_k, top_p, min_p: one number, or a tensor (S,). uniform
        (max_new_tokens, S): the random numbers; None: torch.rand, with `generator`.
        """
        prompts = list(prompts)
        device = self.head.weight.device
        lens = [len(p) for p in prompts]
        if not prompts or min(lens) < 1:
            raise ValueError(f"generate needs prompts of at least one token; got lengths {lens}")
        if uniform is None:
            uniform = torch.rand(max_new_tokens, len(prompts), generator=generator, device=device, dtype=torch.float32)
        if uniform.shape != (max_new_tokens, len(prompts)):
            raise ValueError(f"uniform must be ({max_new_tokens}, {len(prompts)}); got {tuple(uniform.shape)}")
        starts = torch.tensor([0, *lens]).cumsum(0).to(device=device, dtype=torch.int32)
        cache = self.new_cache(len(prompts))
        out = torch.empty(len(prompts), max_new_tokens, dtype=torch.int64, device=device)
        idx = torch.cat([p.to(device) for p in prompts])
        for i in range(max_new_tokens):
            logits = self.serve(idx, cache, starts if i == 0 else None)
            out[:, i] = sample_tokens(logits, uniform[i], temperature, top_k, top_p, min_p, impl=self.cfg.scan_impl)
            idx = out[:, i].clamp(min=0)             # (-1, where no logit is a number, has no embedding)
        return out

    def count_params(self) -> int:
        """Unique parameters (the tied head counts once)."""
        return sum(p.numel() for p in self.parameters())
