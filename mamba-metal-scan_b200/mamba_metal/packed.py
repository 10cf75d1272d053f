"""Packed sequences over a cache of states: prompts of unequal lengths, their pieces, single tokens.

A packed batch holds the rows of several sequences behind one another, without
padding: sequence s has the rows starts[s] to starts[s + 1] - 1. What a sequence goes on
from, the scan's state or the convolution's last inputs, lies in a place of a
cache that the calls read and write in place:

    starts      (S + 1,) ascending integers within [0, rows], or None: one row per
                sequence (the single tokens of S answers). Sequences may be empty; rows
                before the first and behind the last sequence belong to none and give zeros
    slots       (S,) integers, the place of each sequence's state; None: place s. A sequence
                whose place is outside the cache (-1) starts from nothing
    out_slots   (S,) integers, where the state it leaves goes; None: slots. Outside the
                cache: nowhere. Several sequences may go on from one place (answers that
                share a prompt), but a place that one writes is neither read nor written
                by another sequence of the same call

The lists stay on the device and are not looked at by the host: a call is
captured into a CUDA graph once and replayed with other lists of the same size. A list
that breaks these rules gives wrong rows, never an access outside the arrays.

The reference's cache goes on by one token of one batch at a time
(mamba_metal/model.py:203-241).
"""
from __future__ import annotations

import torch

from mamba_metal import _native
from mamba_metal.scan import _IMPLS, _aligned, proj_ref

_FLOATS = (torch.float32, torch.bfloat16)


def dispatch(impl: str, x) -> bool:
    """Whether the kernels run."""
    if impl == "auto":
        return x.is_cuda
    if impl not in _IMPLS:
        raise ValueError(f"unknown scan_impl {impl!r}; want 'auto', 'cuda', 'metal' or 'torch'")
    if impl in ("cuda", "metal") and not x.is_cuda:
        raise RuntimeError(f"scan_impl={impl!r} needs CUDA tensors; got device {x.device.type!r}")
    return impl != "torch" and x.is_cuda


def check_lists(rows: int, places: int, starts, slots, out_slots, x) -> int:
    """The number of sequences, from the lists' shapes; the host does not look inside."""
    if starts is not None:
        if starts.dim() != 1 or starts.shape[0] < 1:
            raise ValueError(f"starts must be (sequences + 1,); got {tuple(starts.shape)}")
        count = starts.shape[0] - 1
    else:
        count = rows
    if slots is None and places < count:
        raise ValueError(f"without slots the cache needs a place for each of {count} sequences; it has {places}")
    for name, t in (("starts", starts), ("slots", slots), ("out_slots", out_slots)):
        if t is None:
            continue
        if name != "starts" and t.shape != (count,):
            raise ValueError(f"{name} must be ({count},), one place a sequence; got {tuple(t.shape)}")
        dtype = t.dtype
        if dtype != torch.int64 and dtype != torch.int32 and (dtype.is_floating_point or dtype.is_complex or dtype == torch.bool):
            raise RuntimeError(f"{name} must hold integers; got {dtype}")
        if t.get_device() != x.get_device():
            raise RuntimeError(f"{name} must be on {x.device}; got {t.device}")
    return count


def same_device(what, x, tensors):
    """RuntimeError unless every tensor (None: no tensor) is on x's device."""
    index = x.get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"{what} needs every tensor on the same CUDA device; saw "
                               + ", ".join(str(t.device) for t in (x, *tensors) if t is not None))


def int_list(t):
    """t as the kernels read it: int32 or int64, contiguous."""
    if t is None:
        return None
    if t.dtype != torch.int32 and t.dtype != torch.int64:
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def rows_of(t, group: int = 1):
    """(tensor, row stride) of a 2-D t with unit column stride: t itself where it has one; with
    `group`, also bases and strides of whole groups of so many elements."""
    ld, step = t.stride()
    rows, d = t.shape
    if rows == 1:
        ld = d
    if (step != 1 and d > 1) or (group > 1 and (ld % group or t.data_ptr() % (group * t.element_size()))):
        t, ld = t.clone(memory_format=torch.contiguous_format), d
    return t, ld


def places_of(rows: int, starts, slots, out_slots, places: int):
    """[(first, end, from, to)] of each sequence, on the host; from and to None for no place. Starts that
    break the rules are brought into the rows as in the kernels."""
    bounds = range(rows + 1) if starts is None else [min(max(v, 0), rows) for v in starts.tolist()]
    count = len(bounds) - 1
    src = list(range(count)) if slots is None else slots.tolist()
    dst = src if out_slots is None else out_slots.tolist()

    def inside(p):
        return p if 0 <= p < places else None

    return [(bounds[s], max(bounds[s], bounds[s + 1]), inside(src[s]), inside(dst[s])) for s in range(count)]


# --------------------------------------------------------------------- the scan

@torch.no_grad()
def selective_scan_packed_ref(x, dt, aneg, b_in, c_in, state, starts=None, slots=None, out_slots=None,
                              z=None, d_skip=None, dt_range=None):
    """selective_scan_packed in PyTorch ops (any device, float type and d_state; reads the lists on the host)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    xf, dtf, bf, cf, af = (t.to(wide) for t in (x, dt, b_in, c_in, aneg))
    if dt_range is not None:
        dtf, af = proj_ref(dtf, af, *dt_range)
    af = af.masked_fill(af == float("inf"), torch.finfo(torch.float32).max)
    y = torch.zeros_like(xf)
    left = []
    for first, end, src, dst in places_of(x.shape[0], starts, slots, out_slots, state.shape[0]):
        h = torch.zeros_like(af) if src is None else state[src].to(wide)
        for t in range(first, end):
            h = torch.exp(-dtf[t, :, None] * af) * h + (dtf[t] * xf[t])[:, None] * bf[t]
            y[t] = h @ cf[t]
        if end > first:
            if d_skip is not None:
                y[first:end] += d_skip.to(wide)
            if z is not None:
                y[first:end] *= torch.nn.functional.silu(z[first:end].to(wide))
        if dst is not None:
            left.append((dst, h))
    for dst, h in left:
        state[dst] = h.to(state.dtype)
    return y.to(x.dtype)


def selective_scan_packed(x: torch.Tensor, dt: torch.Tensor, aneg: torch.Tensor, b_in: torch.Tensor,
                          c_in: torch.Tensor, state: torch.Tensor, starts: torch.Tensor = None,
                          slots: torch.Tensor = None, out_slots: torch.Tensor = None,
                          z: torch.Tensor = None, d_skip: torch.Tensor = None, dt_range=None,
                          impl: str = "auto"):
    """The scan over packed sequences that go on from `state`; updates it in place, returns y (L, D).

        h_t = exp(-dt_t*Aneg) h_{t-1} + dt_t*B_t*x_t,   y_t = (sum_n C_tn h_tn + d_skip) * silu(z_t)

    x, dt, z (L, D) float32 or bfloat16 alike, B, C (L, N) in the same type or float32,
    Aneg (D, N) and d_skip (D,) (used as float32), state (places, D, N) float32, contiguous;
    the lists as in the module docstring. z and d_skip are optional (the block's gate, see
    `gated_output`). dt_range = (dt_min, dt_max): dt holds logits and aneg the raw A, as in
    `selective_scan_proj`. Rows may be strided views. N is a multiple of 4 up to 64. Any Aneg
    above 2.3e38, an infinite one too, counts as that: a step of 0 decays nothing. An x, B
    or state that is not finite makes the states that it enters, and their outputs from there on, not finite,
    but whether infinite or NaN depends on where the sequence's rows lie.
    Arithmetic and state are float32. Not differentiable: it is the inference path
    (`selective_scan` trains). On CUDA tensors 'auto', 'cuda', 'metal' run the kernels
    (csrc/mms_packed.cuh); elsewhere, or with 'torch', PyTorch ops.
    """
    shape = x.shape
    if len(shape) != 2 or dt.shape != shape or aneg.dim() != 2 or aneg.shape[0] != shape[1]:
        raise ValueError(f"bad shapes: x {tuple(shape)}, dt {tuple(dt.shape)}, Aneg {tuple(aneg.shape)}")
    rows, d = shape
    n = aneg.shape[1]
    if b_in.shape != (rows, n) or c_in.shape != (rows, n):
        raise ValueError(f"B {tuple(b_in.shape)} / C {tuple(c_in.shape)} must be ({rows}, {n})")
    if state.dim() != 3 or state.shape[1:] != (d, n):
        raise ValueError(f"state must be (places, {d}, {n}); got {tuple(state.shape)}")
    if (z is not None and z.shape != shape) or (d_skip is not None and d_skip.shape != (d,)):
        raise ValueError(f"z must be {tuple(shape)} and d_skip ({d},)")
    if dt_range is not None and not float(dt_range[1]) > float(dt_range[0]):
        raise ValueError(f"need dt_min < dt_max; got {dt_range}")
    places = state.shape[0]
    count = check_lists(rows, places, starts, slots, out_slots, x)
    if not dispatch(impl, x):
        return selective_scan_packed_ref(x, dt, aneg, b_in, c_in, state, starts, slots, out_slots, z, d_skip, dt_range)
    same_device("selective_scan_packed", x, (dt, aneg, b_in, c_in, state, z, d_skip))
    dtype, f32 = x.dtype, torch.float32
    if dtype not in _FLOATS or dt.dtype != dtype or (z is not None and z.dtype != dtype):
        raise RuntimeError(f"selective_scan_packed takes float32 or bfloat16 x, dt and z alike; got {dtype}, {dt.dtype}"
                           + ("" if z is None else f", {z.dtype}"))
    if b_in.dtype != c_in.dtype or (b_in.dtype != dtype and b_in.dtype != f32):
        if not (b_in.is_floating_point() and c_in.is_floating_point()):
            raise RuntimeError(f"B and C must be floating point; got {b_in.dtype}, {c_in.dtype}")
        b_in, c_in = b_in.float(), c_in.float()
    if aneg.dtype != f32 or (d_skip is not None and d_skip.dtype != f32):
        if not aneg.is_floating_point() or (d_skip is not None and not d_skip.is_floating_point()):
            raise RuntimeError("Aneg and d_skip must be floating point")
        aneg, d_skip = aneg.float(), None if d_skip is None else d_skip.float()
    if n % 4 != 0 or n <= 0 or n > 64:
        raise ValueError(f"d_state must be a positive multiple of 4 no larger than 64 for the CUDA scan; got {n} "
                         "(scan_impl='torch' takes any size)")
    if state.dtype != f32 or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be float32, contiguous and 16-byte aligned (it is updated in place); got "
                         f"{state.dtype}, strides {state.stride()}")
    most = _native.SERVE_MAX
    if rows > most or places > most or count > most or d > _native.SERVE_MAX_DIM:
        raise ValueError(f"selective_scan_packed takes up to {most} rows, sequences and places and "
                         f"{_native.SERVE_MAX_DIM} channels")
    if d == 0 or count == 0 or places == 0 or rows == 0:
        return _nothing_packed(x, state, count, slots, out_slots)
    with _native.on_device(x.device):
        group = 4 if starts is None else 1
        if d_skip is not None and not d_skip.is_contiguous():
            d_skip = d_skip.contiguous()
        return _native.scan_packed(rows_of(x), rows_of(dt), _aligned(aneg, 16), rows_of(b_in, group),
                                   rows_of(c_in, group), None if z is None else rows_of(z), d_skip, dt_range,
                                   state, int_list(starts), int_list(slots), int_list(out_slots), count)


def _nothing_packed(x, cache, count, slots, out_slots):
    """The calls without a kernel: no channels, no sequences, no places or no rows. Without rows
    the (empty) sequences still hand their states on; without places a cache cannot be named."""
    if x.shape[0] and cache.shape[0] == 0 and count and x.shape[1]:
        raise ValueError("the cache has no place; give it one, even where every sequence starts from nothing")
    if count and cache.numel() and out_slots is not None:
        places, lead = cache.shape[0], (-1,) + (1,) * (cache.dim() - 1)
        order = torch.arange(count, device=x.device)
        src, dst = order if slots is None else slots.long(), out_slots.long()
        # every place's sequence, -1 for none (one place more takes those that leave nothing)
        writer = torch.full((places + 1,), -1, dtype=torch.int64, device=x.device)
        writer.scatter_(0, torch.where((dst >= 0) & (dst < places), dst, places), order)
        writer = writer[:places]
        # every place takes what the sequence that names it goes on from; others keep theirs
        src = src[writer.clamp(min=0)]
        old = cache[src.clamp(0, places - 1)]
        old = torch.where(((src >= 0) & (src < places)).view(lead), old, torch.zeros_like(old))
        cache.copy_(torch.where((writer >= 0).view(lead), old, cache))
    return torch.zeros_like(x, memory_format=torch.contiguous_format)
