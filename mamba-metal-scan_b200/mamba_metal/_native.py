"""ctypes binding of libmms_scan.so (C ABI in include/mms_scan.h).

The library is built in-tree (mamba-metal-scan_b200/build.py) into
mamba_metal/lib/. There is no fallback: if the library is missing or does not
load, every CUDA scan call raises RuntimeError naming the problem.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os
import threading
from pathlib import Path

import torch

LIB_PATH = Path(os.environ.get("MMS_SCAN_LIB", Path(__file__).resolve().parent / "lib" / "libmms_scan.so"))

MMS_OK = 0
MMS_ERR_INVALID_ARG = 1
MMS_ERR_UNSUPPORTED_N = 2
MMS_ERR_WORKSPACE = 3
MMS_ERR_MISALIGNED = 4
MMS_ERR_CUDA = 5
MMS_ERR_TOO_LARGE = 6
MMS_ERR_TIMEOUT = 7
MMS_ERR_UNSUPPORTED_BF16 = 8

# Every symbol include/mms_scan.h declares, with its ctypes signature.
_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
_Z = ctypes.c_size_t
_F = ctypes.c_float
SIGNATURES = {
    "mms_abi_version": ([], _I),
    "mms_status_string": ([_I], ctypes.c_char_p),
    "mms_last_cuda_error": ([], ctypes.c_char_p),
    "mms_fwd": ([_P] * 7 + [_I] * 5 + [_P], _I),
    "mms_bwd_workspace_size": ([_I] * 5, ctypes.c_size_t),
    "mms_bwd": ([_P] * 13 + [ctypes.c_size_t] + [_I] * 5 + [_P], _I),
    "mms_bwd_noalloc": ([_P] * 12 + [_I] * 5 + [_P], _I),
    "mms_step": ([_P] * 7 + [_I] * 3 + [_P], _I),
    "mms_device_status": ([], _I),
    "mms_gate_workspace_size": ([_I] * 3, ctypes.c_size_t),
    "mms_gate_fwd": ([_P, _P, ctypes.c_longlong] + [_P] * 2 + [_I] * 3 + [_P], _I),
    "mms_gate_bwd": ([_P] * 3 + [ctypes.c_longlong] + [_P] * 5 + [ctypes.c_size_t] + [_I] * 3
                     + [_P], _I),
    "mms_fwd_proj": ([_P] * 5 + [ctypes.c_float] * 2 + [_P] * 2 + [_I] * 5 + [_P], _I),
    "mms_bwd_proj": ([_P] * 7 + [ctypes.c_float] * 2 + [_P] * 6 + [ctypes.c_size_t] + [_I] * 5
                     + [_P], _I),
    "mms_fwd_bf16": ([_P] * 7 + [_I] * 5 + [_P], _I),
    "mms_bwd_bf16": ([_P] * 13 + [ctypes.c_size_t] + [_I] * 5 + [_P], _I),
    "mms_head_kept_size": ([_I] * 2, _Z),
    "mms_head_workspace_size": ([_I] * 5 + [_L] * 2 + [_I], _Z),
    "mms_linear_ce_fwd": ([_P, _L, _P, _L, _P, _L, _I] + [_P] * 3 + [_Z] + [_I] * 4 + [_P], _I),
    "mms_linear_ce_bwd": ([_P, _L, _P, _L, _P, _L, _I] + [_P] * 5 + [_Z] + [_I] * 4 + [_P], _I),
    "mms_linear_kd_fwd": ([_P, _L, _P, _L, _P, _P, _I, _F, _I] + [_P] * 3 + [_Z] + [_I] * 4
                          + [_P], _I),
    "mms_linear_kd_bwd": ([_P, _L, _P, _L, _P, _I, _F, _I] + [_P] * 5 + [_Z] + [_I] * 4 + [_P], _I),
    "mms_norm_workspace_size": ([_I] * 2, _Z),
    "mms_norm_fwd": ([_P] * 3 + [_L] + [_P] * 3 + [_F] + [_P] * 3 + [_I] * 3 + [_P], _I),
    "mms_norm_bwd": ([_P] * 3 + [_L] + [_P] * 13 + [_Z] + [_I] * 3 + [_P], _I),
    "mms_debug_set_wait": ([ctypes.c_uint, _I], _I),
    "mms_probe_pipe": ([_I] * 3 + [_P] * 4, _I),
    "mms_probe_ops_per_cta": ([_I] * 2, ctypes.c_longlong),
    "mms_probe_exp2": ([_P, _P, ctypes.c_longlong, _I, _P], _I),
}

# mms_probe_pipe kinds
PROBE_KINDS = {"ex2": 0, "ffma": 1, "ffma2": 2, "shfl": 3, "ex2_poly": 4, "ex2_poly2": 5}

_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load (once) and return the library; raises RuntimeError if unavailable."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(
                    f"the CUDA selective-scan library is not built: {LIB_PATH} is missing "
                    "(run `python mamba-metal-scan_b200/build.py`)")
            try:
                lib = ctypes.CDLL(str(LIB_PATH))
            except OSError as e:
                raise RuntimeError(f"cannot load {LIB_PATH}: {e}") from e
            for name, (args, res) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = res
            _lib = lib
    return _lib


def status_string(rc: int) -> str:
    return load().mms_status_string(rc).decode()


def _check(rc: int, what: str) -> None:
    if rc != MMS_OK:
        extra = f": {load().mms_last_cuda_error().decode()}" if rc == MMS_ERR_CUDA else ""
        raise RuntimeError(f"{what} failed: status {rc} ({status_string(rc)}){extra}")


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


# the current stream's handle without building a Stream object, where this torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def fwd(x, dt, aneg, b_in, c_in, chunk: int, proj=None):
    """y (B,T,D) and ckpt (B, ceil(T/chunk), D, N) on the current stream.

    proj = (dt_min, dt_max): dt holds logits and aneg the raw A of the fused
    prologue (mms_fwd_proj)."""
    lib = load()
    bt, t_len, d = x.shape
    n = aneg.shape[1]
    nchunk = (t_len + chunk - 1) // chunk
    y = torch.empty(bt, t_len, d, device=x.device, dtype=torch.float32)
    ckpt = torch.empty(bt, nchunk, d, n, device=x.device, dtype=torch.float32)
    if proj is None:
        rc = lib.mms_fwd(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in), _ptr(y),
                         _ptr(ckpt), bt, t_len, d, n, chunk, _stream(x.device))
        _check(rc, "mms_fwd")
    else:
        rc = lib.mms_fwd_proj(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in),
                              float(proj[0]), float(proj[1]), _ptr(y), _ptr(ckpt),
                              bt, t_len, d, n, chunk, _stream(x.device))
        _check(rc, "mms_fwd_proj")
    return y, ckpt


def bwd_workspace_size(bt: int, t_len: int, d: int, n: int, chunk: int) -> int:
    return int(load().mms_bwd_workspace_size(bt, t_len, d, n, chunk))


def bwd(x, dt, aneg, b_in, c_in, dy, ckpt, chunk: int, workspace=None, proj=None):
    """(dx, ddt, dAneg, dB, dC) on the current stream (with proj: the
    gradients of the logits and of the raw A in place of ddt and dAneg)."""
    lib = load()
    bt, t_len, d = x.shape
    n = aneg.shape[1]
    dx = torch.empty_like(x)
    ddt = torch.empty_like(dt)
    daneg = torch.empty_like(aneg)
    db = torch.empty_like(b_in)
    dc = torch.empty_like(c_in)
    ws_bytes = bwd_workspace_size(bt, t_len, d, n, chunk)
    if workspace is None or workspace.numel() < ws_bytes:
        workspace = torch.empty(max(ws_bytes, 1), device=x.device, dtype=torch.uint8)
    if proj is None:
        rc = lib.mms_bwd(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in), _ptr(dy),
                         _ptr(ckpt), _ptr(dx), _ptr(ddt), _ptr(daneg), _ptr(db), _ptr(dc),
                         _ptr(workspace), workspace.numel(),
                         bt, t_len, d, n, chunk, _stream(x.device))
        _check(rc, "mms_bwd")
    else:
        rc = lib.mms_bwd_proj(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in), _ptr(dy),
                              _ptr(ckpt), float(proj[0]), float(proj[1]),
                              _ptr(dx), _ptr(ddt), _ptr(daneg), _ptr(db), _ptr(dc),
                              _ptr(workspace), workspace.numel(),
                              bt, t_len, d, n, chunk, _stream(x.device))
        _check(rc, "mms_bwd_proj")
    return dx, ddt, daneg, db, dc


def fwd_bf16(x, dt, aneg, b_in, c_in, chunk: int):
    """mms_fwd_bf16: x, dt bf16 (B,T,D), Aneg/B/C fp32; returns y bf16 (B,T,D)
    and the fp32 ckpt (B, ceil(T/chunk), D, N)."""
    lib = load()
    bt, t_len, d = x.shape
    n = aneg.shape[1]
    nchunk = (t_len + chunk - 1) // chunk
    y = torch.empty(bt, t_len, d, device=x.device, dtype=torch.bfloat16)
    ckpt = torch.empty(bt, nchunk, d, n, device=x.device, dtype=torch.float32)
    rc = lib.mms_fwd_bf16(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in), _ptr(y),
                          _ptr(ckpt), bt, t_len, d, n, chunk, _stream(x.device))
    _check(rc, "mms_fwd_bf16")
    return y, ckpt


def bwd_bf16(x, dt, aneg, b_in, c_in, dy, ckpt, chunk: int, workspace=None):
    """mms_bwd_bf16: (dx, ddt) bf16 and (dAneg, dB, dC) fp32."""
    lib = load()
    bt, t_len, d = x.shape
    n = aneg.shape[1]
    dx = torch.empty_like(x)
    ddt = torch.empty_like(dt)
    daneg = torch.empty_like(aneg)
    db = torch.empty_like(b_in)
    dc = torch.empty_like(c_in)
    ws_bytes = bwd_workspace_size(bt, t_len, d, n, chunk)
    if workspace is None or workspace.numel() < ws_bytes:
        workspace = torch.empty(max(ws_bytes, 1), device=x.device, dtype=torch.uint8)
    rc = lib.mms_bwd_bf16(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in), _ptr(dy),
                          _ptr(ckpt), _ptr(dx), _ptr(ddt), _ptr(daneg), _ptr(db), _ptr(dc),
                          _ptr(workspace), workspace.numel(),
                          bt, t_len, d, n, chunk, _stream(x.device))
    _check(rc, "mms_bwd_bf16")
    return dx, ddt, daneg, db, dc


def step(x, dt, aneg, b_in, c_in, h):
    """One decode step: updates h (B,D,N) in place, returns y (B,D)."""
    lib = load()
    bt, d = x.shape
    n = aneg.shape[1]
    y = torch.empty(bt, d, device=x.device, dtype=torch.float32)
    rc = lib.mms_step(_ptr(x), _ptr(dt), _ptr(aneg), _ptr(b_in), _ptr(c_in), _ptr(h), _ptr(y),
                      bt, d, n, _stream(x.device))
    _check(rc, "mms_step")
    return y


def device_status() -> int:
    """MMS_OK, or MMS_ERR_TIMEOUT if a kernel's bounded wait ran out since the last call."""
    return int(load().mms_device_status())


def gate_fwd(y, z, d_skip):
    """out = (y + d_skip) * silu(z) in one kernel; z may have a row stride."""
    lib = load()
    bt, t_len, d = y.shape
    out = torch.empty_like(y)
    rc = lib.mms_gate_fwd(_ptr(y), _ptr(z), z.stride(1), _ptr(d_skip), _ptr(out), bt, t_len, d,
                          _stream(y.device))
    _check(rc, "mms_gate_fwd")
    return out


def gate_bwd(dout, y, z, d_skip):
    """(dy, dz, d_dskip) of gate_fwd in one kernel (plus a fixed-order reduction)."""
    lib = load()
    bt, t_len, d = y.shape
    dy, dd = torch.empty_like(y), torch.empty_like(d_skip)
    dz = torch.empty(y.shape, device=y.device, dtype=torch.float32)
    nb = int(lib.mms_gate_workspace_size(bt, t_len, d))
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=y.device)
    rc = lib.mms_gate_bwd(_ptr(dout), _ptr(y), _ptr(z), z.stride(1), _ptr(d_skip), _ptr(dy),
                          _ptr(dz), _ptr(dd), _ptr(ws), nb, bt, t_len, d, _stream(y.device))
    _check(rc, "mms_gate_bwd")
    return dy, dz, dd


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """torch.cuda.device(device), or a context that costs nothing where it is current already."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _dtype(t) -> int:
    return 1 if t.dtype == torch.bfloat16 else 0


@functools.lru_cache(maxsize=256)
def _head_sizes(m: int, v: int, d: int, k: int, dtype: int, ldx: int, ldw: int, backward: bool):
    """(workspace, kept) bytes, the workspace rounded up to 256."""
    lib = load()
    ws = int(lib.mms_head_workspace_size(m, v, d, k, dtype, ldx, ldw, int(backward)))
    return (ws + 255) // 256 * 256, int(lib.mms_head_kept_size(m, k))


def _head_buffers(x, w, k: int, keep: bool):
    """(workspace address, its bytes, kept address, kept tensor, all that must live until the call).
    Without `keep` what the backward would need goes behind the workspace, in one allocation."""
    nb, kept_nb = _head_sizes(x.shape[0], w.shape[0], x.shape[1], k, _dtype(x), x.stride(0),
                              w.stride(0), False)
    if not keep:
        ws = torch.empty(nb + kept_nb, dtype=torch.uint8, device=x.device)
        base = ws.data_ptr()
        return base, nb, base + nb, None, ws
    ws = torch.empty(nb, dtype=torch.uint8, device=x.device)
    kept = torch.empty(kept_nb, dtype=torch.uint8, device=x.device)
    return ws.data_ptr(), nb, kept.data_ptr(), kept, ws


def _head_workspace(x, w, k: int):
    """The backward's."""
    nb, _ = _head_sizes(x.shape[0], w.shape[0], x.shape[1], k, _dtype(x), x.stride(0), w.stride(0),
                        True)
    return torch.empty(nb, dtype=torch.uint8, device=x.device)


def linear_ce_fwd(x, w, target, ignore_index: int, reduction: str, keep: bool = True):
    """(loss, kept) of mms_linear_ce_fwd; x (M, D), w (V, D) with row strides. kept: what the
    backward needs (None without `keep`)."""
    m, d = x.shape
    red = REDUCTIONS[reduction]
    loss = torch.empty((m,) if red == 0 else (), device=x.device, dtype=torch.float32)
    ws, nb, kept_at, kept, _live = _head_buffers(x, w, 0, keep)
    rc = load().mms_linear_ce_fwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0),
                                  target.data_ptr(), ignore_index, red, loss.data_ptr(),
                                  kept_at, ws, nb, m, w.shape[0], d, _dtype(x),
                                  _stream(x.device))
    if rc:
        _check(rc, "mms_linear_ce_fwd")
    return loss, kept


def _head_grads(x, w, need_x: bool, need_w: bool):
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need_x else None
    dw = torch.empty(w.shape, device=w.device, dtype=w.dtype) if need_w else None
    return dx, dw, 0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr()


def linear_ce_bwd(x, w, target, ignore_index: int, reduction: str, dloss, kept,
                  need_x: bool = True, need_w: bool = True):
    """(dx, dw) of mms_linear_ce_bwd; None for one that is not needed."""
    m, d = x.shape
    dx, dw, pdx, pdw = _head_grads(x, w, need_x, need_w)
    ws = _head_workspace(x, w, 0)
    rc = load().mms_linear_ce_bwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0),
                                  target.data_ptr(), ignore_index, REDUCTIONS[reduction],
                                  dloss.data_ptr(), kept.data_ptr(), pdx, pdw, ws.data_ptr(),
                                  ws.numel(), m, w.shape[0], d, _dtype(x), _stream(x.device))
    if rc:
        _check(rc, "mms_linear_ce_bwd")
    return dx, dw


def linear_kd_fwd(x, w, index, logits, temperature: float, reduction: str, keep: bool = True):
    """(loss, kept) of mms_linear_kd_fwd. kept: what the backward needs (None without `keep`)."""
    m, d = x.shape
    k = index.shape[1]
    red = REDUCTIONS[reduction]
    loss = torch.empty((m,) if red == 0 else (), device=x.device, dtype=torch.float32)
    ws, nb, kept_at, kept, _live = _head_buffers(x, w, k, keep)
    rc = load().mms_linear_kd_fwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0),
                                  index.data_ptr(), logits.data_ptr(), k, temperature, red,
                                  loss.data_ptr(), kept_at, ws, nb, m, w.shape[0], d, _dtype(x),
                                  _stream(x.device))
    if rc:
        _check(rc, "mms_linear_kd_fwd")
    return loss, kept


def linear_kd_bwd(x, w, index, temperature: float, reduction: str, dloss, kept,
                  need_x: bool = True, need_w: bool = True):
    """(dx, dw) of mms_linear_kd_bwd; None for one that is not needed."""
    m, d = x.shape
    k = index.shape[1]
    dx, dw, pdx, pdw = _head_grads(x, w, need_x, need_w)
    ws = _head_workspace(x, w, k)
    rc = load().mms_linear_kd_bwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0),
                                  index.data_ptr(), k, temperature, REDUCTIONS[reduction],
                                  dloss.data_ptr(), kept.data_ptr(), pdx, pdw,
                                  ws.data_ptr(), ws.numel(), m, w.shape[0], d, _dtype(x),
                                  _stream(x.device))
    if rc:
        _check(rc, "mms_linear_kd_bwd")
    return dx, dw


def _opt(t) -> int:
    return 0 if t is None else _ptr(t)


def norm_fwd(x, y, gate, weight, post, scale, eps: float, keep: bool = True):
    """(h, u, stat) of mms_norm_fwd; x, y (M, D) contiguous, gate (M, D) with a row stride.
    stat: what the backward needs (None without `keep`)."""
    m, d = x.shape
    h, u = torch.empty_like(x), torch.empty_like(x)
    stat = torch.empty(m, 2, device=x.device, dtype=torch.float32) if keep else None
    rc = load().mms_norm_fwd(_ptr(x), _ptr(y), _opt(gate), d if gate is None else gate.stride(0),
                             _ptr(weight), _opt(post), _opt(scale), eps, _ptr(h), _ptr(u),
                             _opt(stat), m, d, _dtype(x), _stream(x.device))
    if rc:
        _check(rc, "mms_norm_fwd")
    return h, u, stat


def norm_bwd(x, y, gate, weight, post, scale, stat, dh, du):
    """(dx, dy, dgate, dweight, dpost, dscale) of mms_norm_bwd; None beside an input that is None."""
    m, d = x.shape
    dx = torch.empty_like(x)
    # without gate, post and scale the gradients of x and y are the same values
    dy = dx if gate is None and post is None and scale is None else torch.empty_like(x)
    dgate = None if gate is None else torch.empty_like(x)
    dweight = torch.empty_like(weight)
    dpost, dscale = (None if t is None else torch.empty_like(t) for t in (post, scale))
    lib = load()
    nb = int(lib.mms_norm_workspace_size(m, d))
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=x.device)
    rc = lib.mms_norm_bwd(_ptr(x), _ptr(y), _opt(gate), d if gate is None else gate.stride(0),
                          _ptr(weight), _opt(post), _opt(scale), _ptr(stat), _ptr(dh), _ptr(du),
                          _ptr(dx), _ptr(dy), _opt(dgate), _ptr(dweight), _opt(dpost), _opt(dscale),
                          _ptr(ws), nb, m, d, _dtype(x), _stream(x.device))
    if rc:
        _check(rc, "mms_norm_bwd")
    return dx, dy, dgate, dweight, dpost, dscale


def pipe_rate(kind: str, device=None, iters: int = 4096, ctas_per_sm: int = 4) -> float:
    """Operations per SM per clock of one pipe (mms_probe_pipe), measured on the
    SM cycle counters: per SM, the operations of its CTAs over its longest CTA;
    the median over SMs. kind: one of PROBE_KINDS."""
    lib = load()
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    n_sm = torch.cuda.get_device_properties(device).multi_processor_count
    blocks = n_sm * ctas_per_sm
    sink = torch.empty(256, device=device, dtype=torch.float32)
    cycles = torch.empty(blocks, dtype=torch.int64, device=device)
    sm = torch.empty(blocks, dtype=torch.int32, device=device)
    k = PROBE_KINDS[kind]
    for _ in range(2):                       # the first launch warms the clocks up
        _check(lib.mms_probe_pipe(k, iters, blocks, _ptr(sink), _ptr(cycles), _ptr(sm),
                                  _stream(device)), "mms_probe_pipe")
    torch.cuda.synchronize(device)
    ops = int(lib.mms_probe_ops_per_cta(k, iters))
    per_sm = {}
    for c, s in zip(cycles.tolist(), sm.tolist()):
        n, m = per_sm.get(s, (0, 0))
        per_sm[s] = (n + 1, max(m, c))
    rates = sorted(n * ops / m for n, m in per_sm.values())
    return rates[len(rates) // 2]
