"""The convolution kernels against float64, within the bounds of tests/_serve_ref.py."""
from __future__ import annotations

import pytest
import torch

from _serve_ref import close, conv_bound, conv_grad_bounds
from mamba_metal import causal_conv, causal_conv_packed, causal_conv_packed_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def make(bt, t, d, k, dtype, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(bt, t, d, generator=g).to(dtype)
    w = (torch.randn(d, k, generator=g) / k ** 0.5).to(dtype)
    b = (0.3 * torch.randn(d, generator=g)).to(dtype) if bias else None
    return x, w, b, torch.randn(bt, t, d, generator=g).to(dtype)


def check(x, w, b, dy, silu, got=None):
    dtype = x.dtype
    leaves = [t.detach().to(DEV).requires_grad_(True) for t in (x, w) + (() if b is None else (b,))]
    if got is None:
        y = causal_conv(*leaves, silu=silu)
        got = (y, *torch.autograd.grad(y, leaves, dy.to(DEV)))
    close(got[0], *conv_bound(x, w, b, silu, dtype), "y")
    # rows of a warp (at most 128), its CTA's 4 warps, every eighth of the partial sums, 8 of them
    depth = 128 + 4 + 8 + x.shape[0] * x.shape[1] / 64 / 8
    for n, gr, wb in zip(("dx", "dw", "dbias"), got[1:], conv_grad_bounds(x, w, b, dy, silu, dtype, depth)):
        assert gr.dtype == dtype
        close(gr, *wb, n)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("bt,t,d,k", [(1, 1, 1, 4), (1, 1, 64, 2), (2, 3, 36, 4), (3, 7, 33, 3), (1, 2, 8, 8), (2, 65, 130, 4),
                                      (1, 200, 4, 5), (2, 130, 12, 1), (2, 40, 256, 6), (3, 1001, 21, 4), (1, 4099, 132, 3),
                                      (5, 9, 1433, 4), (2, 33, 260, 8), (40, 2, 16, 7)])
def test_conv_matches_float64(bt, t, d, k, silu, dtype):
    check(*make(bt, t, d, k, dtype, seed=t + d), silu)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_bias(dtype):
    x, w, _, dy = make(2, 50, 72, 4, dtype, bias=False)
    check(x, w, None, dy, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_with_strides_and_unaligned_bases(dtype):
    """x as a half of a wider array, off a group of 4, time first, one row for all; weight as nn.Conv1d has it."""
    x, w, b, dy = make(3, 21, 24, 4, dtype)
    leaves = [t.to(DEV).requires_grad_(True) for t in (w, b)]
    base = causal_conv(x.to(DEV), *leaves)
    wide = torch.full((3, 21, 61), float("nan"), dtype=dtype, device=DEV)
    for off in (0, 1, 4, 37):
        wide[:, :, off:off + 24] = x.to(DEV)
        v = wide[:, :, off:off + 24].detach().requires_grad_(True)
        y = causal_conv(v, leaves[0][:, None], leaves[1])
        check(x, w, b, dy, True, (y, *torch.autograd.grad(y, [v, *leaves], dy.to(DEV))))
    assert torch.equal(causal_conv(x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1), *leaves), base)
    assert torch.equal(causal_conv(x.permute(0, 2, 1).contiguous().to(DEV).permute(0, 2, 1), *leaves), base)
    one = x[:1, :1].to(DEV)
    assert torch.equal(causal_conv(one.expand(2, 5, 24), *leaves), causal_conv(one.repeat(2, 5, 1), *leaves))
    grad = torch.autograd.grad(base, leaves, dy.to(DEV).permute(1, 0, 2).contiguous().permute(1, 0, 2))
    assert all(torch.equal(a, c) for a, c in zip(grad, torch.autograd.grad(causal_conv(x.to(DEV), *leaves), leaves, dy.to(DEV))))


def test_gradient_against_differences():
    x, w, b, dy = make(1, 12, 5, 4, F32)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(causal_conv(*leaves), leaves, dy.to(DEV))
    loss = lambda ts: float((causal_conv(*ts).double() * dy.to(DEV).double()).sum())
    step = 2.0 ** -7
    for i, (leaf, gr) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        moved = [[t.detach() + s * step * way if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1)]
        diff = (loss(moved[0]) - loss(moved[1])) / (2 * step)
        # third derivatives of SiLU are below 1 in magnitude (the pre-activations move by a few steps);
        # the values' float32 roundings are divided by the step
        size = float((dy.abs().sum() * (1 + w.abs().sum(1).max()) ** 3) * way.abs().max() ** 3)
        assert abs(diff - float((gr.double() * way.double()).sum())) <= size * (step ** 2 + 2.0 ** -21 / step)


@pytest.mark.parametrize("k", [3, 4, 5])
def test_infinities_and_nan_stay_with_their_rows(k):
    """A row sees its own K inputs and no others: not the taps that are not there, not its neighbours."""
    x, w, b, _ = make(1, 40, 8, k, F32)
    clean = causal_conv(x.to(DEV), w.to(DEV), b.to(DEV), silu=False)
    for bad in (float("inf"), float("nan")):
        y = x.clone()
        y[0, 20, 3] = bad
        got = causal_conv(y.to(DEV), w.to(DEV), b.to(DEV), silu=False)
        hit = torch.zeros(40, 8, dtype=torch.bool)
        hit[20:20 + k, 3] = True
        assert not torch.isfinite(got[0].cpu()[hit]).any() and torch.equal(got[0].cpu()[~hit], clean[0].cpu()[~hit])
    big = torch.full((1, 3, 4), -1e30, device=DEV)
    assert (causal_conv(big, torch.ones(4, 2, device=DEV), None) == 0).all()


def test_empty_and_refused():
    x, w, b, _ = (t.to(DEV) for t in make(2, 5, 8, 4, F32))
    assert causal_conv(x[:, :0], w, b).shape == (2, 0, 8) and causal_conv(x[:0], w, b).shape == (0, 5, 8)
    v = x[:0].requires_grad_(True)
    assert torch.autograd.grad(causal_conv(v, w, b).sum(), v)[0].shape == (0, 5, 8)
    for bad in ((x.half(), w.half(), b.half()), (x, w.bfloat16(), b), (x.double(), w.double(), b.double())):
        with pytest.raises(RuntimeError, match="float32 or bfloat16"):
            causal_conv(*bad)
    with pytest.raises(RuntimeError, match="same CUDA device"):
        causal_conv(x, w.cpu(), b)
    with pytest.raises(ValueError, match="taps"):
        causal_conv(x, torch.zeros(8, 9, device=DEV), b)
    with pytest.raises(ValueError, match="contiguous"):
        causal_conv_packed(x[0], w, b, torch.zeros(3, 3, 8, device=DEV).transpose(1, 2), torch.tensor([0, 5], device=DEV))


def test_same_result_every_time_and_on_another_stream_and_in_a_graph():
    x, w, b, dy = (t.to(DEV) for t in make(4, 700, 200, 4, BF16))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = causal_conv(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, step()))


# -------------------------------------------------------------------- packed

def packed_case(lens, d, k, dtype, seed=0, lead=0, tail=0, places=9):
    g = torch.Generator().manual_seed(seed)
    rows = lead + sum(lens) + tail
    x = torch.randn(rows, d, generator=g).to(dtype)
    w = (torch.randn(d, k, generator=g) / k ** 0.5).to(dtype)
    b = (0.3 * torch.randn(d, generator=g)).to(dtype)
    starts = torch.tensor([lead] + lens).cumsum(0)
    window = torch.randn(places, d, k - 1, generator=g).to(dtype)
    order = torch.randperm(places, generator=g)
    slots, out = order[:len(lens)].clone(), order[len(order) - len(lens):].clone()
    if len(lens) > 2:
        slots[1], slots[2] = -1, slots[0]                  # one starts from nothing, two share a place
    return x, w, b, window, starts, slots, out


def check_packed(x, w, b, window, starts, slots, out, silu, ints=torch.int32):
    on = lambda t: None if t is None else t.to(DEV)
    mine = window.to(DEV)
    y = causal_conv_packed(on(x), on(w), on(b), mine, on(starts if starts is None else starts.to(ints)),
                           on(slots if slots is None else slots.to(ints)), on(out if out is None else out.to(ints)), silu)
    wide = window.double()
    want = causal_conv_packed_ref(x.double(), w.double(), b.double(), wide, starts, slots, out, silu)
    assert torch.equal(mine.cpu().double(), wide), "the window"
    # a row's output has at most K + 1 terms of these magnitudes
    inputs = torch.cat([x.double().abs().flatten(), window.double().abs().flatten()]).max()
    size = inputs * w.double().abs().sum(1).max() + b.double().abs().max()
    off = (w.shape[1] + 2 + size + 16) * 2.0 ** -24 * size
    close(y, want, off + (2.0 ** -8 if x.dtype == BF16 else 2.0 ** -24) * (want.abs() + off), "y")
    return y, mine


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,k", [(8, 4), (33, 4), (128, 2), (260, 3), (12, 8), (5, 5), (64, 1)])
def test_packed_matches_float64(d, k, dtype):
    for i, lens in enumerate(([1], [7], [0], [1, 1, 1, 1], [3, 0, 1, 40, 2], [9, 8, 200], [0, 0, 5])):
        case = packed_case(lens, d, k, dtype, seed=i + d, lead=i % 3, tail=(i + 1) % 4)
        check_packed(*case, silu=i % 2 == 0, ints=torch.int64 if i % 2 else torch.int32)
    x, w, b, window, _, _, _ = packed_case([1] * 9, d, k, dtype, seed=d)
    check_packed(x, w, b, window, None, None, None, True)                      # single tokens in place
    check_packed(x[:4], w, b, window, None, torch.tensor([5, -1, 5, 0]), torch.tensor([1, 2, 3, 0]), True)


def test_packed_in_place_strided_rows_and_pieces():
    x, w, b, window, starts, slots, _ = packed_case([30, 3, 50], 40, 4, F32, places=5)
    slots = torch.tensor([4, 0, 2])
    y, after = check_packed(x, w, b, window, starts, slots, None, True)
    wide = torch.full((83, 97), float("nan"), device=DEV)
    wide[:, 57:] = x.to(DEV)
    again = window.to(DEV)
    assert torch.equal(causal_conv_packed(wide[:, 57:], w.to(DEV), b.to(DEV), again, starts.to(DEV), slots.to(DEV)), y)
    assert torch.equal(again, after)
    # the same rows in pieces of one to many, the window between them
    whole = causal_conv(x[None].to(DEV), w.to(DEV), b.to(DEV))[0]
    cache = torch.zeros(2, 40, 3, device=DEV)
    got, at = [], 0
    for n in (1, 1, 2, 5, 17, 57):
        got.append(causal_conv_packed(x[at:at + n].to(DEV), w.to(DEV), b.to(DEV), cache,
                                      torch.tensor([0, n], device=DEV), torch.tensor([1], device=DEV)))
        at += n
    assert torch.equal(torch.cat(got), whole) and (cache[0] == 0).all()


def test_lists_that_break_the_rules_stay_inside_the_arrays():
    """Descending starts, starts and places far outside: some rows are wrong, nothing else is touched."""
    x, w, b, window, _, _, _ = packed_case([30], 40, 4, F32, places=5)
    guard = torch.full((7, 40, 3), 7.0, device=DEV)
    guard[1:6] = window.to(DEV)
    rows = torch.full((32, 40), float("nan"), device=DEV)
    rows[1:31] = x.to(DEV)
    for starts in ([20, 3, 9, 30], [-5, 2, 1 << 40, 4], [1 << 33, -(1 << 50), 7, 7], [0, 50, 60, 70]):
        y = causal_conv_packed(rows[1:31], w.to(DEV), b.to(DEV), guard[1:6], torch.tensor(starts, device=DEV),
                               torch.tensor([0, 1 << 40, -3], device=DEV), torch.tensor([1, 3, 1 << 35], device=DEV))
        torch.cuda.synchronize()
        assert y.shape == (30, 40) and (guard[0] == 7).all() and (guard[6] == 7).all()


def test_no_rows_hand_the_windows_on():
    window = torch.randn(4, 8, 3, device=DEV)
    old = window.clone()
    causal_conv_packed(torch.zeros(0, 8, device=DEV), torch.zeros(8, 4, device=DEV), None, window,
                       torch.tensor([0, 0, 0], device=DEV), torch.tensor([3, -1], device=DEV), torch.tensor([0, 1], device=DEV))
    assert torch.equal(window[0], old[3]) and (window[1] == 0).all() and torch.equal(window[2:], old[2:])
