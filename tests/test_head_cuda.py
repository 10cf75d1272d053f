"""The head's losses on the GPU (mms_linear_ce_*, mms_linear_kd_*) against float64.

Every case is compared element by element with the definition in float64 on the CPU, within
bounds that _head_ref.py derives from the number of roundings. A second, norm-wise check is as
sharp as independent roundings make it: bf16 gradients take two roundings (dz, the result), each
at most 2^-8 relative, so 2^-7 of the norm holds when no sum cancels below its largest term;
float32 gradients 2e-5 (sums of up to 4096 terms at 2^-24 each, all in one direction, are 2.4e-4;
independent ones 4e-6).
"""
from __future__ import annotations

import math

import pytest
import torch

from _head_ref import check, check_norm, solve, sparse, u
from mamba_metal import (_native, linear_cross_entropy, linear_cross_entropy_ref,
                         linear_distillation, linear_distillation_ref, residual_rms_norm)

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def head_inputs(rows, vocab, dim, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, dim, generator=gen) * (2.0 / math.sqrt(dim))
    target = torch.randint(0, vocab, (rows,), generator=gen)
    x = torch.randn(rows, dim, generator=gen) + 3 * torch.rand(rows, 1, generator=gen) * w[target]
    return x.to(dtype), w.to(dtype), target, gen


def leaves(x, w):
    return x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)


def compare(x, w, parts, tau, reduction, dloss, loss, grads):
    want = solve(x, w, *parts, tau, reduction, dloss)
    check("loss", loss, want["loss"], want["e_loss"])
    tol = 2.0 ** -7 if x.dtype == BF16 else 2e-5
    for name, got in zip(("dx", "dw"), grads):
        assert got.dtype == x.dtype
        check(name, got, want[name], want["e_" + name])
        # one entry in the vocabulary: q = p = 1 and the gradient is 0 by arithmetic, so a norm
        # has no scale there (0 / 0); the kernels' log2 of a float32 sum near 1 is exact to 2^-24
        # of 1, which the element-wise bound holds in absolute terms
        if w.shape[0] > 1:
            check_norm(name, got, want[name], tol)
    return want


def run_ce(x, w, target, reduction, dloss, ignore=-100):
    xd, wd = leaves(x, w)
    loss = linear_cross_entropy(xd, wd, target.to(DEV), ignore_index=ignore, reduction=reduction)
    return loss, torch.autograd.grad(loss, [xd, wd], dloss.to(DEV).reshape(loss.shape))


SIZES = [(1, 1, 1), (1, 5, 8), (3, 256, 64), (2, 257, 65), (130, 255, 63), (127, 513, 640),
         (128, 32, 200), (129, 1000, 72), (256, 512, 128), (257, 777, 1000), (600, 4100, 136),
         (64, 9001, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,dim", SIZES)
def test_cross_entropy_at_odd_sizes(rows, vocab, dim, dtype):
    x, w, target, gen = head_inputs(rows, vocab, dim, dtype, seed=rows + vocab + dim)
    reduction = ("none", "mean", "sum")[(rows + dim) % 3]
    dloss = torch.randn(rows, generator=gen) if reduction == "none" else torch.tensor(0.7)
    loss, grads = run_ce(x, w, target, reduction, dloss)
    compare(x, w, sparse(1, target=target, ignore=-100), 1.0, reduction, dloss, loss, grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,dim,k,tau", [(1, 1, 1, 1, 1.0), (1, 70, 24, 1, 2.0), (5, 300, 65, 7, 0.5),
                                                  (130, 1000, 72, 33, 2.0), (257, 513, 640, 64, 4.0),
                                                  (40, 2000, 128, 1024, 1.0), (600, 5000, 64, 500, 2.0)])
def test_distillation_at_odd_sizes(rows, vocab, dim, k, tau, dtype):
    x, w, _, gen = head_inputs(rows, vocab, dim, dtype, seed=rows + vocab + dim)
    index = torch.randint(0, vocab, (rows, k), generator=gen)          # with repeats
    logits = 3 * torch.randn(rows, k, generator=gen)
    reduction = ("mean", "none", "sum")[rows % 3]
    dloss = torch.randn(rows, generator=gen) if reduction == "none" else torch.tensor(-1.3)
    xd, wd = leaves(x, w)
    loss = linear_distillation(xd, wd, index.to(DEV), logits.to(DEV), temperature=tau, reduction=reduction)
    grads = torch.autograd.grad(loss, [xd, wd], dloss.to(DEV).reshape(loss.shape))
    parts = sparse(k, index=index, logits=logits, tau=tau)
    compare(x, w, parts, tau, reduction, dloss, loss, grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pieces_of_the_vocabulary(dtype, monkeypatch):
    """More than one piece: rows * 4096 entries of dz exceed the bound on a piece."""
    rows, vocab, dim = (12000, 30000, 16) if dtype == F32 else (36000, 9000, 16)
    x, w, target, gen = head_inputs(rows, vocab, dim, dtype, seed=3)
    target[::3] = -100
    loss, grads = run_ce(x, w, target, "mean", torch.tensor(1.0))
    # float64 on the GPU, in row blocks: the CPU would take minutes
    xd, wd, t = x.to(DEV).double(), w.to(DEV).double(), target.to(DEV)
    keep = t >= 0
    n = keep.sum()
    total, dx, dw = 0.0, torch.empty_like(xd), torch.zeros_like(wd)
    for a in range(0, rows, 4000):
        s = slice(a, a + 4000)
        z = xd[s] @ wd.t()
        lse = torch.logsumexp(z, 1)
        at = t[s].clamp(min=0)[:, None]
        total += float(((lse - z.gather(1, at)[:, 0]) * keep[s]).sum())
        d = torch.exp(z - lse[:, None]).scatter_add(1, at, torch.full_like(at, -1, dtype=z.dtype))
        d = d * (keep[s] / n)[:, None]
        dx[s] = d @ wd
        dw += d.t() @ (xd[s] * keep[s][:, None])
    assert abs(float(loss.detach()) - total / float(n)) <= 2e-6 * abs(total / float(n))
    tol = 2.0 ** -7 if dtype == BF16 else 2e-5
    check_norm("dx", grads[0], dx.cpu(), tol)
    check_norm("dw", grads[1], dw.cpu(), tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_probabilities_of_long_lists(dtype):
    """Teacher probabilities near 1e-3 against student ones near 1e-5: dz is their difference to
    float32's roundoff of its own size (8 roundings: 5e-7), not of 1."""
    rows, vocab, dim, k = 400, 20000, 64, 1024
    x, w, _, gen = head_inputs(rows, vocab, dim, dtype, seed=21)
    index = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)])
    logits = 0.5 * torch.randn(rows, k, generator=gen)
    xd, wd = leaves(x, w)
    grads = torch.autograd.grad(linear_distillation(xd, wd, index.to(DEV), logits.to(DEV), 2.0), [xd, wd])
    want = solve(x, w, *sparse(k, index=index, logits=logits, tau=2.0), 2.0, "mean", torch.tensor(1.0))
    for name, got in zip(("dx", "dw"), grads):
        check(name, got, want[name], want["e_" + name])
        check_norm(name, got, want[name], 2.0 ** -7 if dtype == BF16 else 3e-6)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_left_out_rows_may_hold_anything(dtype):
    """Ignored rows with NaN and infinities: loss and gradient 0 there, none of it elsewhere."""
    x, w, target, gen = head_inputs(150, 400, 72, dtype, seed=5)
    target[::4] = 7777
    x[0], x[4], x[8, 3] = float("nan"), float("inf"), float("-inf")
    dloss = torch.randn(150, generator=gen)
    loss, grads = run_ce(x, w, target, "none", dloss, ignore=7777)
    parts = sparse(1, target=target, ignore=7777)
    compare(x, w, parts, 1.0, "none", dloss, loss, grads)
    assert (loss[::4] == 0).all() and (grads[0][::4] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,kept", [(513, 0.5), (700, 0.02), (1100, 0.9), (1100, 0.47), (2000, 0.0005)])
def test_many_rows_of_which_some_count(rows, kept, dtype):
    """Above 512 rows the products run over the listed rows alone: their numbers fall between
    tiles and steps, what is left out holds NaN, and every reduction puts results in place."""
    vocab, dim = 300, 72
    x, w, target, gen = head_inputs(rows, vocab, dim, dtype, seed=rows)
    out = torch.rand(rows, generator=gen) >= kept
    out[rows // 2] = False
    target[out] = -100
    x[out] = float("nan")
    for reduction in ("none", "mean", "sum"):
        dloss = torch.randn(rows, generator=gen) if reduction == "none" else torch.tensor(1.7)
        loss, grads = run_ce(x, w, target, reduction, dloss)
        compare(x, w, sparse(1, target=target, ignore=-100), 1.0, reduction, dloss, loss, grads)
        assert (grads[0].cpu()[out] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_lists_of_which_some_are_empty(dtype):
    rows, vocab, dim, k = 900, 700, 72, 9
    x, w, _, gen = head_inputs(rows, vocab, dim, dtype, seed=3)
    index = torch.randint(-2, vocab, (rows, k), generator=gen)
    logits = 2 * torch.randn(rows, k, generator=gen)
    index[::3] = -1
    logits[1::3] = float("-inf")
    index[7], logits[7] = 5, 0.25                        # one index nine times
    x[::3] = float("inf")
    parts = sparse(k, index=index, logits=logits, tau=1.5)
    for reduction in ("none", "mean"):
        dloss = torch.randn(rows, generator=gen) if reduction == "none" else torch.tensor(1.0)
        xd, wd = leaves(x, w)
        loss = linear_distillation(xd, wd, index.to(DEV), logits.to(DEV), 1.5, reduction=reduction)
        grads = torch.autograd.grad(loss, [xd, wd], dloss.to(DEV).reshape(loss.shape))
        compare(x, w, parts, 1.5, reduction, dloss, loss, grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 9, 700])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_every_row_left_out(reduction, rows, dtype):
    x, w, target, _ = head_inputs(rows, 50, 24, dtype)
    target[:] = -100
    loss, grads = run_ce(x, w, target, reduction, torch.ones(rows) if reduction == "none" else torch.tensor(1.0))
    if reduction == "mean":
        assert torch.isnan(loss)                                       # 0 / 0, as PyTorch's
    else:
        assert (loss == 0).all()
    assert all((gr == 0).all() for gr in grads)


def test_empty_places_of_a_teacher_list():
    """Negative indices, logits of -inf, NaN in empty places, rows with nothing left."""
    rows, vocab, dim, k = 40, 333, 72, 6
    x, w, _, gen = head_inputs(rows, vocab, dim, F32, seed=8)
    index = torch.randint(0, vocab, (rows, k), generator=gen)
    logits = 2 * torch.randn(rows, k, generator=gen)
    index[::3, 1::2] = -1
    logits[::3, 1] = float("nan")                                      # in an empty place
    logits[1::3, 2] = float("-inf")
    logits[2, :] = torch.finfo(torch.float32).min                      # the type's lowest: all alike
    index[5] = -1                                                      # nothing left
    logits[7] = float("-inf")                                          # nothing left either
    x[5] = float("nan")
    xd, wd = leaves(x, w)
    loss = linear_distillation(xd, wd, index.to(DEV), logits.to(DEV), temperature=2.0)
    grads = torch.autograd.grad(loss, [xd, wd])
    parts = sparse(k, index=index, logits=torch.where(index < 0, 0.0, logits), tau=2.0)
    assert not parts[3][5] and not parts[3][7] and parts[3].sum() == rows - 2
    compare(x, w, parts, 2.0, "mean", torch.tensor(1.0), loss, grads)


def test_indices_outside_the_vocabulary_are_loud_and_stay_in_bounds():
    x, w, target, gen = head_inputs(10, 60, 24, F32)
    target[3], target[6] = 60, -5
    loss, grads = run_ce(x, w, target, "none", torch.ones(10))
    bad = torch.zeros(10, dtype=torch.bool)
    bad[3] = bad[6] = True
    assert torch.equal(torch.isnan(loss.cpu()), bad)
    assert torch.equal(torch.isnan(grads[0].cpu()).all(1), bad) and torch.isnan(grads[1]).all()
    index, logits = torch.randint(0, 60, (10, 4), generator=gen), torch.zeros(10, 4)
    index[2, 1] = 1 << 40
    loss = linear_distillation(x.to(DEV), w.to(DEV), index.to(DEV), logits.to(DEV), reduction="none")
    assert torch.isnan(loss[2]) and torch.isfinite(loss[torch.arange(10) != 2]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [2, 40, 600])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_target_outside_the_vocabulary_makes_its_gradients_nan(reduction, rows, dtype):
    x, w, target, _ = head_inputs(rows, 60, 24, dtype)
    target[1] = 60
    loss, grads = run_ce(x, w, target, reduction, torch.ones(rows) if reduction == "none" else torch.tensor(1.0))
    bad = torch.arange(rows) == 1
    assert torch.equal(torch.isnan(loss.cpu()), bad) if reduction == "none" else torch.isnan(loss)
    assert torch.isnan(grads[0][1]).all() and torch.isnan(grads[1]).all()
    assert torch.isfinite(grads[0].cpu()[~bad]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 12, 600])
def test_tiny_values(rows, dtype):
    """Logits around 1e-45: q is 1 / vocab to its last bit and the loss log(vocab)."""
    x, w, target, _ = head_inputs(rows, 100, 40, dtype, seed=3)
    x, w = (x.float() * 1e-30).to(dtype), (w.float() * 1e-15).to(dtype)
    loss, grads = run_ce(x, w, target, "none", torch.ones(rows))
    # 100 exponentials and their sum to 2^-20 of them, log and the last rounding of 4.6 to 2^-21 each
    assert ((loss.cpu().double() - torch.tensor(100.0).double().log()).abs() <= 3 * 2.0 ** -20).all()
    dz = torch.full((rows, 100), 0.01, dtype=torch.float64)
    dz[torch.arange(rows), target] -= 1
    dx = dz @ w.double()
    # dz to 2^-19 (bf16: two planes or one, 2^-9), sums of 100 terms to 2^-19, the result to its type
    step = 2.0 ** -18 if dtype == F32 else 2.0 ** -8 + 2.0 ** -9 + 2.0 ** -18
    assert ((grads[0].cpu().double() - dx).abs() <= step * (dz.abs() @ w.double().abs())).all()


def test_calls_on_several_streams_at_once():
    """Workspaces of calls that run at the same time are their own."""
    jobs = []
    for i, (rows, vocab, dim, dtype) in enumerate([(700, 5000, 256, BF16), (260, 3001, 136, F32),
                                                   (1, 4096, 64, F32)]):
        x, w, target, gen = head_inputs(rows, vocab, dim, dtype, seed=30 + i)
        index = torch.randint(0, vocab, (rows, 5), generator=gen).to(DEV)
        logits = torch.randn(rows, 5, generator=gen).to(DEV)
        jobs.append((x, w, target.to(DEV), index, logits, torch.cuda.Stream()))

    def both(xd, wd, target, index, logits):
        a = linear_cross_entropy(xd, wd, target)
        b = linear_distillation(xd, wd, index, logits, 2.0)
        return [a.detach(), b.detach(), *torch.autograd.grad(a, [xd, wd]), *torch.autograd.grad(b, [xd, wd])]

    want = [both(*leaves(x, w), *rest) for x, w, *rest, _ in jobs]
    ready = [leaves(x, w) for x, w, *_ in jobs]
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(3):
        for (_, _, *rest, stream), (xd, wd), g in zip(jobs, ready, got):
            with torch.cuda.stream(stream):
                g.append(both(xd, wd, *rest))
    torch.cuda.synchronize()
    for one, g in zip(want, got):
        assert all(torch.equal(a, b) for run in g for a, b in zip(one, run))


def test_infinite_and_nan_logits_reach_the_loss():
    """A row that counts and holds inf or NaN has a NaN loss, as PyTorch's."""
    x, w, target, _ = head_inputs(6, 300, 24, F32)
    x[1, 0], x[2, 5] = float("inf"), float("nan")
    loss = linear_cross_entropy(x.to(DEV), w.to(DEV), target.to(DEV), reduction="none").cpu()
    assert torch.equal(torch.isnan(loss), torch.tensor([False, True, True, False, False, False]))


def test_large_logits_do_not_overflow():
    """Logits of +-3e4: the running maximum keeps every exponential in range."""
    x, w, target, _ = head_inputs(33, 700, 64, F32, seed=2)
    x = x * 4000
    dloss = torch.ones(33)
    loss, grads = run_ce(x, w, target, "none", dloss)
    assert torch.isfinite(loss).all() and all(torch.isfinite(gr).all() for gr in grads)
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, target[:, None])[:, 0]
    # each logit to (dim + 16) 2^-23 of its products' magnitudes
    bound = 2 * (64 + 16) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).amax(1) + 1e-6 * z.abs().amax(1)
    assert ((loss.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_and_unaligned_inputs(dtype):
    """Rows of a wider tensor, a base off 16 bytes, a transposed weight, leading dimensions."""
    x, w, target, _ = head_inputs(90, 301, 40, dtype, seed=4)
    want = run_ce(x, w, target, "mean", torch.tensor(1.0))
    wide = torch.full((90, 131), float("nan"), dtype=dtype, device=DEV)
    views = [wide[:, 8:48], wide[:, 3:43]]
    t = target.to(DEV)
    for v in views:
        wide.fill_(float("nan"))
        v.copy_(x.to(DEV))
        xs = v.detach().requires_grad_(True)
        ws = w.to(DEV).t().contiguous().t().requires_grad_(True)
        loss = linear_cross_entropy(xs, ws, t)
        gr = torch.autograd.grad(loss, [xs, ws])
        assert torch.equal(loss, want[0]) and all(torch.equal(a, b) for a, b in zip(gr, want[1]))
    xs = x.to(DEV).reshape(3, 30, 40).requires_grad_(True)
    loss = linear_cross_entropy(xs, w.to(DEV), t.reshape(3, 30).int(), reduction="none")
    assert loss.shape == (3, 30)
    assert torch.autograd.grad(loss.mean(), xs)[0].shape == (3, 30, 40)


def test_one_gradient_alone_and_none():
    x, w, target, _ = head_inputs(70, 301, 40, F32, seed=4)
    _, (dx, dw) = run_ce(x, w, target, "mean", torch.tensor(1.0))
    t = target.to(DEV)
    xd, wd = leaves(x, w)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xd, w.to(DEV), t), xd)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x.to(DEV), wd, t), wd)[0], dw)
    with torch.no_grad():
        assert not linear_cross_entropy(xd, wd, t).requires_grad
    # a weight used twice: both uses' gradients add up
    loss = linear_cross_entropy(xd, wd, t) + linear_cross_entropy(xd, wd, t)
    assert torch.allclose(torch.autograd.grad(loss, wd)[0], 2 * dw, rtol=1e-6, atol=0)


def test_results_do_not_change_from_call_to_call():
    x, w, target, _ = head_inputs(300, 5000, 256, BF16, seed=4)
    a = run_ce(x, w, target, "mean", torch.tensor(1.0))
    b = run_ce(x, w, target, "mean", torch.tensor(1.0))
    assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1], b[1]))


def test_gradient_against_differences():
    """Central differences of the kernel's own loss along a direction v: off by at most
    h^2 / 6 of the third derivative (third cumulants of a variable within a range R are below
    0.0963 R^3, R the spread of the row's logits along v) and the losses' error over h."""
    x, w, target, gen = head_inputs(64, 500, 96, F32, seed=6)
    v = torch.randn(64, 96, generator=gen)
    dv = torch.randn(500, 96, generator=gen) * 0.1
    h = 2.0 ** -6
    xd, wd, t = x.to(DEV), w.to(DEV), target.to(DEV)
    _, (dx, dw) = run_ce(x, w, target, "sum", torch.tensor(1.0))
    for step_x, step_w, slope in ((v, None, (dx.cpu().double() * v).sum()),
                                  (None, dv, (dw.cpu().double() * dv).sum())):
        vals = []
        for s in (h, -h):
            a = xd if step_x is None else xd + s * step_x.to(DEV)
            b = wd if step_w is None else wd + s * step_w.to(DEV)
            vals.append(float(linear_cross_entropy(a, b, t, reduction="none").double().sum()))
        zv = (v.double() @ w.double().t()) if step_w is None else (x.double() @ dv.double().t())
        spread = zv.amax(1) - zv.amin(1)
        ez = 112 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).amax(1)
        bound = float((h * h / 6 * 0.0963 * spread ** 3).sum() + (2 * ez + 2e-6).sum() / h)
        assert abs((vals[0] - vals[1]) / (2 * h) - float(slope)) <= bound


def test_another_stream_and_a_captured_graph():
    x, w, target, _ = head_inputs(260, 900, 128, BF16, seed=1)
    want_loss, want = run_ce(x, w, target, "mean", torch.tensor(1.0))
    xd, wd = leaves(x, w)
    t = target.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            loss = linear_cross_entropy(xd, wd, t)
            grads = torch.autograd.grad(loss, [xd, wd])
        side.synchronize()
        assert torch.equal(loss, want_loss) and all(torch.equal(a, b) for a, b in zip(grads, want))
    del loss, grads
    xd, wd = leaves(x, w)               # leaves that no eager graph has met
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = linear_cross_entropy(xd, wd, t)
            grads = torch.autograd.grad(loss, [xd, wd])
        graphs.append((graph, loss.detach(), grads))
        del loss
    with torch.no_grad():
        xd.copy_(2 * xd)
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        xd.copy_(xd / 2)
    for graph, loss, grads in graphs:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss) and all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_calls_with_left_out_rows(dtype):
    """Above 512 rows a row map and cleared results stand between the kernels of a call."""
    rows, vocab, dim = 700, 3000, 72
    x, w, target, gen = head_inputs(rows, vocab, dim, dtype, seed=5)
    target[::3] = -100
    index, logits = torch.randint(-1, vocab, (rows, 3), generator=gen), torch.randn(rows, 3, generator=gen)
    index[::4] = -1
    t, index, logits = target.to(DEV), index.to(DEV), logits.to(DEV)

    def calls(xd, wd):
        a = linear_cross_entropy(xd, wd, t, reduction="none")
        b = linear_distillation(xd, wd, index, logits, 2.0, reduction="none")
        return [a.detach(), b.detach(), *torch.autograd.grad(a.sum(), [xd, wd]),
                *torch.autograd.grad(b.sum(), [xd, wd])]

    want = calls(*leaves(x, w))
    xd, wd = leaves(x, w)               # leaves that no eager graph has met
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(xd, wd)
    for _ in range(3):
        for one in got:
            one.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_the_refs_agree_with_the_kernels():
    x, w, target, gen = head_inputs(50, 400, 64, F32, seed=9)
    index, logits = torch.randint(-1, 400, (50, 5), generator=gen), torch.randn(50, 5, generator=gen)
    a = linear_cross_entropy(x.to(DEV), w.to(DEV), target.to(DEV), impl="cuda")
    assert abs(float(a) - float(linear_cross_entropy_ref(x.double(), w.double(), target))) <= 1e-5
    b = linear_distillation(x.to(DEV), w.to(DEV), index.to(DEV), logits.to(DEV), 2.0, impl="metal")
    assert abs(float(b) - float(linear_distillation_ref(x.double(), w.double(), index, logits.double(), 2.0))) <= 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_head_and_both_losses_together(dtype):
    """The end of a training step: residual norm, then cross entropy and distillation on its
    output, gradients of both through the norm to the block's output and the head."""
    rows, vocab, dim, k = 140, 700, 96, 8
    x, w, target, gen = head_inputs(rows, vocab, dim, dtype, seed=12)
    y = (0.5 * torch.randn(rows, dim, generator=gen)).to(dtype)
    nw = (1 + 0.1 * torch.randn(dim, generator=gen)).to(dtype)
    index, logits = torch.randint(0, vocab, (rows, k), generator=gen), torch.randn(rows, k, generator=gen)
    target[3] = -100

    def step(x, y, nw, w, target, index, logits, impl):
        lv = [t.detach().requires_grad_(True) for t in (x, y, nw, w)]
        _, hidden = residual_rms_norm(lv[0], lv[1], lv[2], impl=impl)
        loss = linear_cross_entropy(hidden, lv[3], target, impl=impl) \
            + 0.5 * linear_distillation(hidden, lv[3], index, logits, 2.0, impl=impl)
        return loss, torch.autograd.grad(loss, lv)

    got = step(*(t.to(DEV) for t in (x, y, nw, w, target, index, logits)), "cuda")
    want = step(*(t.double() for t in (x, y, nw, w)), target, index, logits.double(), "torch")
    # bf16: the norm's output, each loss' dz, each loss' gradient, their sum and the norm's
    # gradient are rounded: six roundings of 2^-8; float32 as above
    tol = 6 * u(dtype) if dtype == BF16 else 2e-5
    assert abs(float(got[0].detach()) - float(want[0].detach())) <= tol * float(want[0].detach())
    for name, a, b in zip(("dx", "dy", "dnorm", "dw"), got[1], want[1]):
        check_norm(name, a, b, tol)


def test_gpu_refusals():
    x, w, target, _ = head_inputs(4, 20, 8, F32)
    xd, wd, t = x.to(DEV), w.to(DEV), target.to(DEV)
    with pytest.raises(RuntimeError, match="same CUDA"):
        linear_cross_entropy(xd, w, t)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        linear_cross_entropy(xd.half(), wd.half(), t)
    with pytest.raises(RuntimeError, match="alike"):
        linear_cross_entropy(xd, wd.bfloat16(), t)
    with pytest.raises(RuntimeError, match="integer"):
        linear_cross_entropy(xd, wd, t.float())
    with pytest.raises(ValueError, match="target"):
        linear_cross_entropy(xd, wd, t[:3])
    with pytest.raises(ValueError, match="shapes"):
        linear_cross_entropy(xd, wd[:, :5], t)
    with pytest.raises(ValueError, match="up to"):      # views: refused before anything is copied
        linear_cross_entropy(xd[:1].expand((1 << 24) + 1, 8), wd, t[:1].expand((1 << 24) + 1))
    with pytest.raises(ValueError, match="up to"):
        linear_cross_entropy(xd[:, :1], wd[:1, :1].expand((1 << 30) + 1, 1), t)
    assert linear_cross_entropy(xd[:0], wd, t[:0], reduction="none").shape == (0,)
    assert torch.isnan(linear_cross_entropy(xd[:0], wd, t[:0]))
    loss = linear_cross_entropy(xd.requires_grad_(True), wd, t)
    (dx,) = torch.autograd.grad(loss, xd, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    assert _native.device_status() == _native.MMS_OK


def test_a_wait_that_runs_out_is_reported_and_leaves_the_context_usable():
    """The products' TMA waits, made to run out by withholding one step's copies."""
    x, w, target, _ = head_inputs(300, 1000, 1024, BF16, seed=1)
    want_loss, want = run_ce(x, w, target, "mean", torch.tensor(1.0))
    lib = _native.load()
    assert lib.mms_debug_set_wait(1 << 10, 3) == _native.MMS_OK
    try:
        run_ce(x, w, target, "mean", torch.tensor(1.0))
        status = _native.device_status()
    finally:
        lib.mms_debug_set_wait(0, -1)
    assert status == _native.MMS_ERR_TIMEOUT
    loss, grads = run_ce(x, w, target, "mean", torch.tensor(1.0))
    assert _native.device_status() == _native.MMS_OK
    assert torch.equal(loss, want_loss) and all(torch.equal(a, b) for a, b in zip(grads, want))
