"""The head's losses and the residual norm: their cases, plain forms and exact values.

Three operators that follow one another in a training step of a language model:

  linear_cross_entropy   softmax cross entropy of x W^T, without keeping the logits
  linear_distillation    KL divergence from a teacher's top k logits, through the same product
  residual_rms_norm      the residual sum after a block and the norm before the next one

`run` computes them in elementary torch operations in 32 bits, or, with `own`, by the calls a user
of `mamba_metal` makes. `exact` has the definitions in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "mamba-metal-scan_b200")     # where mamba_metal lies
if _PACKAGE not in sys.path:
    sys.path.append(_PACKAGE)

DEVICE = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ----------------------------------------------------------------------------- cases

def _ce(name, rows, vocab, dim, dtype, reduction, train, ignored=0.0):
    return {"name": name, "op": "cross_entropy", "rows": rows, "vocab": vocab, "dim": dim, "dtype": dtype,
            "reduction": reduction, "train": train, "ignored": ignored}


def _kd(name, rows, vocab, dim, dtype, k, tau, train, padded=0.0):
    return {"name": name, "op": "distillation", "rows": rows, "vocab": vocab, "dim": dim, "dtype": dtype,
            "k": k, "tau": tau, "train": train, "padded": padded}


def _norm(name, rows, dim, dtype, post, gate, scale, train):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "post": post, "gate": gate,
            "scale": scale, "train": train}


def listed():
    return [
        # TinyMamba's training step (vocabulary 32768, d_model 640, batch 16 x 512, fp32)
        _ce("ce train model fp32", 8192, 32768, 640, "fp32", "mean", True),
        # a large vocabulary and a wide model in bf16: the step that logits would not fit beside
        _ce("ce train large bf16", 8192, 131072, 2048, "bf16", "mean", True),
        # a padded batch of odd sizes, weighted row by row by the caller
        _ce("ce train odd bf16", 1000, 50021, 1001, "bf16", "none", True, 0.3),
        # the log-probability of one next token while serving
        _ce("ce score one token fp32", 1, 32768, 640, "fp32", "none", False),
        # scoring of a short answer
        _ce("ce score answer bf16", 77, 50021, 1000, "bf16", "none", False, 0.1),
        # distillation into the model of the first case
        _kd("kd train model fp32", 4096, 32768, 640, "fp32", 32, 2.0, True),
        # distillation at a wide model, top 64
        _kd("kd train large bf16", 8192, 65536, 2048, "bf16", 64, 1.0, True),
        # evaluation of a few rows, short lists with empty places
        _kd("kd score odd bf16", 130, 32001, 771, "bf16", 7, 3.0, False, 0.4),
        # one decode token between two blocks
        _norm("norm decode fp32", 1, 640, "fp32", False, False, False, False),
        # the model's training step: residual sum and norm
        _norm("norm train model fp32", 8192, 640, "fp32", False, False, False, True),
        # a wide block with a norm behind it, its gate and its scale
        _norm("norm train full bf16", 16384, 4096, "bf16", True, True, True, True),
        # odd sizes, gated, without the norm behind the block
        _norm("norm train odd bf16", 777, 1433, "bf16", False, True, True, True),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; about a third of the large ones round."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, n // 64 * 64 if n > 128 and rng.random() < 0.35 else n))


def draw(rng):
    op = rng.choice(["cross_entropy", "distillation", "norm"])
    dtype = rng.choice(["fp32", "bf16"])
    train = rng.random() < 0.65
    if op == "norm":
        c = _norm("", _spread(rng, 1, 16384), _spread(rng, 64, 4096), dtype, rng.random() < 0.5, rng.random() < 0.5,
                  rng.random() < 0.5, train)
        if dtype == "fp32":
            c["rows"] = min(c["rows"], 8192)
    else:
        rows, vocab, dim = _spread(rng, 1, 8192), _spread(rng, 64, 65536), _spread(rng, 64, 2048)
        if op == "cross_entropy":
            c = _ce("", rows, vocab, dim, dtype, rng.choice(["mean", "sum", "none"]), train,
                    rng.choice([0.0, 0.0, 0.2]) if rows > 8 else 0.0)
        else:
            c = _kd("", rows, vocab, dim, dtype, min(_spread(rng, 1, 64), vocab), rng.choice([1.0, 1.5, 2.0, 4.0]),
                    train, rng.choice([0.0, 0.0, 0.3]) if rows > 8 else 0.0)
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    ty = TYPES[case["dtype"]]
    rows, dim = case["rows"], case["dim"]

    def randn(*size):
        return torch.randn(*size, generator=g, device=DEVICE)

    if case["op"] == "norm":
        s = {"x": (2.0 * randn(rows, dim)).to(ty), "y": (0.7 * randn(rows, dim)).to(ty),
             "weight": (1.0 + 0.1 * randn(dim)).to(ty), "post": None, "gate": None, "scale": None}
        if case["post"]:
            s["post"] = (1.0 + 0.1 * randn(dim)).to(ty)
        if case["gate"]:            # the second half of one projection's output, as in the model's block
            s["gate"] = (1.5 * randn(rows, 2 * dim)).to(ty)[:, dim:]
        if case["scale"]:
            s["scale"] = (0.5 + 0.1 * randn(dim)).to(ty)
        if case["train"]:
            s["dh"], s["du"] = randn(rows, dim).to(ty), randn(rows, dim).to(ty)
        names = ("x", "y", "weight", "post", "gate", "scale")
    else:
        vocab = case["vocab"]
        # logits of standard deviation 2 beside a target's, which leads by 0 to 16 as in a trained model
        w = randn(vocab, dim) * (2.0 / math.sqrt(dim))
        target = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
        x = randn(rows, dim) + 4.0 * torch.rand(rows, 1, generator=g, device=DEVICE) * w[target]
        s = {"x": x.to(ty), "weight": w.to(ty)}
        if case["op"] == "cross_entropy":
            if case["ignored"]:
                target = torch.where(torch.rand(rows, generator=g, device=DEVICE) < case["ignored"],
                                     torch.full_like(target, -100), target)
                target[0] = 0
            s["target"] = target
            if case["train"] and case["reduction"] == "none":
                s["dloss"] = torch.rand(rows, generator=g, device=DEVICE) / rows
        else:
            k = case["k"]
            # k different indices: a start, then steps that stay within the vocabulary
            step = torch.randint(1, max(1, vocab // k) + 1, (rows, k), generator=g, device=DEVICE)
            index = (target[:, None] + step.cumsum(1) - step[:, :1]) % vocab
            logits = 2.0 * randn(rows, k)
            logits[:, 0] += 6.0
            if case["padded"]:
                gone = torch.rand(rows, k, generator=g, device=DEVICE) < case["padded"]
                gone[0] = False
                index = torch.where(gone, torch.full_like(index, -1), index)
            s["index"], s["logits"] = index, logits
        names = ("x", "weight")
    s["case"] = dict(case)
    s["leaves"] = [n for n in names if s[n] is not None]
    if case["train"]:
        for n in s["leaves"]:
            s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------- run

def run(s):
    op = s["case"]["op"]
    with torch.set_grad_enabled(bool(own and s["case"]["train"])):
        if own:
            return {"cross_entropy": _own_ce, "distillation": _own_kd, "norm": _own_norm}[op](s)
        return {"cross_entropy": _plain_ce, "distillation": _plain_kd, "norm": _plain_norm}[op](s)


def _own_ce(s):
    from mamba_metal import linear_cross_entropy
    loss = linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=-100, reduction=s["case"]["reduction"])
    if not s["case"]["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, [s["x"], s["weight"]], s.get("dloss"))
    return {"loss": loss.detach(), "dx": dx, "dweight": dw}


def _own_kd(s):
    from mamba_metal import linear_distillation
    loss = linear_distillation(s["x"], s["weight"], s["index"], s["logits"], temperature=s["case"]["tau"])
    if not s["case"]["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, [s["x"], s["weight"]])
    return {"loss": loss.detach(), "dx": dx, "dweight": dw}


def _own_norm(s):
    from mamba_metal import residual_rms_norm
    h, u = residual_rms_norm(s["x"], s["y"], s["weight"], post_weight=s["post"], gate=s["gate"], scale=s["scale"])
    out = {"h": h.detach(), "u": u.detach()}
    if s["case"]["train"]:
        grads = torch.autograd.grad([h, u], [s[n] for n in s["leaves"]], [s["dh"], s["du"]])
        out.update({"d" + n: g for n, g in zip(s["leaves"], grads)})
    return out


def _softmax_parts(z):
    """(exp(z - max), its row sums, log sum exp) over the last dimension."""
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    return e, total, (top + torch.log(total)).squeeze(1)


def _plain_ce(s):
    c, x, w, t = s["case"], s["x"].float(), s["weight"].float(), s["target"]
    valid = t != -100
    at = torch.where(valid, t, torch.zeros_like(t))[:, None]
    z = x @ w.t()
    e, total, lse = _softmax_parts(z)
    rows = torch.where(valid, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    count = valid.sum()
    loss = rows if c["reduction"] == "none" else rows.sum() / (count if c["reduction"] == "mean" else 1)
    if not c["train"]:
        return {"loss": loss}
    weight = s["dloss"] if c["reduction"] == "none" else 1.0 / count if c["reduction"] == "mean" else 1.0
    weight = (weight * valid)[:, None]
    del z
    g = e.div_(total)
    g.scatter_add_(1, at, torch.full_like(at, -1, dtype=g.dtype))
    g.mul_(weight)
    return {"loss": loss, "dx": (g @ w).to(s["x"].dtype), "dweight": (g.t() @ x).to(s["weight"].dtype)}


def _plain_kd(s):
    c, x, w, index, tau = s["case"], s["x"].float(), s["weight"].float(), s["index"], s["case"]["tau"]
    valid = index >= 0
    at = torch.where(valid, index, torch.zeros_like(index))
    some = valid.any(1)
    t = torch.where(valid, s["logits"] / tau, torch.full_like(s["logits"], -math.inf))
    t = torch.where(some[:, None], t, torch.zeros_like(t))
    e, total, lse = _softmax_parts(t)
    keep = valid & some[:, None]
    p = torch.where(keep, e / total, torch.zeros_like(e))
    log_p = torch.where(keep, t - lse[:, None], torch.zeros_like(t))
    z = x @ w.t()
    z /= tau
    e, total, lse = _softmax_parts(z)
    rows = tau * tau * (p * (log_p - (z.gather(1, at) - lse[:, None]))).sum(1)
    count = some.sum()
    loss = rows.sum() / count
    if not c["train"]:
        return {"loss": loss}
    del z
    g = e.div_(total / some[:, None])
    g.scatter_add_(1, at, -p)
    g *= tau / count
    return {"loss": loss, "dx": (g @ w).to(s["x"].dtype), "dweight": (g.t() @ x).to(s["weight"].dtype)}


def _plain_norm(s, eps=1e-6):
    ty = s["x"].dtype
    x, y, w = s["x"].float(), s["y"].float(), s["weight"].float()
    gate, post, scale = (None if s[n] is None else s[n].float() for n in ("gate", "post", "scale"))
    sig = None if gate is None else 1.0 / (1.0 + torch.exp(-gate))
    a = y if gate is None else y * (gate * sig)
    r1 = None if post is None else 1.0 / torch.sqrt((a * a).mean(1, keepdim=True) + eps)
    b = a if post is None else a * r1 * post
    h = x + (b if scale is None else scale * b)
    r2 = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    n = h * r2
    out = {"h": h.to(ty), "u": (n * w).to(ty)}
    if not s["case"]["train"]:
        return out
    du = s["du"].float()
    t = du * w
    dh = s["dh"].float() + r2 * (t - n * (t * n).mean(1, keepdim=True))
    out["dx"], out["dweight"] = dh.to(ty), (du * n).sum(0).to(ty)
    db = dh
    if scale is not None:
        out["dscale"] = (dh * b).sum(0).to(ty)
        db = dh * scale
    da = db
    if post is not None:
        an = a * r1
        out["dpost"] = (db * an).sum(0).to(ty)
        t = db * post
        da = r1 * (t - an * (t * an).mean(1, keepdim=True))
    if gate is not None:
        out["dgate"] = (da * y * (sig * (1.0 + gate * (1.0 - sig)))).to(ty)
        da = da * (gate * sig)
    out["dy"] = da.to(ty)
    return out


# ------------------------------------------------------------------------ work, exact

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    rows, dim, train = case["rows"], case["dim"], case["train"]
    if case["op"] == "norm":
        arrays = 4 + (1 if case["gate"] else 0)                     # x, y, gate in; h, u out
        vectors = 1 + case["post"] + case["scale"]
        if train:
            arrays += 4 + (1 if case["gate"] else 0)                # dh, du in; dx, dy, dgate out
            vectors *= 2
        return {"bytes": size * dim * (rows * arrays + vectors), "flops": rows * dim * (30 if train else 10)}
    vocab = case["vocab"]
    lists = 8 * rows if case["op"] == "cross_entropy" else 12 * rows * case["k"]
    once = size * dim * (rows + vocab)
    return {"bytes": once * (2 if train else 1) + lists + 4 * rows,
            "flops": 2 * rows * vocab * dim * (3 if train else 1)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s)
        return _exact_head(s)


def _exact_head(s):
    """Both losses as sparse targets: row m has the weights p_mj at index_mj, and its own entropy term."""
    c, x, w = s["case"], s["x"].detach().double(), s["weight"].detach().double()
    rows, vocab = c["rows"], c["vocab"]
    if c["op"] == "cross_entropy":
        tau = 1.0
        valid = (s["target"] >= 0)[:, None]
        index, p = s["target"].clamp(min=0)[:, None], valid.double()
        own_term = torch.zeros(rows, dtype=torch.float64, device=x.device)
    else:
        tau = c["tau"]
        valid = s["index"] >= 0
        index = s["index"].clamp(min=0)
        t = (s["logits"].double() / tau).masked_fill(~valid, -1e300)
        p = torch.softmax(t, 1) * valid
        own_term = torch.where(p > 0, p * torch.log(p.clamp(min=1e-300)), torch.zeros_like(p)).sum(1)
    some = valid.any(1)
    count = some.sum().double()
    reduction = c.get("reduction", "mean")
    per_row = {"mean": 1.0 / count, "sum": torch.ones_like(count), "none": s.get("dloss")}[reduction]
    if per_row is None:
        per_row = torch.ones_like(count)
    per_row = per_row.double().expand(rows) * some
    loss = torch.empty(rows, dtype=torch.float64, device=x.device)
    dx, dw = torch.empty_like(x), torch.zeros_like(w)
    step = max(1, (1 << 28) // vocab)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        z = torch.mm(x[a:b], w.t()) / tau
        lse = torch.logsumexp(z, 1)
        loss[a:b] = tau * tau * (own_term[a:b] - (p[a:b] * (z.gather(1, index[a:b]) - lse[:, None])).sum(1))
        if c["train"]:
            z = torch.exp(z - lse[:, None]) * p[a:b].sum(1, keepdim=True)
            z.scatter_add_(1, index[a:b], -p[a:b])
            z *= (tau * per_row[a:b])[:, None]
            dx[a:b] = torch.mm(z, w)
            dw += torch.mm(z.t(), x[a:b])
        del z
    loss = torch.where(some, loss, torch.zeros_like(loss))
    out = {"loss": loss if reduction == "none" else loss.sum() / (count if reduction == "mean" else 1.0)}
    if c["train"]:
        out.update(dx=dx, dweight=dw)
    return out


def _exact_norm(s, eps=1e-6):
    """The definition, and its gradient by automatic differentiation, in 64 bits."""
    leaf = {n: s[n].detach().double().requires_grad_(True) for n in s["leaves"]}
    with torch.enable_grad():
        b = leaf["y"]
        if "gate" in leaf:
            b = b * leaf["gate"] * torch.sigmoid(leaf["gate"])
        if "post" in leaf:
            b = leaf["post"] * b * torch.rsqrt(b.pow(2).mean(1, keepdim=True) + eps)
        if "scale" in leaf:
            b = leaf["scale"] * b
        h = leaf["x"] + b
        u = leaf["weight"] * h * torch.rsqrt(h.pow(2).mean(1, keepdim=True) + eps)
        out = {"h": h.detach(), "u": u.detach()}
        if s["case"]["train"]:
            grads = torch.autograd.grad([h, u], [leaf[n] for n in s["leaves"]], [s["dh"].double(), s["du"].double()])
            out.update({"d" + n: g for n, g in zip(s["leaves"], grads)})
    return out
