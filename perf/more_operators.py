"""Convolution, scan and sampling of a served Mamba model: their cases, plain forms and exact values.

Four operators around the selective scan, in the order in which a token meets them:

  causal_conv            short depthwise causal convolution with SiLU, forward and backward
  causal_conv_packed     the same over packed prompts and single tokens, windows kept in a cache
  selective_scan_packed  the scan over packed prompts and single tokens, states kept in a cache
  sample_tokens          temperature, top-k, top-p and min-p sampling from given random numbers, and the
                         log-probability of what was drawn

`run` computes them in elementary torch operations (32 bits; 64 where a token is drawn, since a sum
next to a border decides it), or, with `own`, by the calls a user of `mamba_metal` makes. `exact`
has the definitions in 64 bits.
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

def _conv(name, batch, length, dim, taps, dtype, bias=True, silu=True):
    return {"name": name, "op": "conv", "batch": batch, "length": length, "dim": dim, "taps": taps, "dtype": dtype,
            "bias": bias, "silu": silu}


def _conv_packed(name, tokens, seqs, dim, taps, dtype, bias=True, silu=True):
    """tokens == seqs: single tokens, without a list of starts."""
    return {"name": name, "op": "conv_packed", "tokens": tokens, "seqs": seqs, "dim": dim, "taps": taps,
            "dtype": dtype, "bias": bias, "silu": silu}


def _scan(name, tokens, seqs, dim, states, dtype, gate, raw, singles=0):
    """singles: how many of the sequences are single tokens (all: without a list of starts)."""
    return {"name": name, "op": "scan_packed", "tokens": tokens, "seqs": seqs, "dim": dim, "states": states,
            "dtype": dtype, "gate": gate, "raw": raw, "singles": singles}


def _sample(name, rows, vocab, dtype, top_k, top_p, min_p, masked=0.0):
    """top_k, top_p, min_p: one value for all rows, or "mixed" for values of each row's own."""
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "masked": masked}


def listed():
    return [
        # TinyMamba's training step (batch 16 x 512, d_inner 1432, 4 taps), x a half of in_proj's output
        _conv("conv train model fp32", 16, 512, 1432, 4, "fp32"),
        # long sequences of a wide model
        _conv("conv train wide bf16", 4, 4096, 8192, 4, "bf16"),
        # one token of one answer
        _conv_packed("conv one token fp32", 1, 1, 1432, 4, "fp32"),
        # prompts of very different lengths, packed behind one another
        _conv_packed("conv prompts bf16", 8192, 37, 2304, 4, "bf16"),
        # one token of one answer
        _scan("scan one token fp32", 1, 1, 1432, 16, "fp32", True, True, 1),
        # a full batch of answers, one token each
        _scan("scan tokens fp32", 256, 256, 2304, 16, "fp32", False, False, 256),
        # packed prompts, gated
        _scan("scan prompts bf16", 8192, 16, 2304, 16, "bf16", True, False),
        # one long prompt
        _scan("scan long prompt fp32", 16384, 1, 2048, 16, "fp32", False, False),
        # answers and prompts in one call, odd sizes, many states
        _scan("scan mixed odd fp32", 3001, 70, 1433, 64, "fp32", True, True, 63),
        # one answer's next token from the model's vocabulary
        _sample("sample one row fp32", 1, 32768, "fp32", 50, 0.95, 0.0),
        # odd sizes, settings of each answer's own, a part of the vocabulary forbidden
        _sample("sample mixed odd fp32", 77, 50021, "fp32", "mixed", "mixed", "mixed", 0.3),
        # a full batch and a large vocabulary, nucleus sampling
        _sample("sample nucleus bf16", 256, 131072, "bf16", 0, 0.9, 0.0),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; about a third of the large ones round."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, n // 64 * 64 if n > 128 and rng.random() < 0.35 else n))


def draw(rng):
    op = rng.choice(["conv", "conv_packed", "scan_packed", "sample"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "sample":
        c = _sample("", _spread(rng, 1, 256), _spread(rng, 64, 131072), dtype, rng.choice([0, 1, 20, 200, "mixed"]),
                    rng.choice([1.0, 0.5, 0.95, "mixed"]), rng.choice([0.0, 0.0, 0.05, "mixed"]),
                    rng.choice([0.0, 0.0, 0.5]))
    elif op == "conv":
        dim, taps = _spread(rng, 64, 8192), rng.choice([2, 3, 4, 4, 4])
        rows = max(1, min(1 << 27, _spread(rng, dim, 1 << 27)) // dim)
        length = min(rows, _spread(rng, 1, 8192))
        c = _conv("", min(64, max(1, rows // length)), length, dim, taps, dtype, rng.random() < 0.8, rng.random() < 0.8)
    else:
        tokens = _spread(rng, 1, 16384)
        kind = rng.choice(["singles", "prompts", "mixed"])
        if kind == "singles":
            tokens = min(tokens, 512)
        seqs = tokens if kind == "singles" else min(tokens, _spread(rng, 1, 64))
        if op == "conv_packed":
            c = _conv_packed("", tokens, seqs, _spread(rng, 64, 8192), rng.choice([2, 3, 4, 4, 4]), dtype,
                             rng.random() < 0.8, rng.random() < 0.8)
        else:
            states = rng.choice([4, 8, 12, 16, 16, 16, 32, 64])
            dim = min(_spread(rng, 64, 8192), max(64, (1 << 29) // (tokens * states)))
            singles = seqs if kind == "singles" else seqs // 2 if kind == "mixed" else 0
            if tokens > seqs and singles == seqs:
                singles = 0
            c = _scan("", tokens, seqs, dim, states, dtype, rng.random() < 0.6, rng.random() < 0.5, singles)
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs

def _lengths(tokens, seqs, singles, seed):
    """seqs lengths of at least 1 that make up `tokens`: `singles` ones, the others of very different sizes."""
    g = torch.Generator().manual_seed(int(seed) + 17)
    if singles >= seqs or tokens == seqs:
        return [1] * seqs
    long = seqs - singles
    rest = tokens - seqs
    share = torch.exp(1.2 * torch.randn(long, generator=g, dtype=torch.float64))
    ends = (share.cumsum(0) / share.sum() * rest).round().long().tolist()
    lens = [1 + b - a for a, b in zip([0] + ends[:-1], ends)] + [1] * singles
    order = torch.randperm(seqs, generator=g).tolist()
    return [lens[i] for i in order]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    ty = TYPES[case["dtype"]]

    def randn(*size):
        return torch.randn(*size, generator=g, device=DEVICE)

    def rand(*size):
        return torch.rand(*size, generator=g, device=DEVICE)

    s = {"case": dict(case)}
    if case["op"] == "conv":
        b, t, d, k = case["batch"], case["length"], case["dim"], case["taps"]
        xz = randn(b, t, 2 * d).to(ty)                      # in_proj's output; its first half is convolved
        s.update(xz=xz, x=xz[..., :d].requires_grad_(True), dy=randn(b, t, d).to(ty))
        s["weight"] = (randn(d, k) / math.sqrt(k)).to(ty).requires_grad_(True)
        s["bias"] = (0.1 * randn(d)).to(ty).requires_grad_(True) if case["bias"] else None
        return s
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        z = 2.0 * randn(rows, vocab)
        lead = torch.randint(0, vocab, (rows, 4), generator=g, device=DEVICE)
        z.scatter_add_(1, lead, 10.0 * rand(rows, 4))       # some rows are sure of a few tokens, some of none
        if case["masked"]:
            gone = rand(rows, vocab) < case["masked"]
            gone[:, 0] = False
            z = z.masked_fill(gone, -math.inf)
        s["logits"] = z.to(ty)
        s["uniform"] = rand(rows)
        s["temperature"] = 0.3 + rand(rows)
        pick = torch.randint(0, 4, (rows,), generator=g, device=DEVICE)
        if case["top_k"] == "mixed":
            s["top_k"] = torch.tensor([0, 1, 40, 2000], device=DEVICE)[pick]
        else:
            s["top_k"] = case["top_k"]
        s["top_p"] = 0.3 + 0.7 * rand(rows) if case["top_p"] == "mixed" else case["top_p"]
        s["min_p"] = 0.1 * rand(rows) * (pick > 1) if case["min_p"] == "mixed" else case["min_p"]
        return s
    tokens, seqs, d = case["tokens"], case["seqs"], case["dim"]
    singles = case.get("singles", 0)
    lens = _lengths(tokens, seqs, singles, seed)
    s["lens"] = lens
    s["starts"] = None
    if tokens != seqs:
        ends = torch.tensor([0] + lens).cumsum(0)
        s["starts"] = ends.to(torch.int32).to(DEVICE)
    # the cache has a place more than two per sequence; each sequence goes on from a place of its own
    # and leaves its state in another; every fifth of several starts anew
    place = torch.randperm(2 * seqs + 1, generator=g, device=DEVICE)
    s["slots"], s["out_slots"] = place[:seqs].clone(), place[seqs:2 * seqs].clone()
    if seqs > 1:
        s["slots"][::5] = -1
    if case["op"] == "conv_packed":
        k = case["taps"]
        s["x"] = randn(tokens, 2 * d).to(ty)[:, :d]
        s["weight"] = (randn(d, k) / math.sqrt(k)).to(ty)
        s["bias"] = (0.1 * randn(d)).to(ty) if case["bias"] else None
        s["window"] = randn(2 * seqs + 1, d, k - 1).to(ty)
        return s
    n = case["states"]
    s["x"] = randn(tokens, d).to(ty)
    s["b"], s["c"] = randn(tokens, n).to(ty), randn(tokens, n).to(ty)
    steps = torch.arange(1, n + 1, device=DEVICE, dtype=torch.float32)
    if case["raw"]:
        s["dt"] = randn(tokens, d).to(ty)
        s["aneg"] = steps * (1.0 + 0.1 * rand(d, n))
        s["dt_range"] = (0.001, 0.1)
    else:
        s["dt"] = torch.log1p(torch.exp(-2.0 + 0.5 * randn(tokens, d))).to(ty)
        s["aneg"] = steps * (1.0 + 0.1 * rand(d, n))
        s["dt_range"] = None
    s["state"] = randn(2 * seqs + 1, d, n)
    s["z"] = randn(tokens, 2 * d).to(ty)[:, d:] if case["gate"] else None
    s["d_skip"] = 1.0 + 0.1 * randn(d) if case["gate"] else None
    return s


# ------------------------------------------------------------------------------- run

def run(s):
    op = s["case"]["op"]
    with torch.set_grad_enabled(bool(own and op == "conv")):
        if own:
            return {"conv": _own_conv, "conv_packed": _own_conv_packed, "scan_packed": _own_scan,
                    "sample": _own_sample}[op](s)
        return {"conv": _plain_conv, "conv_packed": _plain_conv_packed, "scan_packed": _plain_scan,
                "sample": _plain_sample}[op](s)


def _own_conv(s):
    from mamba_metal import causal_conv
    y = causal_conv(s["x"], s["weight"], s["bias"], silu=s["case"]["silu"])
    leaves = [s[n] for n in ("x", "weight", "bias") if s[n] is not None]
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(), "grads": list(grads)}


def _own_conv_packed(s):
    from mamba_metal import causal_conv_packed
    y = causal_conv_packed(s["x"], s["weight"], s["bias"], s["window"], starts=s["starts"], slots=s["slots"],
                           out_slots=s["out_slots"], silu=s["case"]["silu"])
    return {"y": y, "window": s["window"]}


def _own_scan(s):
    from mamba_metal import selective_scan_packed
    y = selective_scan_packed(s["x"], s["dt"], s["aneg"], s["b"], s["c"], s["state"], starts=s["starts"],
                              slots=s["slots"], out_slots=s["out_slots"], z=s["z"], d_skip=s["d_skip"],
                              dt_range=s["dt_range"])
    return {"y": y, "state": s["state"]}


def _own_sample(s):
    from mamba_metal import sample_tokens
    tokens, logprob = sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                    top_p=s["top_p"], min_p=s["min_p"], return_logprob=True)
    return {"tokens": tokens, "logprob": logprob}


def _plain_conv(s):
    c, ty = s["case"], s["dy"].dtype
    x, w, dy = s["x"].detach().float(), s["weight"].detach().float(), s["dy"].float()
    b, t, d, k = c["batch"], c["length"], c["dim"], c["taps"]
    pre = torch.zeros(b, t, d, device=x.device)
    if s["bias"] is not None:
        pre += s["bias"].detach().float()
    for j in range(k):                          # tap j meets the input of k - 1 - j steps before
        back = k - 1 - j
        if back < t:
            pre[:, back:] += w[:, j] * x[:, :t - back]
    if c["silu"]:
        sig = 1.0 / (1.0 + torch.exp(-pre))
        y = (pre * sig).to(ty)
        ds = dy * (sig * (1.0 + pre * (1.0 - sig)))
    else:
        y, ds = pre.to(ty), dy
    del pre
    dx = torch.zeros(b, t, d, device=x.device)
    dw = torch.zeros(d, k, device=x.device)
    for j in range(k):
        back = k - 1 - j
        if back < t:
            dx[:, :t - back] += w[:, j] * ds[:, back:]
            dw[:, j] = (ds[:, back:] * x[:, :t - back]).sum((0, 1))
    grads = [dx.to(ty), dw.to(ty)]
    if s["bias"] is not None:
        grads.append(ds.sum((0, 1)).to(ty))
    return {"y": y, "grads": grads}


def _bounds(s, rows):
    """(first row, length) of each sequence, and each row's sequence."""
    if s["starts"] is None:
        first = torch.arange(rows, device=DEVICE)
        return first, torch.ones_like(first), first
    st = s["starts"].long()
    row = torch.arange(rows, device=DEVICE)
    return st[:-1], st[1:] - st[:-1], torch.searchsorted(st, row, right=True) - 1


def _plain_conv_packed(s):
    c, ty = s["case"], s["x"].dtype
    x, w, k = s["x"].float(), s["weight"].float(), c["taps"]
    first, lens, of = _bounds(s, c["tokens"])
    slots = s["slots"]
    old = torch.where((slots >= 0)[:, None, None], s["window"][slots.clamp(min=0)].float(), torch.zeros((), device=DEVICE))
    at = torch.arange(c["tokens"], device=DEVICE) - first[of]       # a row's place in its sequence
    pre = torch.zeros_like(x)
    if s["bias"] is not None:
        pre += s["bias"].float()
    for j in range(k):
        back = k - 1 - j
        row = torch.arange(c["tokens"], device=DEVICE) - back
        inside = (at >= back)[:, None]
        before = (at - back + k - 1).clamp(0, max(0, k - 2))          # its place in the window, if it is there
        v = x[row.clamp(min=0)]
        if k > 1:
            v = torch.where(inside, v, old[of, :, before])
        pre += w[:, j] * v
    y = pre / (1.0 + torch.exp(-pre)) if c["silu"] else pre
    if k > 1:
        new = torch.empty_like(old)
        for j in range(k - 1):                  # the last k - 1 inputs, older ones from the old window
            p = lens - (k - 1) + j
            v = x[(first + p).clamp(0, c["tokens"] - 1)]
            o = old[torch.arange(len(p), device=DEVICE), :, (p + k - 1).clamp(0, k - 2)]
            new[:, :, j] = torch.where((p >= 0)[:, None], v, o)
        s["window"][s["out_slots"]] = new.to(ty)
    return {"y": y.to(ty), "window": s["window"]}


def _plain_scan(s):
    c, ty = s["case"], s["x"].dtype
    rows, d, n = c["tokens"], c["dim"], c["states"]
    x, dt, bm, cm = (s[m].float() for m in ("x", "dt", "b", "c"))
    aneg = s["aneg"]
    if s["dt_range"] is not None:
        lo, hi = s["dt_range"]
        dt = lo + (hi - lo) / (1.0 + torch.exp(-dt))
        aneg = torch.where(aneg > 20.0, aneg, torch.log1p(torch.exp(aneg)))
    first, lens, of = _bounds(s, rows)
    last = first + lens - 1
    slots, keep = s["slots"], s["slots"] >= 0
    y = torch.empty(rows, d, device=DEVICE)
    step = max(1, (1 << 26) // (rows * n))
    new = torch.empty(c["seqs"], d, n, device=DEVICE)
    for a in range(0, d, step):
        e = min(d, a + step)
        # affine maps h -> A h + H; a sequence's first forgets what lies before it in the rows
        A = torch.exp(-dt[:, a:e, None] * aneg[a:e])
        H = (dt[:, a:e] * x[:, a:e])[:, :, None] * bm[:, None, :]
        old = torch.where(keep[:, None, None], s["state"][slots.clamp(min=0), a:e], torch.zeros((), device=DEVICE))
        H[first] += A[first] * old
        A[first] = 0.0
        shift, longest = 1, max(s["lens"])
        while shift < longest:
            H[shift:] += A[shift:] * H[:-shift].clone()
            A[shift:] *= A[:-shift].clone()
            shift *= 2
        y[:, a:e] = (H * cm[:, None, :]).sum(-1)
        new[:, a:e] = H[last]
    s["state"][s["out_slots"]] = new
    if s["d_skip"] is not None:
        y += s["d_skip"]
    if s["z"] is not None:
        z = s["z"].float()
        y *= z / (1.0 + torch.exp(-z))
    return {"y": y.to(ty), "state": s["state"]}


def _column(v, rows, dtype):
    if isinstance(v, torch.Tensor):
        return v.to(dtype)[:, None]
    return torch.full((rows, 1), v, dtype=dtype, device=DEVICE)


def _plain_sample(s):
    rows, vocab = s["logits"].shape
    k = _column(s["top_k"], rows, torch.int64)
    k = torch.where(k > 0, k, vocab)
    top_p, min_p = _column(s["top_p"], rows, torch.float32).double(), _column(s["min_p"], rows, torch.float32).double()
    t = s["temperature"].double()[:, None]
    z, index = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    w = torch.exp((z.double() - z[:, :1].double()) / t)
    place = torch.arange(vocab, device=DEVICE)
    w = torch.where(place < k, w, torch.zeros_like(w))
    ahead = torch.cumsum(w, 1) - w                         # the weight of those before
    kept = (w > 0) & (w >= min_p) & ((place == 0) | (top_p >= 1.0) | (ahead < top_p * w.sum(1, keepdim=True)))
    w = torch.where(kept, w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, index, w)          # back in the order of the vocabulary
    upto = torch.cumsum(w, 1)
    past = (upto > s["uniform"].double()[:, None] * upto[:, -1:]) & (w > 0)
    token = past.int().argmax(1)
    return {"tokens": token, "logprob": torch.log(w.gather(1, token[:, None])[:, 0] / upto[:, -1]).float()}


# ------------------------------------------------------------------------ work, exact

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "conv":
        elems, d, k = case["batch"] * case["length"] * case["dim"], case["dim"], case["taps"]
        # x and dy in, y and dx out; the weights and their gradients
        return {"bytes": size * (4 * elems + 2 * d * (k + case["bias"])),
                "flops": elems * (6 * k + (20 if case["silu"] else 1))}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (size * case["vocab"] + 32), "flops": 4 * case["rows"] * case["vocab"]}
    tokens, seqs, d = case["tokens"], case["seqs"], case["dim"]
    fresh = 0 if seqs == 1 else (seqs + 4) // 5             # sequences that start anew read no state
    if case["op"] == "conv_packed":
        k = case["taps"]
        return {"bytes": size * (2 * tokens * d + (2 * seqs - fresh) * d * (k - 1) + d * (k + case["bias"])),
                "flops": tokens * d * (2 * k + (5 if case["silu"] else 0))}
    n = case["states"]
    return {"bytes": size * (tokens * d * (4 if case["gate"] else 3) + 2 * tokens * n)
            + 4 * ((2 * seqs - fresh) * d * n + d * n + (d if case["gate"] else 0)),
            "flops": tokens * d * (7 * n + 4)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"conv": _exact_conv, "conv_packed": _exact_conv_packed, "scan_packed": _exact_scan,
                "sample": _exact_sample}[case["op"]](s)


def _exact_conv(s):
    """Sequence by sequence, the taps as one matrix of shifted inputs; gradients by automatic differentiation."""
    c = s["case"]
    k, d = c["taps"], c["dim"]
    y, dx = [], []
    w = s["weight"].detach().double().requires_grad_(True)
    bias = None if s["bias"] is None else s["bias"].detach().double().requires_grad_(True)
    dw, db = torch.zeros_like(w), torch.zeros(d, dtype=torch.float64, device=w.device)
    step = max(1, 4096 * 2048 // max(1, c["length"] * d))
    for a in range(0, c["batch"], step):
        with torch.enable_grad():
            x = s["x"][a:a + step].detach().double().requires_grad_(True)
            wide = torch.cat([torch.zeros(x.shape[0], k - 1, d, dtype=x.dtype, device=x.device), x], 1)
            pre = (wide.unfold(1, k, 1) * w).sum(-1)
            if bias is not None:
                pre = pre + bias
            out = pre * torch.sigmoid(pre) if c["silu"] else pre
            got = torch.autograd.grad(out, [x, w] + ([bias] if bias is not None else []), s["dy"][a:a + step].double())
        y.append(out.detach())
        dx.append(got[0])
        dw = dw + got[1]
        if bias is not None:
            db = db + got[2]
    return {"y": torch.cat(y), "grads": [torch.cat(dx), dw.detach()] + ([db] if bias is not None else [])}


def _exact_conv_packed(s):
    """Sequence by sequence, from the window and the inputs behind it."""
    c = s["case"]
    k = c["taps"]
    x, w, window = s["x"].double(), s["weight"].double(), s["window"].double()
    y, new = torch.empty_like(x), window.clone()
    row = 0
    if c["tokens"] == c["seqs"]:                            # all of them at once
        old = torch.where((s["slots"] >= 0)[:, None, None], window[s["slots"].clamp(min=0)], torch.zeros((), dtype=torch.float64, device=DEVICE))
        wide = torch.cat([old, x[:, :, None]], 2)
        y = (wide * w).sum(-1)
        new[s["out_slots"]] = wide[:, :, 1:]
    else:
        slots, out_slots = s["slots"].tolist(), s["out_slots"].tolist()
        for i, n in enumerate(s["lens"]):
            old = window[slots[i]] if slots[i] >= 0 else torch.zeros_like(window[0])
            wide = torch.cat([old.t(), x[row:row + n]])
            y[row:row + n] = (wide.unfold(0, k, 1) * w).sum(-1)
            new[out_slots[i]] = wide[n:].t()
            row += n
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if c["silu"]:
        y = y * torch.sigmoid(y)
    return {"y": y, "window": new}


def _exact_scan(s):
    """The recurrence step by step, for all sequences that are that long."""
    c = s["case"]
    x, dt, bm, cm, aneg = (s[m].double() for m in ("x", "dt", "b", "c", "aneg"))
    if s["dt_range"] is not None:
        lo, hi = s["dt_range"]
        dt = lo + (hi - lo) * torch.sigmoid(dt)
        aneg = torch.nn.functional.softplus(aneg)
    lens = s["lens"]
    first = [sum(lens[:i]) for i in range(len(lens))]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    at = torch.tensor([first[i] for i in order], device=DEVICE)
    slots, out_slots = s["slots"][torch.tensor(order, device=DEVICE)], s["out_slots"][torch.tensor(order, device=DEVICE)]
    state = s["state"].double()
    h = torch.where((slots >= 0)[:, None, None], state[slots.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=DEVICE))
    y = torch.empty_like(x)
    count = len(lens)
    for t in range(lens[order[0]]):
        while lens[order[count - 1]] <= t:
            count -= 1
        r = at[:count] + t
        g = h[:count]
        g *= torch.exp(-dt[r][:, :, None] * aneg)
        g += (dt[r] * x[r])[:, :, None] * bm[r][:, None, :]
        y[r] = torch.matmul(g, cm[r][:, :, None])[:, :, 0]
    state = state.clone()
    state[out_slots] = h
    if s["d_skip"] is not None:
        y = y + s["d_skip"].double()
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    return {"y": y, "state": state}


def _exact_sample(s):
    """Row by row: cut the ranked list to k, to the mass p, to the share min_p of the first; then draw."""
    rows, vocab = s["logits"].shape

    def value(v, i):
        return v[i].item() if isinstance(v, torch.Tensor) else torch.tensor(float(v), dtype=torch.float32).item()

    out, logprob = [], []
    for i in range(rows):
        z = s["logits"][i].double()
        k = int(s["top_k"][i].item() if isinstance(s["top_k"], torch.Tensor) else s["top_k"]) or vocab
        rank = torch.argsort(-z, stable=True)[:k]
        p = torch.softmax(z[rank] / s["temperature"][i].double(), 0)
        keep = p > 0
        top_p = value(s["top_p"], i)
        if top_p < 1.0:
            before = torch.cat([torch.zeros_like(p[:1]), p.cumsum(0)[:-1]])
            keep &= before < top_p
            keep[0] = True
        keep &= p >= value(s["min_p"], i) * p[0]
        rank, p = rank[keep], p[keep]
        order = torch.argsort(rank)
        upto = p[order].cumsum(0)
        j = int((upto <= s["uniform"][i].double() * upto[-1]).sum())
        j = min(j, len(rank) - 1)
        out.append(int(rank[order][j]))
        logprob.append(float(torch.log(p[order][j]) - torch.log(p.sum())))
    return {"tokens": torch.tensor(out, device=DEVICE), "logprob": torch.tensor(logprob, dtype=torch.float64, device=DEVICE)}
