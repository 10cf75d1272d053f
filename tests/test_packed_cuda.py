"""The packed scan's kernels against float64, within the bounds of tests/_serve_ref.py."""
from __future__ import annotations

import pytest
import torch

from _serve_ref import close, scan_bound
from mamba_metal import gated_output, selective_scan, selective_scan_packed, selective_scan_step
from mamba_metal.packed import places_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def make(rows, d, n, dtype, seed=0, places=9, raw=False, slow=1.0):
    g = torch.Generator().manual_seed(seed)
    x, z = (torch.randn(rows, d, generator=g).to(dtype) for _ in range(2))
    dt = torch.randn(rows, d, generator=g)
    dt = (dt if raw else slow * torch.nn.functional.softplus(0.5 * dt - 2)).to(dtype)
    b, c = (torch.randn(rows, n, generator=g).to(dtype) for _ in range(2))
    aneg = torch.arange(1, n + 1) * (1 + 0.1 * torch.rand(d, n, generator=g))
    return dict(x=x, dt=dt, aneg=aneg, b_in=b, c_in=c, state=torch.randn(places, d, n, generator=g), z=z,
                d_skip=1 + 0.1 * torch.randn(d, generator=g), dt_range=(0.001, 0.1) if raw else None)


def run(t, starts, slots, out_slots, ints=torch.int32):
    on = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in t.items()}
    on["state"] = t["state"].clone().to(DEV)
    lists = [None if v is None else torch.as_tensor(v).to(ints).to(DEV) for v in (starts, slots, out_slots)]
    y = selective_scan_packed(starts=lists[0], slots=lists[1], out_slots=lists[2], **on)
    return y, on["state"]


def check(t, starts, slots, out_slots, ints=torch.int32):
    y, state = run(t, starts, slots, out_slots, ints)
    tensors = [None if v is None else torch.as_tensor(v) for v in (starts, slots, out_slots)]
    seqs = places_of(t["x"].shape[0], *tensors, t["state"].shape[0])
    wy, by, ws, bs = scan_bound(t["x"], t["dt"], t["aneg"], t["b_in"], t["c_in"], t["state"], seqs, t["z"], t["d_skip"],
                                t["dt_range"], t["x"].dtype)
    covered = torch.zeros(t["x"].shape[0], dtype=torch.bool)
    for first, end, _, _ in seqs:
        covered[first:end] = True
    assert (y.cpu()[~covered] == 0).all()
    close(y[covered.to(DEV)], wy[covered], by[covered], "y")
    close(state, ws, bs, "state")
    written = {dst for *_, dst in seqs if dst is not None}
    keep = [p for p in range(t["state"].shape[0]) if p not in written]
    assert torch.equal(state[keep].cpu(), t["state"][keep])
    return y, state


@pytest.mark.parametrize("dtype,raw", [(F32, False), (F32, True), (BF16, False), (BF16, True)])
@pytest.mark.parametrize("d,n", [(1, 4), (33, 8), (128, 16), (130, 12), (40, 20), (64, 32), (31, 48), (70, 64)])
def test_packed_matches_float64(d, n, dtype, raw):
    """Lengths around the tile of 8 and the segment of 64 rows, empty ones, rows of nobody."""
    for i, lens in enumerate(([1], [8], [9, 0, 1], [64, 65, 63], [200], [3, 129, 0, 1, 1, 70])):
        lead, tail = i % 3, (i + 1) % 3
        t = make(lead + sum(lens) + tail, d, n, dtype, seed=i + d, raw=raw, slow=0.1 if i % 2 else 1.0)
        if i % 2:
            t["z"], t["d_skip"] = (None, t["d_skip"]) if i % 4 == 1 else (t["z"], None)
        starts = torch.tensor([lead] + lens).cumsum(0)
        perm = torch.randperm(9, generator=torch.Generator().manual_seed(i)).tolist()
        slots, out = perm[:len(lens)], perm[-len(lens):] if len(lens) < 5 else perm[:len(lens)]
        if len(lens) == 3:
            slots = [-1, perm[0], perm[0]]                 # one from nothing, two from the same place
            out = perm[3:5] + [9]                          # the last leaves nothing
        check(t, starts, slots, out, torch.int64 if i % 2 else torch.int32)


@pytest.mark.parametrize("dtype,raw", [(F32, False), (BF16, True)])
@pytest.mark.parametrize("count,d,n", [(1, 1, 4), (1, 1432, 16), (3, 33, 64), (9, 130, 8), (9, 64, 12), (200, 300, 16), (150, 2000, 16), (70, 1000, 64)])
def test_single_tokens_match_float64(count, d, n, dtype, raw):
    t = make(count, d, n, dtype, seed=count, places=count + 3, raw=raw)
    check(t, None, None, None)
    slots = torch.randperm(count + 3, generator=torch.Generator().manual_seed(1))[:count]
    out = slots.flip(0) if count > 3 else slots
    t["z"] = None
    if count == 9:
        slots = slots.clone()
        slots[2], out = -1, torch.where(torch.arange(9) == 4, -1, slots)
        t["b_in"], t["c_in"] = t["b_in"].float(), t["c_in"].float()
    elif count > 3:
        out = slots
    check(t, None, slots, out, torch.int64)


def test_long_prompts_join_many_segments():
    """dt so small that a state survives all of them."""
    for d, n, rows in ((256, 16, 5000), (64, 64, 2500)):
        t = make(rows, d, n, F32, slow=0.002)
        check(t, [0, rows], [2], [2])
        check(t, [0, 700, 701, rows], [2, 0, 1], [2, 0, 1])


def test_agrees_with_the_scan_and_the_step():
    t = make(300, 64, 16, F32, seed=5)
    t.update(z=None, d_skip=None)
    on = {k: v.to(DEV) for k, v in t.items() if torch.is_tensor(v)}
    want, h = selective_scan(*(on[k][None] if k not in ("aneg",) else on[k] for k in ("x", "dt", "aneg", "b_in", "c_in")),
                             impl="cuda", return_state=True)
    y, state = run(t, [0, 300], [-1], [3])
    assert torch.allclose(y, want[0], rtol=1e-5, atol=1e-5) and torch.allclose(state[3], h[0], rtol=1e-5, atol=1e-5)
    h = on["state"][:5].clone()
    one = {k: (v if k in ("aneg", "state") else v[:5]) if torch.is_tensor(v) else v for k, v in t.items()}
    want = selective_scan_step(on["x"][:5], on["dt"][:5], on["aneg"], on["b_in"][:5], on["c_in"][:5], h)
    y, state = run(one, None, None, None)
    assert torch.allclose(y, want, rtol=1e-6, atol=1e-6) and torch.allclose(state[:5], h, rtol=1e-6, atol=1e-6)
    gate = dict(t, z=torch.randn(300, 64), d_skip=torch.randn(64))
    y, _ = run(gate, [0, 300], [-1], [3])
    plain, _ = run(t, [0, 300], [-1], [3])
    assert torch.allclose(y, gated_output(plain[None], gate["z"][None].to(DEV), gate["d_skip"].to(DEV))[0], rtol=1e-5, atol=1e-5)


def test_pieces_of_a_prompt_are_the_prompt():
    t = make(400, 40, 16, F32, seed=6)
    whole, last = run(t, [0, 400], [-1], [3])
    state = t["state"].clone()
    got, at = [], 0
    for i, n in enumerate((1, 1, 2, 100, 296)):
        piece = {k: (v if k in ("aneg", "d_skip", "state") else v[at:at + n]) if torch.is_tensor(v) else v for k, v in t.items()}
        y, new = run(dict(piece, state=state), [0, n] if n > 1 else None, [-1 if i == 0 else 3], [3])
        state = new.cpu()
        got.append(y)
        at += n
    assert torch.allclose(torch.cat(got), whole, rtol=1e-5, atol=1e-5) and torch.allclose(state[3], last[3].cpu(), rtol=1e-5, atol=1e-5)


def test_strided_rows_and_unaligned_bases():
    for rows, starts in ((90, [0, 90]), (4, None)):
        t = make(rows, 40, 16, BF16, seed=7)
        want, state = run(t, starts, None, None)
        for key, off in (("x", 3), ("dt", 1), ("z", 40), ("b_in", 2), ("c_in", 8)):
            v = t[key]
            wide = torch.full((rows, 97), float("nan"), dtype=BF16)
            wide[:, off:off + v.shape[1]] = v
            on = dict(t)
            on[key] = wide.to(DEV)[:, off:off + v.shape[1]]
            y, s = run(on, starts, None, None)
            assert torch.equal(y, want) and torch.equal(s, state), key
        y, _ = run(dict(t, x=t["x"].t().contiguous().to(DEV).t()), starts, None, None)
        assert torch.equal(y, want)


def test_infinite_steps_forget_and_nan_stays_with_its_sequence():
    t = make(30, 8, 16, F32, seed=8)
    t["x"][12, 3] = float("nan")
    y, state = run(t, [0, 10, 20, 30], [0, 1, 2], [0, 1, 2])
    good = torch.ones(30, 8, dtype=torch.bool)
    good[12:20, 3] = False
    assert torch.isfinite(y.cpu()[good]).all() and torch.isnan(y.cpu()[~good]).all()
    assert torch.isnan(state[1, 3]).all() and torch.isfinite(state[[0, 2]]).all()
    t = make(10, 8, 16, F32, seed=9)
    t["dt"][4] = 1e30                                      # decay 0: the state before is gone
    t["x"][4] = 0
    y, _ = run(t, [0, 10], [0], [0])
    z, _ = run(dict(t, state=torch.randn(9, 8, 16)), [0, 10], [0], [0])
    assert torch.equal(y[4:], z[4:]) and not torch.equal(y[:4], z[:4])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_enters_a_segment_far_from_its_start(dtype):
    """NaN and infinite states reach every later row; negative steps bring decayed states back."""
    rows = 400
    t = make(rows, 8, 16, dtype, seed=12)
    t["dt"] = torch.full_like(t["dt"], 4.0)                # nothing is left of a state after a few rows
    t["x"][3, 2], t["x"][5, 4] = float("nan"), float("inf")
    y, state = run(t, [0, rows], [0], [0])
    assert torch.isnan(y[3:, 2]).all() and torch.isnan(state[0, 2]).all() and not torch.isfinite(y[5:, 4]).any()
    keep = [c for c in range(8) if c not in (2, 4)]
    assert torch.isfinite(y[:, keep]).all() and torch.isfinite(state[:, keep]).all()
    for slow in (False, True):
        t = make(rows, 8, 16, dtype, seed=13)
        t["dt"] = torch.full((rows, 8), 1.0).to(dtype)
        t["dt"][65:130:2] = -1.0 if not slow else 0.0
        t["dt"][130:190] = -0.5 if not slow else 0.0
        t["aneg"] = t["aneg"] * (0.1 if not slow else -0.002)      # slow: states that grow
        check(t, [0, rows], [0], [0])


def test_lists_that_break_the_rules_stay_inside_the_arrays():
    t = make(300, 40, 16, F32, places=5)
    guard = torch.full((7, 40, 16), 7.0, device=DEV)
    on = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in t.items()}
    for starts in ([200, 3, 9, 300], [-5, 2, 1 << 40, 4], [1 << 33, -(1 << 50), 7, 7], [0, 500, 600, 700]):
        guard[1:6] = t["state"].to(DEV)
        y = selective_scan_packed(**{**on, "state": guard[1:6]}, starts=torch.tensor(starts, device=DEV),
                                  slots=torch.tensor([0, 1 << 40, -3], device=DEV), out_slots=torch.tensor([1, 3, 1 << 35], device=DEV))
        torch.cuda.synchronize()
        assert y.shape == (300, 40) and (guard[0] == 7).all() and (guard[6] == 7).all()


def test_same_result_every_time_on_streams_and_in_a_graph_with_other_lists():
    t = make(700, 300, 16, BF16, seed=10)
    on = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in t.items()}
    old = on["state"].clone()
    starts, slots = torch.tensor([0, 1, 2, 400, 700], device=DEV), torch.tensor([0, 1, 2, 3], device=DEV)

    def call(state):
        return selective_scan_packed(**{**on, "state": state}, starts=starts, slots=slots)

    states = [old.clone() for _ in range(4)]
    want = call(states[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s, st in zip(streams, states[1:]):
        with torch.cuda.stream(s):
            got.append(call(st))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got) and all(torch.equal(s, states[0]) for s in states)
    graph = torch.cuda.CUDAGraph()
    state = old.clone()
    with torch.cuda.graph(graph):
        out = call(state)
    for lists in ([0, 100, 300, 301, 650], [0, 0, 0, 700, 700]):
        starts.copy_(torch.tensor(lists, device=DEV))
        state.copy_(old)
        graph.replay()
        again = old.clone()
        assert torch.equal(out, call(again)) and torch.equal(state, again)


def test_refused_on_cuda():
    t = make(6, 8, 16, F32)
    on = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in t.items()}
    starts = torch.tensor([0, 2, 6], device=DEV)

    def call(**kw):
        return selective_scan_packed(**{**on, "starts": starts, **kw})

    call()
    for kw in (dict(x=on["x"].half()), dict(dt=on["dt"].bfloat16()), dict(z=on["z"].double()), dict(state=t["state"]),
               dict(starts=starts.cpu()), dict(b_in=on["b_in"].long()), dict(slots=torch.tensor([0, 1]))):
        with pytest.raises(RuntimeError):
            call(**kw)
    for kw in (dict(state=on["state"].bfloat16()), dict(state=on["state"].transpose(0, 1).contiguous().transpose(0, 1)),
               dict(aneg=on["aneg"][:, :6], b_in=on["b_in"][:, :6], c_in=on["c_in"][:, :6], state=on["state"][:, :, :6].contiguous())):
        with pytest.raises(ValueError):
            call(**kw)
    assert call(x=on["x"][:0], dt=on["dt"][:0], b_in=on["b_in"][:0], c_in=on["c_in"][:0], z=on["z"][:0],
                starts=starts * 0).shape == (0, 8)


@pytest.mark.parametrize("dtype,raw", [(F32, False), (F32, True), (BF16, True)])
@pytest.mark.parametrize("d,n", [(40, 4), (33, 16), (24, 28), (17, 64)])
@pytest.mark.parametrize("singles", [3, 150])
def test_a_long_prompt_among_single_tokens(singles, d, n, dtype, raw):
    """More segments than a segment chains by itself, beside fewer or more sequences than segments; the
    short ones have 1, 2, 3 and no rows."""
    lens = [(1, 2, 3, 0)[i % 4] for i in range(singles)] + [1600] + [(2, 1, 300)[i % 3] for i in range(singles)]
    starts = torch.tensor([5] + lens).cumsum(0)
    places = len(lens)
    slots = torch.randperm(places, generator=torch.Generator().manual_seed(1))
    slots[::7] = -1
    t = make(int(starts[-1]) + 3, d, n, dtype, places=places, raw=raw, slow=0.01)
    check(t, starts, slots, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sequences_of_whole_segments(dtype):
    """Lengths at and beside multiples of a segment (32 rows here), few and many of them, and a captured call
    replayed with other starts."""
    lens = [32, 64, 31, 33, 128, 1, 160, 0, 1600, 96, 65]
    starts = torch.tensor([0] + lens).cumsum(0)
    slots = torch.tensor([3, 1, -1, 0, 10, 9, 2, 4, 5, 6, 7])
    rows = int(starts[-1])
    t = make(rows, 64, 16, dtype, places=11, slow=0.02)
    check(t, starts, slots, None)
    check(t, torch.tensor([0, 32 * 68, rows]), torch.tensor([3, -1]), torch.tensor([3, 2]))
    check(t, torch.tensor([0] * 5 + [rows] * 7), slots, None)
    on = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in t.items()}
    lists = [starts.to(DEV), slots.to(DEV)]
    on["state"] = t["state"].clone().to(DEV)
    call = lambda: selective_scan_packed(starts=lists[0], slots=lists[1], **on)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    other = torch.tensor([0, 700, 700, 701, 760, 1000, 1032, 1064, 1500, 1501, 1502, rows])
    lists[0].copy_(other)
    on["state"].copy_(t["state"])
    graph.replay()
    got, state = y.clone(), on["state"].clone()
    want, want_state = run(t, other, slots, None)
    assert torch.equal(got, want) and torch.equal(state, want_state)
