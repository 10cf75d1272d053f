"""TinyMamba.serve and generate: packed prompts and single tokens against the whole sequences."""
from __future__ import annotations

import pytest
import torch

from mamba_metal import MambaConfig, TinyMamba, sample_tokens

LENS = (5, 1, 12, 3)


def model(**kw):
    torch.manual_seed(0)
    m = TinyMamba(MambaConfig(**{**dict(vocab_size=60, d_model=24, n_layers=2, d_ff=48, d_state=8), **kw}))
    with torch.no_grad():
        for b in m.blocks:                                # biases and skips that matter
            b.conv.bias.normal_()
            b.D_skip.normal_()
    return m


def prompts(vocab=60, lens=LENS):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, vocab, (n,), generator=g) for n in lens]


def whole(m, seq):
    with torch.no_grad():
        return m(seq[None])[0][0, -1]


def run(m, device, tol):
    """Prompts in two calls (the second with single tokens among them), in places out of order, then
    a token each: the logits of the whole sequences every time."""
    ps = [p.to(device) for p in prompts()]
    cache = m.new_cache(6)
    slots = torch.tensor([4, 0, 5, 2], device=device)
    none = torch.full((4,), -1, device=device)
    first = [p[:max(1, len(p) // 2)] for p in ps]
    starts = torch.tensor([0] + [len(p) for p in first], device=device).cumsum(0)
    got = m.serve(torch.cat(first), cache, starts, none, slots)
    for i in range(4):
        assert torch.allclose(got[i], whole(m, first[i]), rtol=tol, atol=tol)
    rest = [p[len(f):] for p, f in zip(ps, first)]
    going = [i for i in range(4) if len(rest[i])]
    starts = torch.tensor([0] + [len(rest[i]) for i in going], device=device, dtype=torch.int32).cumsum(0)
    got = m.serve(torch.cat([rest[i] for i in going]), cache, starts, slots[going])
    for row, i in enumerate(going):
        assert torch.allclose(got[row], whole(m, ps[i]), rtol=tol, atol=tol)
    token = torch.tensor([7, 8, 9, 10], device=device)
    # two answers go on from one place, each into its own
    src, dst = slots[[0, 1, 2, 2]], torch.tensor([4, 0, 1, 3], device=device)
    got = m.serve(token, cache, None, src, dst)
    for i, p in enumerate((ps[0], ps[1], ps[2], ps[2])):
        assert torch.allclose(got[i], whole(m, torch.cat([p, token[i:i + 1]])), rtol=tol, atol=tol)


def check_generate(m, device, **kw):
    """Each token is the one that sample_tokens draws from the logits of the sequence so far."""
    ps, n = [p.to(device) for p in prompts()], 6
    u = torch.rand(n, 4, generator=torch.Generator().manual_seed(2)).to(device)
    out = m.generate(ps, n, uniform=u, **kw)
    assert out.shape == (4, n) and out.dtype == torch.int64
    cache = m.new_cache(4)
    idx, starts = torch.cat(ps), torch.tensor([0, *LENS], device=device).cumsum(0)
    for i in range(n):
        logits = m.serve(idx, cache, starts if i == 0 else None)
        for s, p in enumerate(ps):
            assert torch.allclose(logits[s], whole(m, torch.cat([p, out[s, :i]])), rtol=1e-4, atol=1e-4)
        idx = sample_tokens(logits, u[i], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
        assert torch.equal(idx, out[:, i])


@pytest.mark.parametrize("fuse_norm", [False, True])
def test_serve_on_the_cpu(fuse_norm):
    run(model(fuse_norm=fuse_norm), "cpu", 1e-5)
    check_generate(model(fuse_norm=fuse_norm), "cpu", temperature=0.8, top_k=20, top_p=0.9)


def test_generate_refuses_and_repeats():
    m = model()
    for bad in ([], [torch.zeros(0, dtype=torch.int64)]):
        with pytest.raises(ValueError, match="at least one token"):
            m.generate(bad, 2)
    with pytest.raises(ValueError, match="uniform"):
        m.generate(prompts(), 2, uniform=torch.rand(4, 2))
    a = m.generate(prompts(), 5, generator=torch.Generator().manual_seed(3))
    assert torch.equal(a, m.generate(prompts(), 5, generator=torch.Generator().manual_seed(3)))
    assert m.generate(prompts(), 0).shape == (4, 0)
    assert torch.equal(m.generate(torch.stack([prompts()[0]] * 2), 3, temperature=0.0)[0], m.generate(prompts()[:1], 3, top_k=1)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(fuse_norm=True, fuse_conv=True, fuse_loss=True), dict(d_conv=2, d_state=20, d_inner=33),
                                dict(scan_impl="torch")])
def test_serve_and_generate_on_the_gpu(kw):
    m = model(**kw).cuda()
    run(m, "cuda", 2e-4)
    check_generate(m, "cuda", temperature=0.8, top_k=20, top_p=0.9)
    check_generate(m, "cuda", top_p=0.7, min_p=0.02)


@pytest.mark.gpu
def test_a_captured_step_of_serving():
    """One token of every answer, drawn and handed to the next step: captured once, replayed."""
    m = model(fuse_norm=True).cuda()
    ps = [p.cuda() for p in prompts()]
    n = 8
    u = torch.rand(n, 4, generator=torch.Generator().manual_seed(5)).cuda()
    want = m.generate(ps, n, top_k=10, uniform=u)
    cache = m.new_cache(4)
    starts = torch.tensor([0, *LENS], device="cuda").cumsum(0)
    token = sample_tokens(m.serve(torch.cat(ps), cache, starts), u[0], top_k=10)
    got, now = [token.clone()], torch.empty(4, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                         # (cuBLAS and the allocator warm up)
        warm = {"blocks": [{k: v.clone() for k, v in b.items()} for b in cache["blocks"]]}
        sample_tokens(m.serve(token, warm), now, top_k=10)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    keep = {"blocks": [{k: v.clone() for k, v in b.items()} for b in cache["blocks"]]}
    with torch.cuda.graph(graph):
        token.copy_(sample_tokens(m.serve(token, cache), now, top_k=10))
    for b, k in zip(cache["blocks"], keep["blocks"]):
        for name in k:
            b[name].copy_(k[name])
    for i in range(1, n):
        now.copy_(u[i])
        graph.replay()
        got.append(token.clone())
    assert torch.equal(torch.stack(got, 1), want)


@pytest.mark.gpu
def test_fused_convolution_trains_and_decodes_like_the_layers():
    base, fused = model().cuda(), model(fuse_conv=True).cuda()
    fused.load_state_dict(base.state_dict())
    idx = torch.randint(0, 60, (3, 40), generator=torch.Generator().manual_seed(4)).cuda()
    grads = []
    for m in (base, fused):
        _, loss = m(idx[:, :-1], idx[:, 1:])
        loss.backward()
        grads.append([loss.detach(), *(p.grad for p in m.parameters())])
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-5)
    with torch.no_grad():
        caches = [{}, {}]
        logits = [m(idx[:, :8], cache=c)[0] for m, c in zip((base, fused), caches)]
        for t in range(8, 14):
            assert torch.allclose(logits[0], logits[1], rtol=1e-4, atol=1e-4)
            logits = [m(idx[:, t:t + 1], cache=c)[0] for m, c in zip((base, fused), caches)]
    # with gradients the one-token step stays differentiable, its window untouched
    window = caches[1]["blocks"][0]["conv"]
    before = window.clone()
    out = fused(idx[:, :1], cache=caches[1])[0]
    assert torch.equal(window, before)
    out.sum().backward()
