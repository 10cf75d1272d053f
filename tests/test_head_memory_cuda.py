"""Peak memory of the head's losses: no logits beside them.

torch.cuda.max_memory_allocated above what is held before the call. A call allocates its gradients,
the float32 loss, what the forward keeps, and one direction's workspace at a time, each asked for
here; the allocator rounds each of the (fewer than ten) blocks up to 2 MB at most.
"""
from __future__ import annotations

import pytest
import torch

from mamba_metal import MambaConfig, TinyMamba, _native, linear_cross_entropy, linear_distillation

pytestmark = pytest.mark.gpu
MB = 1 << 20


def peak_of(step):
    step()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = step()
    torch.cuda.synchronize()
    del out
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("kd", [False, True])
@pytest.mark.parametrize("rows,vocab,dim,dtype", [(8192, 32768, 640, torch.float32), (8192, 131072, 256, torch.bfloat16),
                                                  (4096, 50021, 771, torch.bfloat16)])
def test_a_loss_and_its_gradients(rows, vocab, dim, dtype, kd):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype).requires_grad_(True)
    w = (0.05 * torch.randn(vocab, dim, generator=gen, device="cuda")).to(dtype).requires_grad_(True)
    k = 16 if kd else 0
    index = torch.randint(0, vocab, (rows, max(k, 1)), generator=gen, device="cuda")
    logits = torch.randn(rows, max(k, 1), generator=gen, device="cuda")

    def step():
        loss = linear_distillation(x, w, index, logits, 2.0) if kd else linear_cross_entropy(x, w, index[:, 0])
        return torch.autograd.grad(loss, [x, w])

    lib, bf16 = _native.load(), int(dtype == torch.bfloat16)
    ws = [lib.mms_head_workspace_size(rows, vocab, dim, k, bf16, dim, dim, back) for back in (0, 1)]
    kept, grads = lib.mms_head_kept_size(rows, k), (rows + vocab) * dim * x.element_size()
    peak = peak_of(step)
    assert peak <= kept + max(ws[0], ws[1] + grads) + rows * 8 + 20 * MB
    # without the logits (float32, as the plain form has them): less than one copy of them
    assert peak - grads < rows * vocab * 4


def test_a_fused_training_step():
    """Beside the blocks' activations the plain step holds the logits, their log-softmax and its gradient
    at once; the fused one's workspace is no larger than one of them (mms_head_workspace_size)."""
    kw = dict(vocab_size=32768, d_model=128, n_layers=1, d_ff=256, d_state=8, scan_impl="cuda")
    idx = torch.randint(0, 32768, (16, 513), generator=torch.Generator().manual_seed(2)).cuda()
    logits = 16 * 512 * 32768 * 4

    def peak(**flags):
        model = TinyMamba(MambaConfig(**kw, **flags)).cuda()

        def step():
            model.zero_grad(set_to_none=True)
            model(idx[:, :-1], idx[:, 1:])[1].backward()

        return peak_of(step)

    plain, fused = peak(), peak(fuse_norm=True, fuse_loss=True)
    print(f"peak above the model, MB: plain {plain / MB:.0f}, fused {fused / MB:.0f}")
    assert fused <= plain - logits
