"""The packed scan's ends joined beside as many sequences as there are segments, or more."""
from __future__ import annotations

import pytest
import torch

from test_packed_cuda import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,raw", [(torch.float32, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("d,n", [(40, 4), (33, 16), (17, 64)])
@pytest.mark.parametrize("prompts,singles", [((2400,), 100), ((2400,), 300), ((33, 1600, 500), 150), ((700, 0, 1500), 2300)])
def test_prompts_beside_more_single_tokens(prompts, singles, d, n, dtype, raw):
    """Segments of 32 rows: 70 to 150 of them, a decay that lets a state survive them all. Then the same
    rows as sequences of one segment each, where the launch finds nothing to join."""
    half = singles // 2
    lens = [1] * half + list(prompts) + [1] * (singles - half)
    starts = torch.tensor([3] + lens).cumsum(0)
    rows = int(starts[-1]) + 2
    slots = torch.randperm(len(lens) + 4, generator=torch.Generator().manual_seed(1))[:len(lens)]
    slots[::9] = -1
    t = make(rows, d, n, dtype, seed=singles, places=len(lens) + 4, raw=raw, slow=0.01)
    check(t, starts, slots, None)
    check(t, torch.arange(0, rows, 16)[:len(lens) + 1], slots[:len(range(0, rows, 16)[:len(lens) + 1]) - 1], None)
