"""What the head's losses ask for beside their inputs: bounded in the vocabulary, linear in the rows;
and what they say of an array that is not aligned."""
from __future__ import annotations

import pytest

from mamba_metal import _native

MB = 1 << 20


def test_the_misaligned_status_names_the_heads_arrays():
    text = _native.status_string(_native.MMS_ERR_MISALIGNED)
    assert all(word in text for word in ("x, w, kept, dx, dw", "Aneg", "workspace"))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows", [257, 8192, 1 << 16, 1 << 17, 1 << 20, 1 << 22])
def test_dz_stays_within_its_bound(rows, dtype):
    """dz's piece takes 512 MB, or up to 2 GB for 4096 entries; of the rest x is staged twice (two planes
    each of float32), dx has float32 sums, each row some numbers, and split sums take up to 74 MB, w's
    piece its rows."""
    lib, dim, vocab = _native.load(), 64, 131072
    planes = 2 - dtype
    total = lib.mms_head_workspace_size(rows, vocab, dim, 0, dtype, dim, dim, 1)
    rest = rows * dim * (2 * 2 * planes + 4) + 16 * rows + vocab * dim * 2 * planes + 80 * MB
    per_entry = rows * 2 * planes
    dz = max(512 * MB, min(2048 * MB, 4096 * per_entry), 256 * per_entry)
    assert 0 < total <= dz + rest
    # the logits of a large batch are never asked for
    if rows >= 1 << 16:
        assert total < rows * vocab * 2 / 2


@pytest.mark.parametrize("dtype", [0, 1])
def test_wide_rows_of_w(dtype):
    """A staged piece of w is bounded in the same way: 2^20 columns, 4 MB a float32 row."""
    lib, dim, rows, vocab = _native.load(), 1 << 20, 300, 50000
    total = lib.mms_head_workspace_size(rows, vocab, dim, 0, dtype, dim, dim, 1)
    assert 0 < total <= 2048 * MB + rows * dim * (2 * 2 * (2 - dtype) + 4) + 512 * MB + 256 * MB
