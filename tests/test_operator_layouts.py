"""How linear_attention, its step and block_norm read and allocate tensors, without a GPU."""

from __future__ import annotations

import pytest
import torch


def _views():
    """(B, ..., D) views with leading dimensions of size 1, whose strides say nothing."""
    yield torch.arange(2 * 5 * 3.0).view(2, 1, 5, 3)[:, :, :2]  # a prefix of every sequence
    yield torch.arange(2 * 5 * 3.0).view(2, 1, 5, 3)[:, :, :1]  # its first token
    yield torch.arange(6 * 8.0).view(1, 6, 1, 8).permute(1, 2, 0, 3)[..., :4]
    yield torch.arange(4 * 6 * 5.0).view(4, 6, 5)[:, 2:3]
    yield torch.arange(4 * 6 * 5.0).view(4, 6, 5)[:1, :4, 1:4]
    yield torch.arange(3 * 2 * 4 * 5.0).view(3, 2, 4, 5).transpose(1, 2)
    yield torch.arange(7.0).expand(2, 1, 3, 7)
    yield torch.arange(40.0)[::2]
    yield torch.arange(12.0).view(3, 4)[:, 1:2]
    yield torch.zeros(0, 4, 6)[:, :2]


@pytest.mark.parametrize("x", list(_views()), ids=lambda x: f"{tuple(x.shape)}-{x.stride()}")
def test_rows_of_a_norm(x):
    """The tensor and row stride that the norm's kernels read hold x's rows, and nothing outside its storage."""
    from mingru_b200.norm_ops import _rows

    D = x.shape[-1]
    t, ld = _rows(x, D)
    rows = x.numel() // D
    end = t.storage_offset() + (rows - 1) * ld + D
    assert rows == 0 or end <= t.untyped_storage().nbytes() // t.element_size()
    assert t.stride(-1) == 1 or D == 1 or rows == 0
    assert torch.equal(torch.as_strided(t, (rows, D), (ld, 1)), x.reshape(rows, D))


def test_rows_are_read_in_place():
    """One stride from row to row needs no copy, whatever the strides of dimensions of size 1."""
    from mingru_b200.norm_ops import _rows

    for x, ld in ((torch.zeros(4, 6, 5)[:, 2:3], 30), (torch.zeros(2, 1, 5, 3)[:, :, :1], 15),
                  (torch.zeros(4, 6, 8)[..., 1:5], 8)):
        t, got = _rows(x, x.shape[-1])
        assert t is x and got == ld
