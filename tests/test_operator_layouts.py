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


def _attention_views():
    """(1, 1, T, d) views and what is to be dense of them: the last dimension, for every output."""
    line = torch.zeros(937)
    yield line.as_strided((1, 1, 8, 64), (937, 937, 1, 1))  # sliding windows: time is as dense
    yield line.as_strided((1, 4, 8, 64), (937, 1, 64, 1))  # heads that overlap
    yield line.as_strided((4, 1, 8, 64), (1, 937, 64, 1))
    yield torch.zeros(2, 3, 64, 8).transpose(2, 3)
    yield torch.zeros(2, 8, 3, 64).transpose(1, 2)
    yield torch.zeros(2, 1, 8, 64).expand(2, 3, 8, 64)
    yield torch.zeros(2, 3, 8, 1).expand(2, 3, 8, 64)
    yield torch.zeros(2, 3, 8, 65)[..., 1:]
    yield torch.zeros(1, 1, 1, 64)
    yield torch.zeros(3, 8, 2, 1).permute(2, 0, 1, 3)


def _one_place_each(t):
    """Every element in a place of its own, rows dense: what a kernel writes row by row."""
    places = torch.zeros(t.shape, dtype=torch.int64)
    for n, s, d in zip(t.shape, t.stride(), range(t.dim())):
        places += (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
    return places.unique().numel() == t.numel() and (t.stride(-1) == 1 or t.shape[-1] == 1)


@pytest.mark.parametrize("x", list(_attention_views()), ids=lambda x: f"{tuple(x.shape)}-{x.stride()}")
def test_outputs_of_attention_are_dense_rows(x, monkeypatch):
    """The C entry takes no stride of the last dimension: outputs have 1 there, whatever the inputs' order."""
    import contextlib

    from mingru_b200 import attn_ops

    class Library:
        mgs_linear_attn_fwd = mgs_linear_attn_bwd = staticmethod(lambda *a: 0)

    monkeypatch.setattr(attn_ops._lib, "load", lambda: Library)
    monkeypatch.setattr(attn_ops, "_sizes", lambda *a: (0, 0))
    monkeypatch.setattr(attn_ops, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(attn_ops, "raw_stream", lambda d: 0)
    lg = torch.zeros(x.shape[:3])
    y, HT, saved = attn_ops._forward(x, x, x, lg, None, True)
    assert _one_place_each(y) and _one_place_each(HT)
    for g in attn_ops._gradients(x, x, x, lg, saved, y, None, True):
        assert _one_place_each(g)


def test_step_reads_no_state_that_it_is_writing(monkeypatch):
    """A buffer that lies over a part of H_prev: the kernel gets a copy; in place it gets the one buffer."""
    from mingru_b200 import step_ops

    got = []
    monkeypatch.setattr(step_ops, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(step_ops._lib, "load", lambda: type("L", (), {"mgs_linear_attn_step": None}))
    monkeypatch.setattr(step_ops, "_run", lambda op, fn, dev, *a: got.append((a[6], a[8])))
    q, lg = torch.zeros(2, 3, 4), torch.zeros(2, 3)
    n = 2 * 3 * 4 * 4
    line = torch.zeros(2 * n)
    state = lambda i: line[i:i + n].view(2, 3, 4, 4)  # noqa: E731
    for prev, out in ((state(0), state(16)), (state(16), state(0)), (state(1), state(0)), (state(0), state(n - 1))):
        step_ops.linear_attention_step(q, q, q, lg, prev, out=out)
        a, b = got.pop()
        assert b == out.data_ptr() and abs(a - b) >= 4 * n
    for prev, out in ((state(0), state(0)), (state(0), state(n)), (state(n), state(0))):
        step_ops.linear_attention_step(q, q, q, lg, prev, out=out)
        assert got.pop() == (prev.data_ptr(), out.data_ptr())
