"""linear_attention and block_norm as compilers and other tracers see them: fake CUDA tensors, no GPU."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import ShapeEnv


@pytest.fixture
def fake():
    import mingru_b200  # noqa: F401  (registers the ops)

    with FakeTensorMode(shape_env=ShapeEnv()) as mode:
        yield mode


def _cuda(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_strides_that_the_fakes_give(fake):
    """Outputs as the op allocates them: in the input's order where its rows are dense, else contiguous."""
    ops = torch.ops.mingru_b200
    Q = _cuda(2, 150, 3, 32).transpose(1, 2)
    K = _cuda(2, 3, 32, 150).transpose(2, 3)  # copied by the op: rows are not dense
    V = torch.as_strided(_cuda(2000), (2, 3, 150, 40), (0, 500, 1, 1))  # windows
    lg = _cuda(2, 3, 150)
    y, H, saved = ops.linear_attn_fwd(Q, K, V, lg, None, True)
    dQ, dK, dV, dlg, dH0 = ops.linear_attn_bwd(Q, K, V, lg, saved, y, None, True)
    assert dQ.stride() == (150 * 96, 32, 96, 1)
    assert dK.stride() == (450 * 32, 150 * 32, 32, 1)
    assert y.stride() == dV.stride() and y.stride(-1) == 1
    assert H.stride() == dH0.stride() == (3 * 32 * 40, 32 * 40, 40, 1) and dlg.stride() == (450, 150, 1)
