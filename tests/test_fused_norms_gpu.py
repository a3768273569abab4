"""fused_norms and RetentionMinGRU under autocast on the GPU, against the modules without them.

Tolerance: activations pass through bf16 (2^-9 a rounding) in both, and the two differ where a sum is rounded
once or twice; outputs are LayerNorms, of size one, over two layers of three such roundings: 2^-6."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _near(a, b):
    assert a.dtype == b.dtype and a.shape == b.shape
    assert ((a - b).double().norm() <= 2.0**-6 * b.double().norm()).item()


def test_retention_under_autocast(cuda):
    import mingru_b200 as mb

    torch.manual_seed(0)
    mod = mb.RetentionMinGRU(24, 64, n_heads=2).to(cuda)
    x = torch.randn(2, 150, 24, device=cuda, requires_grad=True)
    want, S = mod(x, return_state=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got, S16 = mod(x, return_state=True)
        assert got.dtype == torch.bfloat16 and S16.dtype == torch.float32
        _near(got.float(), want)
        with torch.no_grad():
            out, _ = mod.step(x[:, 0])
            _near(out.float(), want[:, 0])
        g = torch.autograd.grad(got.float().sum(), x)[0]
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("mixer", ["log", "signed", "retention"])
@pytest.mark.parametrize("width", [32, 20])
def test_stack_under_autocast(cuda, mixer, width):
    """The stream is 32 bits where there is no input projection (width = d_model), 16 where there is."""
    import mingru_b200 as mb

    torch.manual_seed(1)
    a = mb.MinGRUStack(width, 32, 2, mixer=mixer).to(cuda)
    b = mb.MinGRUStack(width, 32, 2, mixer=mixer, fused_norms=True).to(cuda)
    b.load_state_dict(a.state_dict())
    x = torch.randn(2, 40, width, device=cuda)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        ya, sa = a(x)
        yb, sb = b(x)
        _near(yb, ya)
        for u, v in zip(sb, sa):
            _near(u, v)
        block = a.blocks[0]
        h = torch.randn(2, 40, 32, device=cuda)
        want = block(h)
        block.fused_norms = True
        for u, v in zip(block(h), want):
            _near(u, v)
