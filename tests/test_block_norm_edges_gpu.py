"""block_norm where fp32 overflows, and on infinities and NaN: what 1 / sqrt(mean of squares) gives, row by
row. A row's values never reach another row's, so the others are compared with the plain form in float64 at
the tolerance of the operator's own tests."""

from __future__ import annotations

import pytest
import test_block_norm_gpu as norm
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 512, 4096, 63, 5001])  # vectors, several to a thread, odd rows, elements
@pytest.mark.parametrize("rms", [False, True])
def test_squares_beyond_fp32(cuda, rms, D):
    """The sum of squares overflows: 1 / sqrt(inf) = 0, rows of zeros (the bias) and no gradient for them."""
    import mingru_b200 as mb

    g = torch.Generator(device=cuda).manual_seed(D)
    x = torch.randn(6, D, device=cuda, generator=g)
    big = torch.tensor([0, 1, 0, 0, 1, 0], dtype=torch.bool, device=cuda)
    x[big] *= 1e25
    w, b = 1 + torch.rand(D, device=cuda, generator=g), torch.rand(D, device=cuda, generator=g)
    xl = x.clone().requires_grad_(True)
    y = mb.block_norm(xl, w, b, rms=rms)
    assert torch.equal(y[big], b.expand(2, D))
    want = norm.plain(x[~big].double(), w.double(), b.double(), None, None, None, 1, 1e-5, rms)
    norm.close(y[~big], want, norm.TOL[torch.float32], "y")
    dx = torch.autograd.grad(y.sum(), xl)[0]
    assert not dx[big].any() and torch.isfinite(dx).all()
