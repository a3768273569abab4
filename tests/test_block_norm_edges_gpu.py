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


@pytest.mark.parametrize("D", [64, 512, 63, 5001])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_what_is_not_finite_stays_in_its_row(cuda, value, dtype, rms, D):
    import mingru_b200 as mb

    g = torch.Generator(device=cuda).manual_seed(D)
    x, r, gate = (torch.randn(9, D, device=cuda, generator=g).to(dtype) for _ in range(3))
    w, b, s = (1 + torch.rand(D, device=cuda, generator=g) for _ in range(3))
    good = torch.ones(9, dtype=torch.bool, device=cuda)
    good[3] = good[8] = False
    x[3, D // 2] = r[8, -1] = value
    leaves = [t.requires_grad_(True) for t in (x, r, gate)]
    y, h = mb.block_norm(x, w, b, residual=r, scale=s, gate=gate, rms=rms)
    d = [t.detach()[good].double().requires_grad_(True) for t in leaves]
    want = norm.plain(d[0], w.double(), b.double(), d[1], s.double(), d[2], 1, 1e-5, rms)
    for n, a, e in zip("yh", (y, h), want):
        norm.close(a[good], e, norm.TOL[dtype], n)
    bad = y[~good].detach().float()
    assert bad.isnan().any(-1).all()  # at least where the value was; all of a row that has no mean
    assert rms and value == float("inf") or bad.isnan().all()
    dy = torch.randn(9, D, device=cuda, generator=g).to(dtype)
    got = torch.autograd.grad((y, h), leaves, (dy, dy))
    ref = torch.autograd.grad(want, d, (dy[good].double(), dy[good].double()))
    for n, a, e in zip(("dx", "dresidual", "dgate"), got, ref):
        norm.close(a[good], e, 3 * norm.TOL[dtype] if dtype == torch.float32 else norm.TOL[dtype], n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 2, 3, 5])
def test_rows_shorter_than_a_vector(cuda, D, dtype):
    norm.check(cuda, (37,), D, dtype, ("residual", "gate", "bias"), rms=True)


def test_rows_that_overlap(cuda):
    """Windows of one line, an element apart: rows of 9 that start everywhere."""
    import mingru_b200 as mb

    g = torch.Generator(device=cuda).manual_seed(0)
    line = torch.randn(28, device=cuda, generator=g).bfloat16()
    x = line.unfold(0, 9, 1)
    w = 1 + torch.rand(9, device=cuda, generator=g)
    xl = x.detach().requires_grad_(True)
    y = mb.block_norm(xl, w)
    d = x.double().requires_grad_(True)
    want = norm.plain(d, w.double(), None, None, None, None, 1, 1e-5, False)
    norm.close(y, want, norm.TOL[torch.bfloat16], "y")
    dy = torch.randn(20, 9, device=cuda, generator=g).bfloat16()
    got = torch.autograd.grad(y, xl, dy)[0]
    norm.close(got, torch.autograd.grad(want, d, dy.double())[0], norm.TOL[torch.bfloat16], "dx")
