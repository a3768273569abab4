"""linear_attention, its step and block_norm on tensors that lie in uncommon ways, against float64:
tolerances and plain forms are those of the operators' own test files."""

from __future__ import annotations

import pytest
import test_block_norm_gpu as norm
import test_linear_attn_gpu as attn
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 63])
@pytest.mark.parametrize("tokens", [1, 3])
def test_norm_of_the_first_tokens(cuda, tokens, D, dtype):
    """A dimension of size 1 before the tokens: its stride is not the tokens' extent."""

    def view(a):  # (B, 1, tokens, D), tokens of five
        wide = torch.full((a.shape[0], 1, 5, D), 7.0, dtype=a.dtype, device=a.device)
        return wide[:, :, :tokens].copy_(a)

    norm.check(cuda, (6, 1, tokens), D, dtype, ("residual", "gate", "bias"), view=view)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,strides", [
    ((1, 1, 8, 64), (0, 0, 1, 1)),  # windows a token apart, fewer than channels
    ((1, 1, 150, 64), (0, 0, 1, 1)),
    ((1, 1, 300, 64), (0, 0, 8, 1)),
    ((2, 3, 20, 48), (2000, 1, 48, 1)),  # heads that overlap
    ((3, 2, 20, 72), (1, 2000, 72, 1)),
    ((2, 2, 40, 32), (3000, 1300, 1, 40)),  # channels before time
])
def test_attention_on_overlapping_views(cuda, shape, strides, dtype):
    import mingru_b200 as mb

    B, H, T, d = shape
    g = torch.Generator(device=cuda).manual_seed(T + d)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g)  # noqa: E731
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    view = lambda scale=1.0: (scale * r(size)).to(dtype).as_strided(shape, strides)  # noqa: E731
    Q, K, V, dy = view(d**-0.5), view(d**-0.5), view(), view()
    lg = -torch.nn.functional.softplus(r(B, H, T) - 3)
    H0, dH = r(B, H, d, d), r(B, H, d, d)
    own = [t.detach().requires_grad_(True) for t in (Q, K, V, lg, H0)]
    ref = [t.detach().double().requires_grad_(True) for t in (Q, K, V, lg, H0)]
    y, HT = mb.linear_attention(*own)
    ry, rH = attn.recurrence(*ref)
    tol, f32 = attn.TOL[dtype], attn.TOL[torch.float32]
    attn.close(y, ry, tol, "y")
    attn.close(HT, rH, f32, "H_T")
    got = torch.autograd.grad((y, HT), own, (dy, dH))
    want = torch.autograd.grad((ry, rH), ref, (dy.double(), dH.double()))
    mb.raise_device_error(cuda)
    for n, a, b, t in zip(("dQ", "dK", "dV", "dlg", "dH0"), got, want, (tol, tol, tol, attn.DLG, f32)):
        attn.close(a, b, t, n)
