"""RetentionMinGRU, and a stack of it with fused norms: linear_attention,
linear_attention_step and block_norm as a model runs them.

* The mixer against its recurrence in float64 torch (outputs, final state,
  gradients of every parameter and of x), with and without time decay and a
  state handed in; fp32, rtol 1e-4 / atol 1e-4 as for the other mixers' modules
  (the projections are fp32 GEMMs of up to 64 terms).
* step() over the tokens gives forward()'s outputs.
* fused_norms changes no weights and, to fp32 rounding over the layers, no
  outputs: 1e-4.
* A stack trains: bf16 loss falls."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

TOL = dict(rtol=1e-4, atol=1e-4)


def plain(mod, x, h0, dt):
    """The mixer in float64, token by token; ``mod`` is a double copy."""
    B, T, _ = x.shape
    H, dk, dv = mod.n_heads, mod.d_k, mod.d_v
    q = mod.linear_q(x).view(B, T, H, dk) * dk**-0.5
    k = F.normalize(mod.linear_k(x).view(B, T, H, dk), dim=-1)
    z = torch.sigmoid(mod.linear_z(x))
    v = mod.linear_v(x).view(B, T, H, dv)
    S = torch.zeros(B, H, dk, dv, dtype=x.dtype, device=x.device) if h0 is None else h0.view(B, H, dk, dv)
    ys = []
    for t in range(T):
        keep = 1 - z[:, t]
        if dt is not None:
            keep = keep * torch.exp(-mod._decay_lambda() * dt[:, t, None])
        S = keep[..., None, None] * S + z[:, t, :, None, None] * k[:, t, :, :, None] * v[:, t, :, None, :]
        ys.append((q[:, t, :, None, :] @ S).squeeze(-2))
    y = torch.stack(ys, 1)
    y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    gate = mod.linear_g(x)
    y = y.reshape(B, T, H * dv) * mod.norm_weight * gate * torch.sigmoid(gate)
    return mod.out_proj(y), S.reshape(B, 1, -1)


@pytest.mark.parametrize("kw", [dict(), dict(n_heads=2, d_k=24, d_v=40), dict(decay="fixed"),
                                dict(decay="learnable", n_heads=8)])
@pytest.mark.parametrize("with_state", [False, True])
def test_mixer(cuda, kw, with_state):
    import copy

    import mingru_b200 as mb

    torch.manual_seed(0)
    mod = mb.RetentionMinGRU(48, 64, **kw).to(cuda)
    ref = copy.deepcopy(mod).double()
    B, T = 3, 150
    x = torch.randn(B, T, 48, device=cuda, requires_grad=True)
    xd = x.detach().double().requires_grad_(True)
    dt = torch.rand(B, T, device=cuda) if "decay" in kw else None
    h0 = 0.3 * torch.randn(B, 1, mod.n_heads * mod.d_k * mod.d_v, device=cuda) if with_state else None
    y, S = mod(x, h0, dt, return_state=True)
    yr, Sr = plain(ref, xd, None if h0 is None else h0.double(), None if dt is None else dt.double())
    torch.testing.assert_close(y.double(), yr, **TOL)
    torch.testing.assert_close(S.double(), Sr, **TOL)
    w, ws = torch.randn_like(y) / T, torch.randn_like(S) / T
    got = torch.autograd.grad((y * w).sum() + (S * ws).sum(), [x, *mod.parameters()])
    want = torch.autograd.grad((yr * w.double()).sum() + (Sr * ws.double()).sum(), [xd, *ref.parameters()])
    mb.raise_device_error(cuda)
    for n, a, b in zip(["x", *dict(mod.named_parameters())], got, want):
        torch.testing.assert_close(a.double(), b, msg=n, **TOL)


@pytest.mark.parametrize("fused", [False, True])
def test_steps_are_forward(cuda, fused):
    import mingru_b200 as mb

    torch.manual_seed(1)
    mod = mb.MinGRUStack(20, 64, 2, mixer="retention", mixer_kwargs=dict(n_heads=4), fused_norms=fused).to(cuda).eval()
    x = torch.randn(2, 40, 20, device=cuda)
    with torch.no_grad():
        y, last = mod(x)
        state, ys = mod.init_state(), []
        for t in range(x.shape[1]):
            out, state = mod.step(x[:, t], state)
            ys.append(out)
    torch.testing.assert_close(torch.stack(ys, 1), y, **TOL)
    for a, b in zip(state, last):
        torch.testing.assert_close(a.view(-1), b.view(-1), **TOL)


@pytest.mark.parametrize("mixer", ["log", "delta", "retention", ["retention", "log", "signed"]])
@pytest.mark.parametrize("mlp", [0, 2])
def test_fused_norms(cuda, mixer, mlp):
    import mingru_b200 as mb

    torch.manual_seed(2)
    a = mb.MinGRUStack(16, 32, 3, mlp_expansion=mlp, mixer=mixer).to(cuda)
    b = mb.MinGRUStack(16, 32, 3, mlp_expansion=mlp, mixer=mixer, fused_norms=True).to(cuda)
    b.load_state_dict(a.state_dict())
    x = torch.randn(2, 33, 16, device=cuda)
    ya, sa = a(x)
    yb, sb = b(x)
    torch.testing.assert_close(yb, ya, **TOL)
    for u, v in zip(sa, sb):
        torch.testing.assert_close(v, u, **TOL)
    w = torch.randn_like(ya) / 33
    for (n, u), v in zip(a.named_parameters(), b.parameters()):
        gu = torch.autograd.grad((ya * w).sum(), u, retain_graph=True)[0]
        gv = torch.autograd.grad((yb * w).sum(), v, retain_graph=True)[0]
        torch.testing.assert_close(gv, gu, msg=n, **TOL)


def test_stack_trains_in_bf16(cuda):
    import mingru_b200 as mb

    torch.manual_seed(3)
    mod = mb.MinGRUStack(32, 128, 2, mixer="retention", mixer_kwargs=dict(n_heads=2), fused_norms=True)
    mod = mod.to(cuda).bfloat16()
    opt = torch.optim.SGD(mod.parameters(), lr=0.5)
    x = torch.randn(4, 300, 32, device=cuda).bfloat16()
    target = torch.roll(x, 1, 1).repeat(1, 1, 4)  # the token before
    losses = []
    for _ in range(20):
        y, state = mod(x)
        assert state[0].dtype == torch.float32
        loss = F.mse_loss(y.float(), target.float())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    mb.raise_device_error(cuda)
    assert losses[-1] < 0.9 * losses[0]
