"""linear_attention_step against its formula in float64 and against the whole
sequence's kernel, in place and into a buffer, and its refusals.

Tolerances: the state is one fused product and sum per entry in fp32 (2^-23,
with exp of the decay 2^-22 more: 1e-6); y sums d_k of them in a tree (at most
10 roundings deep: 2e-6) and is rounded once, 2^-8 for bf16, 2^-11 for fp16."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def near(got, ref, tol):
    d, rms = (got.double() - ref).abs(), ref.square().mean().sqrt()
    assert (d <= tol * (ref.abs() + 2 * rms)).all()


def inputs(B, H, dk, dv, dtype, dev):
    g = torch.Generator(device=dev).manual_seed(B + dk)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    lg = -torch.nn.functional.softplus(r(B, H) - 2)
    return r(B, H, dk).to(dtype), r(B, H, dk).to(dtype), r(B, H, dv).to(dtype), lg, r(B, H, dk, dv)


def plain(q, k, v, lg, S):
    S = lg.double().exp()[..., None, None] * S.double() + k.double()[..., None] * v.double()[..., None, :]
    return (q.double()[..., None, :] @ S).squeeze(-2), S


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (1, 4, 64, 64), (3, 5, 33, 40), (2, 3, 40, 33), (2, 2, 128, 128),
                                       (1, 2, 7, 300), (1, 1, 300, 1028), (70, 3, 16, 16)])
def test_step(cuda, B, H, dk, dv, dtype):
    from mingru_b200 import step_ops as so

    q, k, v, lg, S = inputs(B, H, dk, dv, dtype, cuda)
    ry, rS = plain(q, k, v, lg, S)
    keep = S.clone()
    y, S1 = so.linear_attention_step(q, k, v, lg, S)
    assert torch.equal(S, keep) and y.dtype == dtype
    near(y, ry, TOL[dtype])
    near(S1, rS, 1e-6)
    y2, S2 = so.linear_attention_step(q, k, v, lg, S, out=S)  # in place
    assert S2 is S and torch.equal(S, S1) and torch.equal(y2, y)


def test_odd_buffers(cuda):
    """A state that starts off 16 bytes; decays of a head, wiped and whole."""
    from mingru_b200 import step_ops as so

    q, k, v, _, S = inputs(2, 3, 24, 20, torch.float32, cuda)
    buf = torch.empty(S.numel() + 1, device=cuda)[1:].view_as(S).copy_(S)
    lg = torch.tensor([0.0, -0.3, -float("inf")], device=cuda)
    y, S1 = so.linear_attention_step(q, k, v, lg, buf, out=torch.empty_like(S))
    ry, rS = plain(q, k, v, lg.expand(2, 3), S)
    near(y, ry, TOL[torch.float32])
    near(S1, rS, 1e-6)
    y, S1 = so.linear_attention_step(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, lg, S.transpose(2, 3).contiguous().transpose(2, 3))
    near(S1, rS, 1e-6)


def test_steps_are_the_sequence(cuda):
    import mingru_b200 as mb
    from mingru_b200 import step_ops as so

    g = torch.Generator(device=cuda).manual_seed(0)
    B, H, T, d = 2, 3, 140, 64
    Q, K, V = (torch.randn(B, H, T, d, device=cuda, generator=g) * d**-0.5 for _ in range(3))
    lg = -torch.rand(B, H, T, device=cuda, generator=g) * 0.2
    y, HT = mb.linear_attention(Q, K, V, lg)
    S = torch.zeros(B, H, d, d, device=cuda)
    ys = [so.linear_attention_step(Q[:, :, t], K[:, :, t], V[:, :, t], lg[:, :, t], S, out=S)[0] for t in range(T)]
    # both within their tolerance of the recurrence; the steps' roundings add up over a decay's reach
    near(torch.stack(ys, 2), y.double(), 1e-5)
    near(S, HT.double(), 1e-5)


def test_empty_batch(cuda):
    from mingru_b200 import step_ops as so

    z = torch.zeros(0, 2, 8, device=cuda)
    y, S = so.linear_attention_step(z, z, z, torch.zeros(0, 2, device=cuda), torch.zeros(0, 2, 8, 8, device=cuda))
    assert y.shape == (0, 2, 8) and S.shape == (0, 2, 8, 8)


def test_refusals(cuda):
    from mingru_b200 import step_ops as so

    q, k, v, lg, S = inputs(1, 2, 8, 8, torch.float32, cuda)
    for args, kw, match in [
        ((q, k[..., :4], v, lg, S), {}, "need q"),
        ((q, k, v[:, :1], lg, S), {}, "need q"),
        ((q[0], k[0], v[0], lg, S), {}, "need q"),
        ((q, k, v, lg, S[..., :4]), {}, "H_prev"),
        ((q, k, v, lg, S.bfloat16()), {}, "H_prev"),
        ((q, k, v, lg, S), dict(out=S[..., :4]), "out"),
        ((q, k, v, lg, S), dict(out=S.transpose(2, 3)), "contiguous"),
        ((q, k, v, lg[:, :1].expand(1, 3), S), {}, "broadcast"),
        ((q, k.bfloat16(), v, lg, S), {}, "dtype"),
        ((q.double(), k.double(), v.double(), lg, S), {}, "not supported"),
        ((q.cpu(), k.cpu(), v.cpu(), lg.cpu(), S.cpu()), {}, "CUDA"),
        ((q, k, v, lg, S.cpu()), {}, "CUDA"),
    ]:
        with pytest.raises(ValueError, match=match):
            so.linear_attention_step(*args, **kw)
