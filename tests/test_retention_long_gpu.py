"""RetentionMinGRU's step with a time decay, and heads of several blocks over long sequences.

Tolerances: the mixer's as in its own tests; linear attention's as in its own, whose bound for fp32 counts the
roundings of a chunk and of as many joins of chunks: the same for any length."""

from __future__ import annotations

import pytest
import test_linear_attn_gpu as attn
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(decay="fixed"), dict(decay="learnable", n_heads=2, d_k=24, d_v=40),
                                dict(decay="learnable", log1p_delta=True)])
def test_steps_with_a_time_decay(cuda, kw):
    import mingru_b200 as mb

    torch.manual_seed(0)
    mod = mb.RetentionMinGRU(20, 64, **kw).to(cuda)
    x = torch.randn(3, 40, 20, device=cuda)
    dt = 2 * torch.rand(3, 40, device=cuda)
    with torch.no_grad():
        want, last = mod(x, None, dt, return_state=True)
        state, ys = None, []
        for t in range(x.shape[1]):
            y, state = mod.step(x[:, t], state, dt[:, t])
            ys.append(y)
    torch.testing.assert_close(torch.stack(ys, 1), want, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(state, last[:, 0], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype,dk,dv", [(torch.float32, 128, 72), (torch.float16, 40, 130), (torch.bfloat16, 136, 64)])
def test_blocks_over_long_sequences(cuda, dtype, dk, dv):
    attn.check(cuda, 1, 2, 2500, dk, dv, dtype)
    attn.check(cuda, 2, 1, 1100, dk, dv, dtype, kind="resets", h0=False, layout="slice")
