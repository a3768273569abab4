"""dlog_gamma against float64 as closely as its sums allow.

A row's or a column's sum of R has at most 128 terms, of random sign, within 2^-24 of their size each: 16 * 2^-24,
1e-6 of it. dlog_gamma inside a chunk takes differences of such sums over the 16 tokens to the next edge of a
quarter at most, and the sums of the quarters beyond it: 32 errors of random sign, 5.7 times one, 6e-6 of a sum
that is no larger than the pairs across a token are where a memory is longer than a token or two. What comes
through the state is summed as it is: 1e-6. Together within 1e-5, norm over norm."""

from __future__ import annotations

import pytest
import test_linear_attn_gpu as attn
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["token", "head", "none", "resets"])
@pytest.mark.parametrize("T,d", [(128, 64), (333, 64), (700, 40), (1500, 64)])
def test_decay_gradient(cuda, T, d, kind, dtype):
    import mingru_b200 as mb

    Q, K, V, lg, H0, dy, dH = attn.inputs(2, 3, T, d, d, dtype, cuda, kind=kind, seed=T)
    lg = lg.expand(2, 3, T).contiguous()  # a gradient for every token, not their sum
    own, ref = lg.clone().requires_grad_(True), lg.double().requires_grad_(True)
    got = torch.autograd.grad(mb.linear_attention(Q, K, V, own, H0), own, (dy, dH))[0]
    want = torch.autograd.grad(attn.recurrence(*(t.double() for t in (Q, K, V)), ref, H0.double()), ref,
                               (dy.double(), dH.double()))[0]
    want = torch.nan_to_num(want)  # 0 * inf of the reference at a wipe
    assert (got.double() - want).norm() <= 1e-5 * want.norm()
