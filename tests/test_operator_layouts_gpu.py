"""linear_attention, its step and block_norm on tensors that lie in uncommon ways, against float64:
tolerances and plain forms are those of the operators' own test files."""

from __future__ import annotations

import pytest
import test_block_norm_gpu as norm
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
