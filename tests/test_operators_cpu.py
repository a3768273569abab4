"""The linear-attention and norm operators without a GPU: sizes, refusals that
come before any launch, and the modules' constructors."""

from __future__ import annotations

import pytest
import torch


def test_sizes():
    from mingru_b200 import _lib

    lib = _lib.load()
    # states at each chunk of 128 tokens, 64 x 64 or 128 x 128 in fp32
    assert lib.mgs_linear_attn_saved_size(2, 3, 300, 64, 40, 1) == 6 * 3 * 64 * 64 * 4
    assert lib.mgs_linear_attn_saved_size(2, 3, 300, 65, 40, 1) == 6 * 3 * 128 * 128 * 4
    # fp32 heads of 130 x 70: three blocks by two
    assert lib.mgs_linear_attn_saved_size(1, 1, 128, 130, 70, 0) == 6 * 1 * 64 * 64 * 4
    assert lib.mgs_linear_attn_saved_size(1, 1, 128, 129, 8, 1) == 0
    assert lib.mgs_linear_attn_saved_size(-1, 1, 128, 8, 8, 1) == 0
    assert lib.mgs_linear_attn_workspace_size(1, 1, 128, 8, 8, 9) == 0
    assert lib.mgs_linear_attn_workspace_size(1, 1, 100000, 64, 64, 1) > 0
    assert lib.mgs_block_norm_workspace_size(100, 512, 1, 1) > 0
    assert lib.mgs_block_norm_workspace_size(100, 512, 3, 1) == 0
    assert lib.mgs_block_norm_workspace_size(100, 16385, 1, 1) == 0


def test_cpu_tensors_raise():
    import mingru_b200 as mb
    from mingru_b200 import step_ops

    q, lg, S = torch.rand(1, 2, 4, 8), torch.zeros(1, 2, 4), torch.zeros(1, 2, 8, 8)
    with pytest.raises(ValueError, match="CUDA"):
        mb.linear_attention(q, q, q, lg)
    with pytest.raises(ValueError, match="CUDA"):
        step_ops.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], lg[:, :, 0], S)
    with pytest.raises(ValueError, match="CUDA"):
        mb.block_norm(torch.rand(3, 8), torch.ones(8))
    with pytest.raises(ValueError, match="shapes disagree"):
        mb.linear_attention(q, q[..., :4], q, lg)
    with pytest.raises(ValueError, match="groups"):
        mb.block_norm(torch.rand(3, 8), torch.ones(8), groups=3)


def test_constructors():
    import mingru_b200 as mb

    with pytest.raises(ValueError, match="n_heads"):
        mb.RetentionMinGRU(8, 8, n_heads=0)
    with pytest.raises(ValueError, match="divisible"):
        mb.RetentionMinGRU(8, 10, n_heads=4)
    mod = mb.MinGRUStack(8, 16, 2, mixer=["retention", "log"], fused_norms=True)
    assert mod.blocks[0].fused_norms and isinstance(mod.blocks[0].mingru, mb.RetentionMinGRU)
    # the option adds no weights: checkpoints go both ways
    assert mod.state_dict().keys() == mb.MinGRUStack(8, 16, 2, mixer=["retention", "log"]).state_dict().keys()
