"""A bounded wait of linear attention that runs out: the launch ends, the sticky word has it, tensor memory
is free again and the next call is right. The hook's barrier is one that nothing arrives on, and every wait
on it is bounded by a small number of polls."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TIMEOUT_BIT = 1 << 6  # MGS_LOOKBACK_TIMEOUT


def test_wait_that_runs_out(cuda):
    import mingru_b200 as mb
    import test_linear_attn_gpu as attn
    from mingru_b200 import _lib

    lib = _lib.load()
    mb.take_device_error(cuda)
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(3):
        assert lib.mgs_test_linear_attn_timeout(1000, stream) == 0
    torch.cuda.synchronize()
    assert mb.take_device_error(cuda) & TIMEOUT_BIT
    assert mb.take_device_error(cuda) == 0  # read and cleared
    assert lib.mgs_test_linear_attn_timeout(1000, stream) == 0
    with pytest.raises(RuntimeError, match="MGS_LOOKBACK_TIMEOUT"):
        mb.raise_device_error(cuda)
    attn.check(cuda, 8, 8, 700, 64, 64, torch.bfloat16)


def test_hook_refuses(cuda):
    from mingru_b200 import _lib

    st = _lib.load().mgs_test_linear_attn_timeout(0, torch.cuda.current_stream().cuda_stream)
    assert _lib.STATUS_NAMES[st] == "MGS_BAD_SHAPE"
