"""fused_norms against the modules' own calls, without a GPU: types, hooks, wrappers, old pickles."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.mark.parametrize("stream,branch", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float32)])
def test_stream_and_branch_of_two_types(stream, branch):
    """A 32-bit stream with a 16-bit branch, as autocast makes them: promoted, as x + branch is."""
    from mingru_b200.modules import _add_norm

    norm = nn.LayerNorm(32)
    with FakeTensorMode(allow_non_fake_inputs=True):
        norm.to("cuda")
        x, b = torch.empty(3, 32, device="cuda", dtype=stream), torch.empty(3, 32, device="cuda", dtype=branch)
        y, h = _add_norm(x, b, norm)
    assert y.dtype == h.dtype == (x + b).dtype == torch.float32
