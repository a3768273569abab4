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


def test_keys_of_zeros_in_fp16():
    """A token whose keys are zeros (padding, no bias) has no direction, and writes nothing."""
    from mingru_b200 import RetentionMinGRU

    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        mod = RetentionMinGRU(16, 32, bias=False, n_heads=2).to(dtype)
        q, k, v, log_gamma = mod._coeffs(torch.zeros(2, 3, 16, dtype=dtype), None)
        assert not k.any() and torch.isfinite(log_gamma).all()


def test_coefficients_share_a_type_under_autocast(monkeypatch):
    """Where normalising comes out in 32 bits, as under autocast, keys take the queries' type."""
    import torch.nn.functional as F

    from mingru_b200 import RetentionMinGRU

    normalize = F.normalize
    monkeypatch.setattr(F, "normalize", lambda x, **kw: normalize(x.float(), **kw))
    mod = RetentionMinGRU(16, 32, n_heads=2).bfloat16()
    q, k, v, _ = mod._coeffs(torch.randn(2, 3, 16).bfloat16(), None)
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16
