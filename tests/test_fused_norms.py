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


def _stack():
    """On fake CUDA tensors, in a FakeTensorMode."""
    from mingru_b200 import MinGRUStack

    with torch.device("cuda"):
        return MinGRUStack(16, 32, 3, mixer="retention", mixer_kwargs=dict(n_heads=2), fused_norms=True)


def test_hooks_of_blocks_and_norms_run(monkeypatch):
    """What is hooked to a block, a norm or every module runs with fused_norms too."""
    from mingru_b200 import step_ops

    monkeypatch.setattr(step_ops, "linear_attention_step", lambda q, k, v, lg, H: (v, H))
    with FakeTensorMode():
        stack = _stack()
        x = torch.empty(2, 5, 16, device="cuda")
        seen = []
        hooked = [*stack.blocks, stack.blocks[1].norm1, stack.blocks[2].norm2, stack.norm_out]
        handles = [m.register_forward_hook(lambda m, a, out: seen.append(m)) for m in hooked]
        y, _ = stack(x)
        assert len(seen) == len(hooked) and set(seen) == set(hooked) and y.shape == (2, 5, 32)
        for h in handles:
            h.remove()
        seen.clear()
        stack.blocks[0].norm1.register_forward_pre_hook(lambda m, a: seen.append(m))
        stack.step(x[:, 0], stack.init_state())
        assert seen == [stack.blocks[0].norm1]
        seen.clear()
        handle = nn.modules.module.register_module_forward_hook(lambda m, a, out: seen.append(m))
        stack(x)
        handle.remove()
        assert {*stack.blocks, *(b.norm1 for b in stack.blocks), *(b.norm2 for b in stack.blocks), stack.norm_out} <= set(seen)


def test_replaced_parts_run():
    """Wrapped blocks, other norms and replaced forwards are called, not gone past."""

    class Wrapper(nn.Module):  # as checkpointing or sharding wraps a block
        def __init__(self, inner):
            super().__init__()
            self.inner, self.calls = inner, 0

        def forward(self, *args):
            self.calls += 1
            return self.inner(*args)

        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                return getattr(self.inner, name)

    class Half(nn.LayerNorm):
        def forward(self, x):
            return 0.5 * super().forward(x)

    with FakeTensorMode():
        stack = _stack()
        x = torch.empty(2, 5, 16, device="cuda")
        stack.blocks[1] = Wrapper(stack.blocks[1])
        calls = []
        forward = stack.blocks[2].forward
        stack.blocks[2].forward = lambda *a: calls.append(2) or forward(*a)
        stack.blocks[0].norm2 = Half(32, device="cuda")
        half = stack.blocks[0].norm2
        half.forward = lambda t: calls.append(0) or Half.forward(half, t)
        stack.norm_out = nn.Identity()
        y, state = stack(x)
        assert stack.blocks[1].calls == 1 and calls == [0, 2] and y.shape == (2, 5, 32) and len(state) == 3


def test_fused_calls_stay_few():
    """Without hooks every norm of a stack is one op with its sum: 3 blocks of two norms, and the last."""
    import mingru_b200  # noqa: F401

    calls = []

    def backend(gm, _):
        calls.extend(n for n in gm.graph.nodes if "block_norm_fwd" in str(n.target))
        return gm.forward

    with FakeTensorMode():
        stack = _stack()
        torch._dynamo.reset()
        torch.compile(stack, backend=backend, fullgraph=True)(torch.empty(2, 5, 16, device="cuda"))
    assert len(calls) == 7 + 3  # and the mixers' own


def test_modules_pickled_before_the_option():
    """Blocks and stacks that were pickled whole before fused_norms existed have no such attribute."""
    import copy

    import mingru_b200 as mb

    stack = mb.MinGRUStack(8, 16, 2)
    for m in (stack, *stack.blocks):
        del m.__dict__["fused_norms"]
    old = copy.deepcopy(stack)
    assert not old.fused_norms and not old.blocks[0].fused_norms


def test_rows_beyond_the_kernels(monkeypatch):
    """block_norm takes up to 16384 channels; wider streams keep the norm's own call."""
    from mingru_b200 import modules

    def refuse(x, *a, **kw):
        assert x.shape[-1] <= 16384, "MGS_UNSUPPORTED"
        return x if kw.get("residual") is None else (x, x)

    monkeypatch.setattr(modules, "block_norm", refuse)
    for D in (16384, 16385):
        norm, x = nn.LayerNorm(D), torch.randn(2, D)
        y, h = modules._add_norm(x, x, norm)
        if D > 16384:
            torch.testing.assert_close(y, norm(x + x))
            torch.testing.assert_close(h, x + x)
        modules._add_norm(x, None, norm)
