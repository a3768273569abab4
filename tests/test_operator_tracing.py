"""linear_attention and block_norm as compilers and other tracers see them: fake CUDA tensors, no GPU."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import ShapeEnv


@pytest.fixture
def fake():
    import mingru_b200  # noqa: F401  (registers the ops)

    with FakeTensorMode(shape_env=ShapeEnv()) as mode:
        yield mode


def _cuda(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_strides_that_the_fakes_give(fake):
    """Outputs as the op allocates them: in the input's order where its rows are dense, else contiguous."""
    ops = torch.ops.mingru_b200
    Q = _cuda(2, 150, 3, 32).transpose(1, 2)
    K = _cuda(2, 3, 32, 150).transpose(2, 3)  # copied by the op: rows are not dense
    V = torch.as_strided(_cuda(2000), (2, 3, 150, 40), (0, 500, 1, 1))  # windows
    lg = _cuda(2, 3, 150)
    y, H, saved = ops.linear_attn_fwd(Q, K, V, lg, None, True)
    dQ, dK, dV, dlg, dH0 = ops.linear_attn_bwd(Q, K, V, lg, saved, y, None, True)
    assert dQ.stride() == (150 * 96, 32, 96, 1)
    assert dK.stride() == (450 * 32, 150 * 32, 32, 1)
    assert y.stride() == dV.stride() and y.stride(-1) == 1
    assert H.stride() == dH0.stride() == (3 * 32 * 40, 32 * 40, 40, 1) and dlg.stride() == (450, 150, 1)


def test_saved_states_of_the_fake_are_the_librarys(fake):
    from mingru_b200 import _lib

    size = _lib.load().mgs_linear_attn_saved_size
    for code, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        for B, H, T, dk, dv in [(2, 3, 300, 64, 40), (1, 1, 1, 1, 1), (1, 2, 128, 65, 3), (3, 1, 129, 7, 128),
                                (2, 2, 0, 8, 8), (0, 2, 5, 8, 8), (1, 3, 5000, 128, 128), (2, 1, 257, 130, 70)]:
            if dtype == torch.bfloat16 and max(dk, dv) > 128:
                continue  # not a call of the op's
            Q, V, lg = _cuda(B, H, T, dk, dtype=dtype), _cuda(B, H, T, dv, dtype=dtype), _cuda(B, H, T)
            saved = torch.ops.mingru_b200.linear_attn_fwd(Q, Q, V, lg, None, True)[2]
            assert 4 * saved.numel() == size(B, H, T, dk, dv, code)


def test_lengths_that_are_symbols():
    """Dynamic shapes: batch and length are not numbers while a compiler looks at the op."""
    import mingru_b200  # noqa: F401
    from torch._dynamo.source import ConstantSource
    from torch.fx.experimental.symbolic_shapes import DimDynamic, StatelessSymbolicContext

    mode = FakeTensorMode(shape_env=ShapeEnv())

    def symbolic(name, *shape):
        kinds = [DimDynamic.DYNAMIC if i in (0, 2) else DimDynamic.STATIC for i in range(len(shape))]
        return mode.from_tensor(torch.empty(*shape, device="meta"), source=ConstantSource(name),
                                symbolic_context=StatelessSymbolicContext(kinds))

    q, g = symbolic("q", 2, 3, 300, 64), symbolic("g", 2, 3, 300)
    assert not isinstance(q.shape[2], int)
    with mode:
        y, H, saved = torch.ops.mingru_b200.linear_attn_fwd(q, q, q, g, None, True)
        assert y.shape == q.shape
        assert saved.shape[0].node.expr.free_symbols == (q.shape[0] * q.shape[2]).node.expr.free_symbols
        grads = torch.ops.mingru_b200.linear_attn_bwd(q, q, q, g, saved, y, None, False)
        assert all(t.shape == q.shape for t in grads[:3]) and grads[4].numel() == 0


def _compiled_calls(f, *args):
    """Name and arguments of every op that a compiler sees in f(*args)."""
    calls = []

    def backend(gm, _):
        calls.extend((str(n.target), n.args) for n in gm.graph.nodes if "mingru_b200" in str(n.target))
        return gm.forward

    torch._dynamo.reset()
    torch.compile(f, backend=backend, fullgraph=True)(*args)
    return dict(calls)


def test_compiled_inference_saves_nothing(fake):
    """States and statistics are for a backward: written only where one can follow, compiled as eager."""
    import mingru_b200 as mb

    q, lg, w = _cuda(1, 2, 300, 32), _cuda(1, 2, 300), _cuda(32)

    def f(q, lg, w):
        return mb.linear_attention(q, q, q, lg), mb.block_norm(q, w)

    def saves():
        calls = _compiled_calls(f, q, lg, w)
        return (calls["mingru_b200.linear_attn_fwd.default"][-1], calls["mingru_b200.block_norm_fwd.default"][-1])

    assert saves() == (False, False)  # no tensor wants a gradient
    q.requires_grad_(True)
    assert saves() == (True, True)
    with torch.no_grad():
        assert saves() == (False, False)
    stats = torch.ops.mingru_b200.block_norm_fwd(q.detach(), w, None, None, None, None, 1, 1e-5, False, False)[2]
    assert stats.numel() == 0


def test_calls_under_dispatch_modes(fake):
    """Fake tensors, tracers and dispatch modes see the ops, as they see the scans'."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    import mingru_b200 as mb

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.add(str(func))
            return func(*args, **(kwargs or {}))

    q, lg, w = _cuda(1, 2, 300, 32), _cuda(1, 2, 300), _cuda(32)
    ops = {"mingru_b200.linear_attn_fwd.default", "mingru_b200.block_norm_fwd.default"}

    def f(q, lg, w):
        y, H = mb.linear_attention(q, q, q, lg)
        return mb.block_norm(y, w), H

    for grad in (False, True):
        q.requires_grad_(grad)
        with Seen() as seen:
            y, H = f(q, lg, w)
        assert y.shape == q.shape and H.shape == (1, 2, 32, 32) and y.requires_grad == grad
        assert ops <= seen.names
        assert ops <= {str(n.target) for n in make_fx(f)(q, lg, w).graph.nodes}
