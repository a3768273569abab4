"""linear_attention and block_norm under compilers and tracers on the GPU: the same bits as eager calls."""

from __future__ import annotations

import pytest
import test_linear_attn_gpu as attn
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def fresh_compiler():
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


def _same(f, g, x, weights):
    """Outputs of f and g on x, and gradients of every tensor that takes one."""
    a, b = f(*x), g(*x)
    leaves = [t for t in x if t.requires_grad]
    da, db = torch.autograd.grad(a, leaves, weights), torch.autograd.grad(b, leaves, weights)
    assert all(torch.equal(s, t) and s.dtype == t.dtype for s, t in zip((*a, *da), (*b, *db)))


def _attention_case(cuda, T, dtype, transposed=False, B=2):
    Q, K, V, lg, H0, dy, dH = attn.inputs(B, 3, T, 32, 40, dtype, cuda, seed=T)
    if transposed:
        V = V.transpose(2, 3).contiguous().transpose(2, 3)
    return [t.detach().requires_grad_(True) for t in (Q, K, V, lg, H0)], (dy, dH)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dynamic", [True, None])
def test_attention_at_several_lengths(cuda, dynamic, dtype):
    """With None the second length makes it a symbol."""
    import mingru_b200 as mb

    f = torch.compile(lambda *a: mb.linear_attention(*a), backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for T, B in ((150, 2), (300, 2), (129, 3)):
        x, w = _attention_case(cuda, T, dtype, B=B)
        _same(f, mb.linear_attention, x, w)


@pytest.mark.parametrize("dynamic", [True, False])
def test_retention_at_several_lengths(cuda, dynamic):
    import mingru_b200 as mb

    torch.manual_seed(0)
    mod = mb.RetentionMinGRU(24, 64, n_heads=2).to(cuda)
    compiled = torch.compile(mod, backend="aot_eager", dynamic=dynamic)
    for T in (140, 260):
        x = torch.randn(2, T, 24, device=cuda, requires_grad=True)
        want, got = mod(x), compiled(x)
        torch.testing.assert_close(got, want)
        w = torch.randn_like(want)
        for a, b in zip(torch.autograd.grad(got, [x, *mod.parameters()], w),
                        torch.autograd.grad(want, [x, *mod.parameters()], w)):
            torch.testing.assert_close(a, b)


@pytest.mark.parametrize("save", [True, False])
@pytest.mark.parametrize("transposed", [False, True])
def test_fakes_against_the_op(cuda, transposed, save):
    x, _ = _attention_case(cuda, 150, torch.float32, transposed)
    args = (*(t.detach() for t in x), save)
    torch.library.opcheck(torch.ops.mingru_b200.linear_attn_fwd, args,
                          test_utils=("test_schema", "test_faketensor"))
    if save:
        y, H, saved = torch.ops.mingru_b200.linear_attn_fwd(*args)
        torch.library.opcheck(torch.ops.mingru_b200.linear_attn_bwd, (*args[:4], saved, y, H, True),
                              test_utils=("test_schema", "test_faketensor"))


def test_under_a_dispatch_mode(cuda):
    """A mode sees the ops, forward and backward, and results are those of calls without one."""
    from torch.utils._python_dispatch import TorchDispatchMode

    import mingru_b200 as mb

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.add(str(func))
            return func(*args, **(kwargs or {}))

    def f(q, lg, w):
        y = mb.block_norm(mb.linear_attention(q, q, q, lg)[0], w)
        return [y, *torch.autograd.grad(y, (q, lg, w), y.detach())]

    g = torch.Generator(device=cuda).manual_seed(0)
    x = [torch.randn(1, 2, 300, 32, device=cuda, generator=g), -torch.rand(1, 2, 300, device=cuda, generator=g),
         1 + torch.rand(32, device=cuda, generator=g)]
    x = [t.requires_grad_(True) for t in x]
    with Seen() as seen:
        got = f(*x)
    assert {f"mingru_b200.{n}.default" for n in ("linear_attn_fwd", "linear_attn_bwd", "block_norm_fwd",
                                                 "block_norm_bwd")} <= seen.names
    assert all(torch.equal(a, b) for a, b in zip(got, f(*x)))
