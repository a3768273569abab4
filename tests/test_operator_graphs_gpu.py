"""linear_attention, its step and block_norm in CUDA graphs: captured once, forward and backward, and
replayed on other inputs. The kernels sum in a fixed order, so a replay gives the bits of an eager call."""

from __future__ import annotations

import pytest
import test_block_norm_gpu as norm
import test_linear_attn_gpu as attn
import torch

pytestmark = pytest.mark.gpu


def _captured(f, static, cases):
    """f() on the static tensors, warmed up on a side stream and captured; then one replay for each case's values."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for case in cases:
        with torch.no_grad():
            for t, v in zip(static, case):
                t.copy_(v)
        graph.replay()
        replayed = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(replayed, f()))


@pytest.mark.parametrize("dtype,d,T", [(torch.bfloat16, 64, 1000), (torch.bfloat16, 128, 300), (torch.float32, 64, 700),
                                       (torch.float16, 72, 130)])
def test_attention(cuda, dtype, d, T):
    import mingru_b200 as mb

    cases = [attn.inputs(2, 3, T, d, d, dtype, cuda, seed=s, layout="bthd") for s in range(3)]
    static = [t.detach().clone() for t in cases[0]]
    leaves = [t.requires_grad_(True) for t in static[:5]]

    def f():
        out = mb.linear_attention(*leaves)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, static[5:])]

    _captured(f, static, cases)
    mb.raise_device_error(cuda)


def test_step(cuda):
    from mingru_b200 import step_ops

    def case(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        r = lambda *s: torch.randn(*s, device=cuda, generator=g)  # noqa: E731
        return [r(5, 4, 64).bfloat16(), r(5, 4, 64).bfloat16(), r(5, 4, 64).bfloat16(), -r(5, 4).abs(), r(5, 4, 64, 64)]

    static = case(0)
    out = torch.empty_like(static[4])
    _captured(lambda: step_ops.linear_attention_step(*static, out=out), static, [case(1), case(2)])


@pytest.mark.parametrize("D,kinds", [(512, ("residual", "bias")), (512, ("gate",)), (5001, ("residual", "scale"))])
def test_norm(cuda, D, kinds):
    import mingru_b200 as mb

    def case(seed):
        t, dy, dh = norm.inputs((300,), D, torch.float16, torch.float32, cuda, kinds, seed)
        return [*t.values(), dy, dh], list(t)

    static, names = case(0)
    leaves = [t.requires_grad_(True) for t in static[:-2]]

    def f():
        t = dict(zip(names, leaves))
        out = mb.block_norm(t["x"], t["weight"], t.get("bias"), residual=t.get("residual"), scale=t.get("scale"),
                            gate=t.get("gate"))
        out = out if isinstance(out, tuple) else (out,)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, static[-2:][:len(out)])]

    _captured(f, static, [case(1)[0], case(2)[0]])
