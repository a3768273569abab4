"""block_norm against its definition in float64 (gradients by autograd through
it), against differences of its own forward, and its refusals.

Tolerances (2-norm of the error over 2-norm of the result, and the largest
error over |result| + 8 rms): outputs are fp32 sums of at most 16384 terms in a
tree (a thread's 16 in order, then pairs: 30 roundings of 2^-24 at most, 2e-6)
rounded once to the type, 2^-9 for bf16 and 2^-12 for fp16 (half a unit in the
last place, 2^-8 and 2^-11 of the smaller neighbours). The gradients of weight,
bias and scale sum rows with random signs, whose result is smaller than the
terms by the root of their number: 1e-5 in fp32. A directional derivative by a
central step of 1e-2 is off by the cubic term, 1e-4 of the slope's scale, and by
the forward's rounding over the step, 2e-6 / 1e-2: 1e-3."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SUMS = 1e-5


def close(got, ref, tol, name):
    got, ref = got.detach().double(), ref.detach().double()
    assert got.shape == ref.shape and torch.isfinite(got).all(), name
    if not ref.numel():
        return
    d, rms = (got - ref).abs(), ref.square().mean().sqrt()
    if rms == 0:
        assert d.max() == 0, name
        return
    rel, big = (d.norm() / ref.norm()).item(), (d / (ref.abs() + 8 * rms)).max().item()
    assert rel <= tol and big <= tol, f"{name}: rel {rel:.3g}, max {big:.3g} (tolerance {tol:.3g})"


def plain(x, weight, bias, residual, scale, gate, groups, eps, rms):
    h = x if scale is None else x * scale
    h = h if residual is None else h + residual
    z = h.unflatten(-1, (groups, -1))
    z = z if rms else z - z.mean(-1, keepdim=True)
    z = (z / (z.square().mean(-1, keepdim=True) + eps).sqrt()).flatten(-2) * weight
    z = z if bias is None else z + bias
    z = z if gate is None else z * gate * torch.sigmoid(gate)
    return z if residual is None else (z, h)


NAMES = ("x", "weight", "bias", "residual", "scale", "gate")


def inputs(rows, D, dtype, wdtype, dev, kinds, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    t = {"x": (r(*rows, D) + 0.5).to(dtype), "weight": (1 + 0.3 * r(D)).to(wdtype)}
    if "bias" in kinds:
        t["bias"] = (0.3 * r(D)).to(wdtype)
    if "residual" in kinds:
        t["residual"] = (2 * r(*rows, D)).to(dtype)
    if "scale" in kinds:
        t["scale"] = (0.5 + 0.3 * r(D)).to(wdtype)
    if "gate" in kinds:
        t["gate"] = (2 * r(*rows, D)).to(dtype)
    return t, r(*rows, D).to(dtype), r(*rows, D).to(dtype)


def check(dev, rows, D, dtype, kinds=(), wdtype=None, groups=1, rms=False, eps=1e-5, view=None):
    import mingru_b200 as mb

    wdtype = wdtype or dtype
    t, dy, dh = inputs(rows, D, dtype, wdtype, dev, kinds)
    if view is not None:
        t = {n: view(a) if a.dim() > 1 else a for n, a in t.items()}
        dy, dh = view(dy), view(dh)
    own = {n: a.detach().requires_grad_(True) for n, a in t.items()}
    ref = {n: a.detach().double().requires_grad_(True) for n, a in t.items()}
    kw = lambda a: dict(residual=a.get("residual"), scale=a.get("scale"), gate=a.get("gate"),  # noqa: E731
                        groups=groups, eps=eps, rms=rms)
    got = mb.block_norm(own["x"], own["weight"], own.get("bias"), **kw(own))
    want = plain(ref["x"], ref["weight"], ref.get("bias"), **kw(ref))
    with torch.no_grad():
        again = mb.block_norm(own["x"], own["weight"], own.get("bias"), **kw(own))
    got, want, again = (a if isinstance(a, tuple) else (a,) for a in (got, want, again))
    for n, a, b, c in zip(("y", "h"), got, want, again):
        assert a.dtype == dtype and torch.equal(a, c)
        close(a, b, TOL[dtype], n)
    outs = (dy, dh)[:len(got)]
    grads = torch.autograd.grad(got, list(own.values()), outs)
    refs = torch.autograd.grad(want, list(ref.values()), [o.double() for o in outs])
    for n, a, b in zip(own, grads, refs):
        per_row = n in ("x", "residual", "gate")
        tol = TOL[dtype] if per_row else max(SUMS, TOL[wdtype])
        # the gradient through a norm is a difference of terms of its size, three of them
        close(a, b, 3 * tol if dtype == torch.float32 or not per_row else tol, "d" + n)
    mb.raise_device_error(dev)


ALL = [(), ("bias",), ("residual", "bias"), ("residual", "scale"), ("gate",), ("gate", "bias"),
       ("residual", "scale", "gate", "bias")]


@pytest.mark.parametrize("kinds", ALL)
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_parts(cuda, dtype, rms, kinds):
    check(cuda, (37,), 256, dtype, kinds, rms=rms)
    check(cuda, (5, 9), 99, dtype, kinds, rms=rms)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 64, 127, 129, 512, 1000, 1024, 2047, 4096, 5001, 8192, 16384])
def test_widths(cuda, D, dtype):
    # a single channel has no spread: its LayerNorm is the bias, with gradients of nothing but rounding
    check(cuda, (19,), D, dtype, ("residual", "scale"), rms=D <= 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("D,groups", [(64, 8), (512, 8), (512, 64), (360, 5), (91, 13), (4096, 2), (8192, 128),
                                      (6000, 3)])
def test_groups(cuda, D, groups, dtype):
    check(cuda, (23,), D, dtype, ("gate", "bias"), groups=groups, rms=True)
    if D // groups > 2:
        check(cuda, (23,), D, dtype, ("residual",), groups=groups)


@pytest.mark.parametrize("rows", [1, 2, 1000, 5003])
def test_rows(cuda, rows):
    check(cuda, (rows,), 512, torch.bfloat16, ("residual", "bias"))
    check(cuda, (rows,), 48, torch.float32, ("gate",), groups=3, rms=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp32_weights(cuda, dtype):
    check(cuda, (300,), 256, dtype, ("residual", "scale", "bias"), wdtype=torch.float32)
    check(cuda, (300,), 63, dtype, ("gate",), wdtype=torch.float32, rms=True)


def test_strided_rows(cuda):
    """Slices of a wider tensor, aligned and not; transposed rows are copied."""

    def slice_of(first, width):
        def view(a):
            wide = torch.zeros(*a.shape[:-1], width, dtype=a.dtype, device=a.device)
            out = wide[..., first:first + a.shape[-1]]
            return out.copy_(a)
        return view

    for dtype in (torch.float32, torch.bfloat16):
        for view in (slice_of(64, 512), slice_of(3, 517), lambda a: a.transpose(0, 1).contiguous().transpose(0, 1)):
            check(cuda, (6, 11), 128, dtype, ("residual", "gate"), view=view)


def test_offset_rows(cuda):
    """Large means: the spread is taken about the mean, not from squares."""
    import mingru_b200 as mb

    x = torch.randn(50, 512, device=cuda) + 1000
    w = torch.ones(512, device=cuda)
    # x keeps 1000's unit in the last place, 6e-5 of its spread, whatever the kernel does
    close(mb.block_norm(x, w), plain(x.double(), w.double(), None, None, None, None, 1, 1e-5, False), 2e-6, "y")


def test_constant_and_zero_rows(cuda):
    """Rows without a spread: eps alone under the root."""
    import mingru_b200 as mb

    x = torch.zeros(4, 64, device=cuda)
    x[1] = 3.0
    x.requires_grad_(True)
    w = torch.ones(64, device=cuda)
    for rms in (False, True):
        y = mb.block_norm(x, w, rms=rms)
        close(y, plain(x.double(), w.double(), None, None, None, None, 1, 1e-5, rms), 2e-6, "y")
        g = torch.autograd.grad(y.sum(), x)[0]
        assert torch.isfinite(g).all()


def test_no_rows(cuda):
    import mingru_b200 as mb

    x = torch.zeros(0, 32, device=cuda, requires_grad=True)
    w = torch.ones(32, device=cuda, requires_grad=True)
    y, h = mb.block_norm(x, w, residual=x.detach())
    assert y.shape == h.shape == (0, 32)
    g = torch.autograd.grad(y.sum() + h.sum(), (x, w))
    assert g[0].shape == (0, 32) and not g[1].any()


def test_differences(cuda):
    import mingru_b200 as mb

    t, dy, dh = inputs((40,), 96, torch.float32, torch.float32, cuda, ("bias", "residual", "scale", "gate"), 5)
    x = [a.requires_grad_(True) for a in t.values()]

    def loss(a):
        a = dict(zip(t, a))
        y, h = mb.block_norm(a["x"], a["weight"], a["bias"], residual=a["residual"], scale=a["scale"],
                             gate=a["gate"], groups=4)
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()

    grads = torch.autograd.grad(loss(x), x)
    gen = torch.Generator(device=cuda).manual_seed(6)
    for i, (n, g) in enumerate(zip(t, grads)):
        v = torch.randn(x[i].shape, device=cuda, generator=gen)
        with torch.no_grad():
            up, down = ([a + s * v if j == i else a for j, a in enumerate(x)] for s in (1e-2, -1e-2))
            diff = (loss(up) - loss(down)) / 2e-2
        want = (g.double() * v.double()).sum()
        assert abs(diff - want) <= 1e-3 * g.double().norm() * v.double().norm(), n


def test_one_output_used(cuda):
    import mingru_b200 as mb

    x, r = (torch.randn(10, 64, device=cuda, requires_grad=True) for _ in range(2))
    w = torch.ones(64, device=cuda, requires_grad=True)
    y, h = mb.block_norm(x, w, residual=r)
    gx, gr = torch.autograd.grad(h.sum(), (x, r))
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, torch.ones_like(r))
    xd, rd = (a.detach().double().requires_grad_(True) for a in (x, r))
    want = torch.autograd.grad(plain(xd, w.detach().double(), None, rd, None, None, 1, 1e-5, False)[0].square().sum(), xd)[0]
    y, h = mb.block_norm(x, w, residual=r)
    got = torch.autograd.grad(y.square().sum(), x)[0]
    # y^2 summed over a row does not change with the row: a gradient of rounding alone
    assert (got.double() - want).abs().max() <= 1e-5


def test_another_stream_and_repeats(cuda):
    import mingru_b200 as mb

    t, dy, dh = inputs((2000,), 320, torch.bfloat16, torch.bfloat16, cuda, ("bias", "residual", "scale"))
    x = [a.requires_grad_(True) for a in t.values()]

    def go():
        out = mb.block_norm(x[0], x[1], x[2], residual=x[3], scale=x[4])
        return [*out, *torch.autograd.grad(out, x, (dy, dh))]

    first = go()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = go()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals(cuda):
    import mingru_b200 as mb

    x, w = torch.zeros(4, 24, device=cuda), torch.ones(24, device=cuda)
    for args, kw, match in [
        ((x, w), dict(groups=5), "groups"),
        ((x, w), dict(groups=0), "groups"),
        ((x, w), dict(scale=w), "residual"),
        ((x, w), dict(residual=x[:2]), "residual"),
        ((x, w), dict(residual=x.bfloat16()), "residual"),
        ((x, w), dict(gate=x[:, :8]), "gate"),
        ((x, w[:8]), {}, "weight"),
        ((x, w, w[:8]), {}, "bias"),
        ((x, w, w.bfloat16()), {}, "bias"),
        ((x, w.bfloat16()), {}, "weight"),
        ((x.double(), w.double()), {}, "not supported"),
        ((x.cpu(), w.cpu()), {}, "CUDA"),
        ((x, w.cpu()), {}, "CUDA"),
        ((torch.zeros(2, 16385, device=cuda), torch.ones(16385, device=cuda)), {}, "MGS_UNSUPPORTED"),
        ((torch.zeros((), device=cuda), w), {}, "D >= 1"),
    ]:
        with pytest.raises(ValueError, match=match):
            mb.block_norm(*args, **kw)
    a = torch.randn(3, 24, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="second-order"):
        torch.autograd.grad(mb.block_norm(a, w).sum(), a, create_graph=True)


def test_under_compile(cuda):
    """torch.compile sees opaque ops, forward and backward."""
    import mingru_b200 as mb

    t, dy, dh = inputs((20,), 96, torch.float32, torch.float32, cuda, ("bias", "residual", "scale", "gate"), 7)
    x = [a.requires_grad_(True) for a in t.values()]

    def run(x, w, b, r, s, g):
        return mb.block_norm(x, w, b, residual=r, scale=s, gate=g, groups=4)

    got, want = torch.compile(run, backend="aot_eager", fullgraph=True)(*x), run(*x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(torch.autograd.grad(got, x, (dy, dh)), torch.autograd.grad(want, x, (dy, dh))):
        assert torch.equal(a, b)
