"""Linear attention with per-head decay: the kernels against the recurrence in
float64 (token by token, gradients by autograd through it), against
differences of their own forward, and their refusals.

Tolerances (2-norm of the error over 2-norm of the result, and the largest
error over |result| + 8 rms), from the arithmetic:

* fp32 results: operands are exact to 2^-24 and a result sums at most 256
  fp32 roundings of random sign in a chunk (16 * 2^-24 ~ 1e-6) and as many
  joins of chunks again: 4e-6. dlog_gamma is a difference of sums over a chunk
  that are up to ten times its size: 4e-5.
* bf16 results: one rounding of the result and one of the masked products or
  the state it is made of, 2^-9 each at most: 2^-8. fp16: 2^-11 each: 2^-10.
* differences: the forward is linear in each of Q, K, V and H0, so only its
  own rounding remains (a step of 1 against 4e-6 of the result: 1e-4 with the
  cancellation of a random direction); for log_gamma the cubic term of a
  central step of 1e-2 is below 1e-4 of the slope, the rounding 4e-6 / 1e-2:
  2e-3.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 4e-6, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-10}
DLG = 4e-5


def close(got, ref, tol, name):
    got, ref = got.detach().double(), ref.detach().double()
    assert got.shape == ref.shape, name
    if not ref.numel():
        return
    d, rms = (got - ref).abs(), ref.square().mean().sqrt()
    assert torch.isfinite(got).all(), name
    if rms == 0:
        assert d.max() == 0, name
        return
    rel, big = (d.norm() / ref.norm()).item(), (d / (ref.abs() + 8 * rms)).max().item()
    assert rel <= tol and big <= tol, f"{name}: rel {rel:.3g}, max {big:.3g} (tolerance {tol:.3g})"


def recurrence(Q, K, V, lg, H0):
    """Token by token in float64."""
    B, H, T, dk = Q.shape
    S = torch.zeros(B, H, dk, V.shape[3], dtype=torch.float64, device=Q.device) if H0 is None else H0
    g = lg.exp().expand(B, H, T)
    ys = []
    for t in range(T):
        S = g[:, :, t, None, None] * S + K[:, :, t, :, None] * V[:, :, t, None, :]
        ys.append((Q[:, :, t, None, :] @ S).squeeze(-2))
    y = torch.stack(ys, 2) if ys else torch.zeros_like(V)
    return y, S


def decays(kind, B, H, T, gen, dev):
    r = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    if kind == "token":
        return -torch.nn.functional.softplus(r(B, H, T) - 3)
    if kind == "head":
        return -torch.logspace(-4, -0.3, H, device=dev).view(1, H, 1)
    if kind == "none":
        return torch.zeros(1, 1, 1, device=dev)
    if kind == "strong":  # from forgetting at once to below what fp32 holds
        return -(5 * r(B, H, T)).exp()
    if kind == "resets":  # documents packed together, one starting at the first token
        lg = -torch.nn.functional.softplus(r(B, H, T) - 3)
        cut = torch.rand(B, 1, T, device=dev, generator=gen) < 0.02
        cut[:, :, 0] = True
        return torch.where(cut, torch.full_like(lg, -float("inf")), lg)
    if kind == "wiped":  # no token sees another
        return torch.full((B, H, T), -float("inf"), device=dev)
    raise KeyError(kind)


def inputs(B, H, T, dk, dv, dtype, dev, kind="token", h0=True, layout="bhtd", seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731

    def seq(d, scale=1.0):
        if layout == "bhtd":
            return (r(B, H, T, d) * scale).to(dtype)
        if layout == "bthd":
            return (r(B, T, H, d) * scale).to(dtype).transpose(1, 2)
        # one projection sliced into heads, at offsets that are not 16-byte aligned
        return (r(B, T, H, d + 3) * scale).to(dtype).transpose(1, 2)[..., 1:d + 1]

    Q, K, V, dy = seq(dk, dk**-0.5), seq(dk, dk**-0.5), seq(dv), seq(dv)
    lg = decays(kind, B, H, T, gen, dev)
    H0 = r(B, H, dk, dv) if h0 else None
    return Q, K, V, lg, H0, dy, r(B, H, dk, dv)


def check(dev, B, H, T, dk, dv, dtype, **kw):
    import mingru_b200 as mb

    Q, K, V, lg, H0, dy, dH = inputs(B, H, T, dk, dv, dtype, dev, **kw)
    leaves = [t for t in (Q, K, V, lg, H0) if t is not None]
    own = [t.detach().requires_grad_(True) for t in leaves]
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    args = lambda x: x if H0 is not None else [*x, None]  # noqa: E731
    y, HT = mb.linear_attention(*args(own))
    ry, rH = recurrence(*args(ref))
    assert y.dtype == dtype and HT.dtype == torch.float32
    tol = TOL[dtype]
    close(y, ry, tol, "y")
    close(HT, rH, TOL[torch.float32], "H_T")
    with torch.no_grad():  # the call without a graph is the same computation
        y2, HT2 = mb.linear_attention(*args(own))
    assert torch.equal(y2, y) and torch.equal(HT2, HT)
    got = torch.autograd.grad((y, HT), own, (dy, dH), allow_unused=True)
    want = torch.autograd.grad((ry, rH), ref, (dy.double(), dH.double()))
    mb.raise_device_error(dev)
    for n, a, b, t in zip(("dQ", "dK", "dV", "dlg", "dH0"), got, want, (tol, tol, tol, DLG, TOL[torch.float32])):
        b = torch.nan_to_num(b) if n == "dlg" else b  # 0 * inf of the reference at a wipe
        close(a, b, t, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 2, 127, 128, 129, 300])
def test_lengths(cuda, T, dtype):
    check(cuda, 2, 3, T, 64, 64, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dk,dv", [(1, 1), (5, 3), (16, 32), (33, 40), (64, 8), (40, 72), (128, 128), (96, 65),
                                   (130, 200)])
def test_head_sizes(cuda, dk, dv, dtype):
    check(cuda, 1, 2, 200, dk, dv, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["token", "head", "none", "strong", "resets", "wiped"])
def test_decays(cuda, kind, dtype):
    check(cuda, 2, 2, 333, 64, 64, dtype, kind=kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["bthd", "slice"])
def test_layouts(cuda, layout, dtype):
    check(cuda, 2, 3, 150, 64, 48, dtype, layout=layout, h0=False)
    if dtype == torch.bfloat16:
        check(cuda, 2, 3, 150, 104, 128, dtype, layout=layout)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_one_long_sequence(cuda, dtype, d):
    """One (batch, head): every chunk is a segment of its own or shares one."""
    check(cuda, 1, 1, 2050, d, d, dtype, kind="head")
    check(cuda, 1, 2, 2050, d, d, dtype, kind="resets", h0=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_heads(cuda, dtype):
    """More (batch, head) pairs than CTAs: one segment, chunks in order."""
    check(cuda, 50, 7, 260, 32, 32, dtype)


def test_several_chunks_to_a_segment(cuda):
    check(cuda, 8, 8, 1300, 64, 64, torch.bfloat16)
    check(cuda, 8, 8, 1300, 16, 16, torch.float32, kind="resets")


def test_decay_late_in_a_strong_chunk(cuda):
    """Spans stay exact where the sums before them are large."""
    import mingru_b200 as mb

    Q, K, V, _, H0, _, _ = inputs(1, 1, 256, 64, 64, torch.float32, cuda)
    lg = torch.cat([torch.full((64,), -80.0), torch.full((64,), -0.01)] * 2).to(cuda).view(1, 1, 256)
    y, HT = mb.linear_attention(Q, K, V, lg, H0)
    ry, rH = recurrence(Q.double(), K.double(), V.double(), lg.double(), H0.double())
    close(y, ry, TOL[torch.float32], "y")
    close(HT, rH, TOL[torch.float32], "H_T")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_no_tokens(cuda, dtype):
    import mingru_b200 as mb

    Q = torch.zeros(2, 3, 0, 16, dtype=dtype, device=cuda, requires_grad=True)
    V = torch.zeros(2, 3, 0, 24, dtype=dtype, device=cuda)
    H0 = torch.randn(2, 3, 16, 24, device=cuda, requires_grad=True)
    y, HT = mb.linear_attention(Q, Q, V, torch.zeros(2, 3, 0, device=cuda), H0)
    assert y.shape == (2, 3, 0, 24) and torch.equal(HT, H0)
    g = torch.autograd.grad(HT.sum(), H0)[0]
    assert torch.equal(g, torch.ones_like(g))
    _, HT = mb.linear_attention(Q, Q, V, torch.zeros(2, 3, 0, device=cuda))
    assert not HT.any()
    E = torch.zeros(0, 3, 5, 16, dtype=dtype, device=cuda)
    y, HT = mb.linear_attention(E, E, E, torch.zeros(0, 3, 5, device=cuda))
    assert y.shape == (0, 3, 5, 16) and HT.shape == (0, 3, 16, 16)


@pytest.mark.parametrize("d", [64, 80])
def test_differences(cuda, d):
    """Directional derivatives of the kernel's own forward."""
    import mingru_b200 as mb

    Q, K, V, lg, H0, dy, dH = inputs(2, 2, 200, d, d, torch.float32, cuda, seed=3)
    x = [t.requires_grad_(True) for t in (Q, K, V, lg, H0)]
    loss = lambda a: sum((o.double() * w.double()).sum() for o, w in zip(mb.linear_attention(*a), (dy, dH)))  # noqa: E731
    grads = torch.autograd.grad(loss(x), x)
    gen = torch.Generator(device=cuda).manual_seed(4)
    for i, (g, n) in enumerate(zip(grads, ("Q", "K", "V", "log_gamma", "H0"))):
        step, tol = (1e-2, 2e-3) if n == "log_gamma" else (1.0, 1e-4)
        v = torch.randn(x[i].shape, device=cuda, generator=gen)
        with torch.no_grad():
            up, down = ([t + s * v if j == i else t for j, t in enumerate(x)] for s in (step, -step))
            diff = (loss(up) - loss(down)) / (2 * step)
        want = (g.double() * v.double()).sum()
        scale = g.double().norm() * v.double().norm()
        assert abs(diff - want) <= tol * scale, n


def test_parts_of_a_sequence(cuda):
    """A sequence in two calls, the state handed on, is the sequence in one."""
    import mingru_b200 as mb

    Q, K, V, lg, H0, _, _ = inputs(2, 2, 400, 64, 64, torch.float32, cuda)
    y, HT = mb.linear_attention(Q, K, V, lg, H0)
    cut = lambda a, b: [t[:, :, a:b] for t in (Q, K, V, lg)]  # noqa: E731
    y1, H1 = mb.linear_attention(*cut(0, 150), H0)
    y2, H2 = mb.linear_attention(*cut(150, 400), H1)
    close(torch.cat([y1, y2], 2), y.double(), 2 * TOL[torch.float32], "y")
    close(H2, HT.double(), 2 * TOL[torch.float32], "H_T")


def test_another_stream_and_repeats(cuda):
    """The same bits on every run, and on a stream of the caller's."""
    import mingru_b200 as mb

    Q, K, V, lg, H0, dy, dH = inputs(4, 4, 1000, 64, 64, torch.bfloat16, cuda)
    x = [t.requires_grad_(True) for t in (Q, K, V, lg, H0)]

    def go():
        out = mb.linear_attention(*x)
        return [*out, *torch.autograd.grad(out, x, (dy, dH))]

    first = go()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = go()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_partial_gradients(cuda):
    """Only one of the outputs has a gradient; expanded ones are read as they are."""
    import mingru_b200 as mb

    Q, K, V, lg, H0, _, dH = inputs(1, 2, 140, 32, 32, torch.float32, cuda)
    x = [t.requires_grad_(True) for t in (Q, K, V, lg, H0)]
    r = [t.detach().double().requires_grad_(True) for t in x]
    got = torch.autograd.grad(mb.linear_attention(*x)[0].sum(), x)
    want = torch.autograd.grad(recurrence(*r)[0].sum(), r)
    for n, a, b in zip(("dQ", "dK", "dV", "dlg", "dH0"), got, want):
        close(a, b, DLG if n == "dlg" else TOL[torch.float32], n)
    got = torch.autograd.grad((mb.linear_attention(*x)[1] * dH).sum(), x[1:])
    want = torch.autograd.grad((recurrence(*r)[1] * dH.double()).sum(), r[1:])
    for n, a, b in zip(("dK", "dV", "dlg", "dH0"), got, want):
        close(a, b, DLG if n == "dlg" else TOL[torch.float32], n)


def test_rows_past_2_31_elements(cuda):
    """Offsets into a large buffer are 64-bit: the last rows of a strided view."""
    import mingru_b200 as mb

    T, stride = 130, 1 << 24  # rows 16.8 million elements apart: the last past 2^31
    buf = torch.empty(T * stride, dtype=torch.bfloat16, device=cuda)
    V = torch.randn(1, 1, T, 8, device=cuda).bfloat16()
    view = torch.as_strided(buf, (1, 1, T, 8), (0, 0, stride, 1))
    view.copy_(V)
    Q, K, _, lg, _, _, _ = inputs(1, 1, T, 8, 8, torch.bfloat16, cuda)
    y, HT = mb.linear_attention(Q, K, view, lg)
    y2, HT2 = mb.linear_attention(Q, K, V, lg)
    assert torch.equal(y, y2) and torch.equal(HT, HT2)


def test_refusals(cuda):
    import mingru_b200 as mb

    z = lambda *s, **k: torch.zeros(*s, device=cuda, **k)  # noqa: E731
    Q, lg = z(1, 2, 5, 8), z(1, 2, 5)
    for bad, match in [
        ((z(2, 5, 8), Q, Q, lg), "4-D"),
        ((Q, z(1, 2, 5, 9), Q, lg), "shapes disagree"),
        ((Q, Q, z(1, 2, 6, 8), lg), "shapes disagree"),
        ((z(1, 2, 5, 0), z(1, 2, 5, 0), Q, lg), "shapes disagree"),
        ((Q, Q, Q, z(3, 2, 5)), "broadcast"),
        ((Q, Q, Q, lg, z(1, 2, 8, 9)), "H0"),
        ((Q, Q, Q.bfloat16(), lg), "share a dtype"),
        ((Q.double(), Q.double(), Q.double(), lg), "not supported"),
        ((Q, Q, Q, lg.long()), "floating point"),
        ((Q.cpu(), Q.cpu(), Q.cpu(), lg.cpu()), "CUDA"),
        ((Q, Q, Q, lg.cpu()), "CUDA"),
    ]:
        with pytest.raises(ValueError, match=match):
            mb.linear_attention(*bad)
    q = torch.randn(1, 2, 5, 8, device=cuda, requires_grad=True)
    y, _ = mb.linear_attention(q, q, q, lg)
    with pytest.raises(RuntimeError, match="second-order"):
        torch.autograd.grad(y.sum(), q, create_graph=True)


def test_c_entry_refuses(cuda):
    import ctypes

    from mingru_b200 import _lib

    lib = _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    s = (ctypes.c_int64 * 15)(*([0] * 15))
    x = torch.zeros(1024, device=cuda)
    p = x.data_ptr()
    call = lambda B, H, T, dk, dv, code, ws=None, n=0, saved=None: lib.mgs_linear_attn_fwd(  # noqa: E731
        p, p, p, p, None, p, p, saved, s, B, H, T, dk, dv, code, ws, n, st)
    name = lambda r: _lib.STATUS_NAMES[r]  # noqa: E731
    assert name(call(-1, 1, 1, 8, 8, 0)) == "MGS_BAD_SHAPE"
    assert name(call(1, 1, 1, 0, 8, 0)) == "MGS_BAD_SHAPE"
    assert name(call(1, 1, 1, 8, 8, 7)) == "MGS_BAD_DTYPE"
    assert name(call(1, 1, 1, 8, 129, 1)) == "MGS_UNSUPPORTED"
    assert name(call(1, 1, 1, 130, 8, 0)) == "MGS_WORKSPACE_TOO_SMALL"
    assert name(call(1, 1, 1, 129, 8, 1)) == "MGS_UNSUPPORTED"
    assert name(call(1, 1, 1000, 8, 8, 0)) == "MGS_WORKSPACE_TOO_SMALL"
    assert name(call(1, 1, 1, 8, 8, 0, saved=p + 4)) == "MGS_BAD_ALIGNMENT"
    assert name(call(0, 1, 5, 8, 8, 0)) == "MGS_OK"
    assert lib.mgs_linear_attn_saved_size(1, 1, 128, 129, 8, 1) == 0


def test_under_compile(cuda):
    """torch.compile sees opaque ops, forward and backward."""
    import mingru_b200 as mb

    Q, K, V, lg, H0, dy, dH = inputs(1, 2, 150, 32, 32, torch.float32, cuda)
    x = [t.requires_grad_(True) for t in (Q, K, V, lg, H0)]
    f = torch.compile(lambda *a: mb.linear_attention(*a), backend="aot_eager", fullgraph=True)
    got = f(*x)
    want = mb.linear_attention(*x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(torch.autograd.grad(got, x, (dy, dH)), torch.autograd.grad(want, x, (dy, dH))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 5, 33, 128, 200, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_first_token_without_a_state_has_no_decay_gradient(T, dtype):
    """dlog_gamma_0 = gamma_0 <H0, dS_0>: exactly zero when nothing enters, not what sums cancel to."""
    import mingru_b200 as mb

    g = torch.Generator(device="cuda").manual_seed(T)
    q, k, v, dy = (torch.randn(2, 3, T, 40, device="cuda", generator=g).to(dtype) for _ in range(4))
    lg = (-0.2 * torch.rand(2, 3, T, device="cuda", generator=g)).requires_grad_(True)
    y, H = mb.linear_attention(q, k, v, lg)
    (dlg,) = torch.autograd.grad((y, H), (lg,), (dy, torch.ones_like(H)))
    assert dlg[..., 0].abs().max().item() == 0.0


@pytest.mark.parametrize("T", [260, 500, 1000])
def test_decay_gradient_of_a_short_memory(T):
    """A decay of a few tokens: dlog_gamma_t is a sum over few pairs, and is as exact as these.

    R_ij = e^{c_i - c_j} (q_i . k_j)(dy_i . v_j), each within 2^-19 of its size (products of 64 in fp32,
    factors within some 2^-21); a token takes the pairs of 16 tokens' rows and columns at most twice:
    within 32 * 2 * 2^-19 of the largest row's or column's sum of sizes.
    """
    import mingru_b200 as mb

    g = torch.Generator(device="cuda").manual_seed(T)
    q, k, v, dy = (torch.randn(2, 2, T, 64, device="cuda", generator=g).bfloat16() for _ in range(4))
    lg = torch.full((2, 2, T), -0.2, device="cuda", requires_grad=True)
    y, _ = mb.linear_attention(q, k, v, lg)
    (dlg,) = torch.autograd.grad(y, (lg,), dy)
    qd, kd, vd, dyd = (t.double() for t in (q, k, v, dy))
    i = torch.arange(T, device="cuda")
    D = torch.where(i[:, None] >= i, torch.exp(-0.2 * (i[:, None] - i).clamp_min(0).double()), 0.0)
    R = D * (qd @ kd.mT) * (dyd @ vd.mT)
    # over pairs i >= t > j: the suffix over rows of the prefix over columns before t
    before = torch.cat((torch.zeros_like(R[..., :1]), R.cumsum(-1)[..., :-1]), -1)
    ref = torch.stack([before[..., t:, t].sum(-1) for t in range(T)], -1)
    most = torch.maximum(R.abs().sum(-1).amax(), R.abs().sum(-2).amax())
    assert (dlg.double() - ref).abs().max() <= 64 * 2**-19 * most
