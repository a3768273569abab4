"""The norms around a block, each one kernel (:func:`block_norm`).

Before a mixer or an MLP: the residual add, with a scale for the branch, and
the LayerNorm or RMS norm of the sum. After a mixer: the norm of each head's
channels and the gate. No counterpart in the reference, whose blocks run
torch's LayerNorm and adds (``min_gru.py:3698-3922``).
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .scan_ops import (_dense, _dtype_code, _ptr, _require_cuda, _traced, _wants_grad, _workspace, on_device,
                       raw_stream)

__all__ = ["block_norm"]

_OP = "block_norm"
MAX_GROUP = 16384  # channels of a group that the kernels take


def _rows(t: torch.Tensor | None, D: int):
    """``t`` as rows of D: (tensor that owns them, row stride)."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, D
    if t.stride(-1) == 1 or D == 1:
        # one stride from row to row over all the leading dimensions; one of size 1 has none that counts
        lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()) if n != 1]
        if all(s == inner * n for (_, s), (n, inner) in zip(lead, lead[1:])):
            return t, lead[-1][1] if lead else D
    return t.contiguous(), D


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device: int, rows: int, D: int, groups: int, code: int) -> int:
    """On a device, which must be current."""
    return _lib.load().mgs_block_norm_workspace_size(rows, D, groups, code)


def _dense_like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _codes(x, weight):
    return _dtype_code(_OP, x), _dtype_code(_OP, weight)


def _forward(x, weight, bias, residual, scale, gate, groups, eps, rms, save):
    with on_device(x.device):  # sizes are queried on the launch device
        D = x.shape[-1]
        rows = x.numel() // D
        (x, lx), (residual, lr), (gate, lg) = _rows(x, D), _rows(residual, D), _rows(gate, D)
        weight, bias, scale = (None if t is None else _dense(t) for t in (weight, bias, scale))
        y = _dense_like(x)
        h = torch.empty_like(y) if residual is not None else None
        stats = torch.empty(rows * groups * 3, dtype=torch.float32, device=x.device) if save else None
        code, wcode = _codes(x, weight)
        st = _lib.load().mgs_block_norm_fwd(
            _ptr(x), _ptr(residual), _ptr(gate), _ptr(weight), _ptr(bias), _ptr(scale), _ptr(y),
            _ptr(h), _ptr(stats),
            (ctypes.c_int64 * 3)(lx, lr, lg), rows, D, groups, int(rms), eps, code, wcode, raw_stream(x.device),
        )
        _lib.check(st, f"{_OP} forward")
        return y, h, stats


@torch.library.custom_op("mingru_b200::block_norm_fwd", mutates_args=())
def _block_norm_fwd(
    x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None,
    scale: torch.Tensor | None, gate: torch.Tensor | None, groups: int, eps: float, rms: bool,
    save: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    y, h, stats = _forward(x, weight, bias, residual, scale, gate, groups, eps, rms, save)
    return (y, x.new_empty(0) if h is None else h,
            x.new_empty(0, dtype=torch.float32) if stats is None else stats)


@_block_norm_fwd.register_fake
def _(x, weight, bias, residual, scale, gate, groups, eps, rms, save):
    y = x.new_empty(x.shape)
    h = x.new_empty(x.shape) if residual is not None else x.new_empty((0,))
    return y, h, x.new_empty((x.numel() // x.shape[-1] * groups * 3 if save else 0,), dtype=torch.float32)


def _gradients(x, weight, bias, residual, scale, gate, stats, dy, dh, groups, rms):
    lib = _lib.load()
    with on_device(x.device):  # sizes are queried on the launch device
        D = x.shape[-1]
        rows = x.numel() // D
        dy = dy.to(x.dtype)
        dh = None if dh is None else dh.to(x.dtype)
        (x, lx), (residual, lr), (gate, lg) = _rows(x, D), _rows(residual, D), _rows(gate, D)
        (dy, ly), (dh, lh) = _rows(dy, D), _rows(dh, D)
        weight, bias, scale = (None if t is None else _dense(t) for t in (weight, bias, scale))
        dx, dw = _dense_like(x), torch.empty_like(weight)
        dres, ds = (None, None) if scale is None else (torch.empty_like(dx), torch.empty_like(weight))
        db = None if bias is None else torch.empty_like(weight)
        dgate = None if gate is None else torch.empty_like(dx)
        code, wcode = _codes(x, weight)
        ws = _workspace(_workspace_bytes(x.device.index, rows, D, groups, code), x.device)
        st = lib.mgs_block_norm_bwd(
            _ptr(x), _ptr(residual), _ptr(gate), _ptr(weight), _ptr(bias), _ptr(scale), _ptr(stats),
            _ptr(dy), _ptr(dh), _ptr(dx), _ptr(dres), _ptr(dgate), _ptr(dw), _ptr(db), _ptr(ds),
            (ctypes.c_int64 * 5)(lx, lr, lg, ly, lh), rows, D, groups, int(rms), code, wcode, _ptr(ws),
            ws.numel(), raw_stream(x.device),
        )
        _lib.check(st, f"{_OP} backward")
        return dx, dw, db, dres, ds, dgate


@torch.library.custom_op("mingru_b200::block_norm_bwd", mutates_args=())
def _block_norm_bwd(
    x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None,
    scale: torch.Tensor | None, gate: torch.Tensor | None, stats: torch.Tensor, dy: torch.Tensor,
    dh: torch.Tensor | None, groups: int, rms: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    got = _gradients(x, weight, bias, residual, scale, gate, stats, dy, dh, groups, rms)
    return tuple(x.new_empty(0) if t is None else t for t in got)


@_block_norm_bwd.register_fake
def _(x, weight, bias, residual, scale, gate, stats, dy, dh, groups, rms):
    e = lambda on, t: t.new_empty(t.shape if on else (0,))  # noqa: E731
    return (e(True, x), e(True, weight), e(bias is not None, weight), e(scale is not None, x),
            e(scale is not None, weight), e(gate is not None, x))


def _setup(ctx, inputs, output):
    x, weight, bias, residual, scale, gate, groups, _eps, rms, _save = inputs
    ctx.save_for_backward(x, weight, bias, residual, scale, gate, output[2])
    ctx.groups, ctx.rms = groups, rms
    ctx.mark_non_differentiable(output[2], *(() if residual is not None else (output[1],)))
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, dh, _gstats=None, run=_block_norm_bwd):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{_OP} does not support second-order autograd (create_graph=True)")
    x, weight, bias, residual, scale, gate, stats = ctx.saved_tensors
    if dy is None and dh is None:
        return (None,) * 10
    if dy is None:
        dy = torch.zeros_like(x)
    dx, dw, db, dres, ds, dgate = run(x, weight, bias, residual, scale, gate, stats, dy,
                                      dh if residual is not None else None, ctx.groups, ctx.rms)
    return (dx, dw, db if bias is not None else None,
            None if residual is None else dx if scale is None else dres,
            ds if scale is not None else None, dgate if gate is not None else None, None, None, None, None)


torch.library.register_autograd("mingru_b200::block_norm_fwd", _backward, setup_context=_setup)


class _Eager(torch.autograd.Function):
    """The custom op's forward and backward without the dispatcher's Python layers."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, scale, gate, groups, eps, rms):
        y, h, stats = _forward(x, weight, bias, residual, scale, gate, groups, eps, rms, True)
        ctx.save_for_backward(x, weight, bias, residual, scale, gate, stats)
        ctx.groups, ctx.rms = groups, rms
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        return _backward(ctx, dy, dh, run=_gradients)[:9]


def block_norm(
    x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
    residual: torch.Tensor | None = None, scale: torch.Tensor | None = None,
    gate: torch.Tensor | None = None, groups: int = 1, eps: float = 1e-5, rms: bool = False,
):
    """Residual add, norm and gate over the last dimension, in one kernel.

    ``h = residual + scale * x`` (``h = x`` without a ``residual``; ``scale``
    ``(D,)`` only with one), the LayerNorm (``rms``: the RMS norm) of each of
    ``groups`` equal groups of channels, ``* weight + bias``, and ``*
    silu(gate)`` where there is a ``gate``. Returns ``y``, or ``(y, h)`` with a
    ``residual``: ``h`` is the residual stream that goes on.

    ``x``, ``residual`` and ``gate`` ``(..., D)`` share a shape and a dtype
    (fp32, bf16, fp16); ``weight``, ``bias`` and ``scale`` ``(D,)`` are in that
    dtype or in fp32. Arithmetic is fp32, the norm is taken of the unrounded
    sum, and outputs are rounded once. Rows may lie at any one stride. Groups
    of up to 16384 channels. Differentiable w.r.t. all tensors.
    """
    D = x.shape[-1] if x.ndim else 0
    if D < 1:
        raise ValueError(f"{_OP}: need x (..., D) with D >= 1 (got {tuple(x.shape)})")
    if groups < 1 or D % groups:
        raise ValueError(f"{_OP}: D={D} does not split into groups={groups}")
    if scale is not None and residual is None:
        raise ValueError(f"{_OP}: scale needs a residual")
    for name, t in (("residual", residual), ("gate", gate)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"{_OP}: {name} must have x's shape {tuple(x.shape)} and dtype {x.dtype} "
                             f"(got {tuple(t.shape)}, {t.dtype})")
    for name, t in (("weight", weight), ("bias", bias), ("scale", scale)):
        if t is not None and (tuple(t.shape) != (D,) or t.dtype != weight.dtype):
            raise ValueError(f"{_OP}: {name} must have shape {(D,)} and weight's dtype (got "
                             f"{tuple(t.shape)}, {t.dtype})")
    _dtype_code(_OP, x)
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{_OP}: weight must be {x.dtype} or float32 (got {weight.dtype})")
    given = [t for t in (x, weight, bias, residual, scale, gate) if t is not None]
    _require_cuda(_OP, *given)
    args = (x, weight, bias, residual, scale, gate, groups, float(eps), bool(rms))
    save = _wants_grad(*given)
    if _traced(*given):
        y, h, _ = _block_norm_fwd(*args, save)
    elif save:
        return _Eager.apply(*args)
    else:
        y, h, _ = _forward(*args, False)
    return y if residual is None else (y, h)
