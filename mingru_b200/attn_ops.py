"""Linear attention with a decay for each head, on the sm_100a kernels.

Per (batch, head), with ``gamma_t = exp(log_gamma_t)``::

    S_t = gamma_t S_{t-1} + k_t v_t^T        (d_k x d_v, fp32)
    y_t = S_t^T q_t

:func:`linear_attention` runs whole sequences (forward and backward);
``step_ops.linear_attention_step`` is the same recurrence for single tokens.
No counterpart in the reference, whose matrix-state mixer is the delta rule;
this is the recurrence that rule is without its correction, ``k^T S`` taken
from ``v``.

As the scan ops: CUDA tensors only, ``ValueError`` for what is outside the
kernels' envelope, ``torch.library`` custom ops for ``torch.compile``, no
second-order autograd.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .scan_ops import _dense, _dtype_code, _ptr, _require_cuda, _traced, _wants_grad, on_device, raw_stream

__all__ = ["linear_attention"]

_OP = "linear_attention"
_MAX_BF16 = 128  # d_k, d_v of a bf16 kernel call


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A dense last dimension; the other strides are the kernels' business."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like(t: torch.Tensor) -> torch.Tensor:
    """An output in the memory order of ``t``, one of the ``_rows``, its last dimension
    dense, as the kernels write it: PyTorch puts another one innermost where it is as
    dense in ``t`` (overlapping windows, heads)."""
    o = torch.empty_like(t)
    return o if o.stride(-1) == 1 or o.shape[-1] == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _strides(*ts: torch.Tensor):
    flat = []
    for t in ts:
        flat += t.stride()[:3]
    return (ctypes.c_int64 * len(flat))(*flat)


@functools.lru_cache(maxsize=1024)
def _sizes(device: int, B: int, H: int, T: int, dk: int, dv: int, code: int) -> tuple[int, int]:
    """(workspace bytes, saved floats) on a device, which must be current."""
    lib = _lib.load()
    return (lib.mgs_linear_attn_workspace_size(B, H, T, dk, dv, code),
            lib.mgs_linear_attn_saved_size(B, H, T, dk, dv, code) // 4)


def _saved_floats(B, H, T, dk, dv, dtype):
    """What ``mgs_linear_attn_saved_size`` asks for, of sizes that may be a compiler's
    symbols: a D x D state at every chunk of 128 tokens of every block of a head."""
    D = 128 if dtype == torch.bfloat16 and (dk > 64 or dv > 64) else 64
    return B * H * ((T + 127) // 128) * (-(-dk // D)) * (-(-dv // D)) * D * D


def _forward(Q, K, V, lg, H0, save):
    dev = Q.device
    with on_device(dev):  # sizes are queried on the launch device
        Q, K, V = _rows(Q), _rows(K), _rows(V)
        B, H, T, dk = Q.shape
        dv = V.shape[3]
        code = _dtype_code(_OP, Q)
        n, nsaved = _sizes(dev.index, B, H, T, dk, dv, code)
        y = _like(V)
        HT = lg.new_empty((B, H, dk, dv))  # log_gamma is fp32 and on the same device
        saved = lg.new_empty(nsaved) if save else None
        if T == 0:  # no token: the state passes through
            HT.zero_() if H0 is None else HT.copy_(H0)
            return y, HT, saved
        if H0 is not None:
            H0 = _dense(H0)
        ws = lg.new_empty(n // 4) if n else None
        st = _lib.load().mgs_linear_attn_fwd(
            Q.data_ptr(), K.data_ptr(), V.data_ptr(), lg.data_ptr(), _ptr(H0), y.data_ptr(), HT.data_ptr(),
            _ptr(saved), _strides(Q, K, V, lg, y), B, H, T, dk, dv, code, _ptr(ws), n,
            raw_stream(dev),
        )
        if st:
            _lib.check(st, f"{_OP} forward")
        return y, HT, saved


@torch.library.custom_op("mingru_b200::linear_attn_fwd", mutates_args=())
def _linear_attn_fwd(
    Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, lg: torch.Tensor, H0: torch.Tensor | None,
    save: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    y, HT, saved = _forward(Q, K, V, lg, H0, save)
    return y, HT, lg.new_empty(0) if saved is None else saved


@_linear_attn_fwd.register_fake
def _(Q, K, V, lg, H0, save):
    B, H, T, dk = Q.shape
    dv = V.shape[3]
    return (_like(_rows(V)), Q.new_empty((B, H, dk, dv), dtype=torch.float32),
            Q.new_empty((_saved_floats(B, H, T, dk, dv, Q.dtype) if save else 0,), dtype=torch.float32))


def _gradients(Q, K, V, lg, saved, dy, dHT, want_dH0):
    dev = Q.device
    with on_device(dev):  # sizes are queried on the launch device
        Q, K, V, dy = _rows(Q), _rows(K), _rows(V), _rows(dy.to(Q.dtype))
        B, H, T, dk = Q.shape
        dv = V.shape[3]
        code = _dtype_code(_OP, Q)
        dQ, dK, dV = _like(Q), _like(K), _like(V)
        dlg = lg.new_empty((B, H, T))
        dH0 = lg.new_empty((B, H, dk, dv)) if want_dH0 else None
        if dHT is not None:
            dHT = _dense(dHT.float())
        if T == 0:
            if want_dH0:
                dH0.zero_() if dHT is None else dH0.copy_(dHT)
            return dQ, dK, dV, dlg, dH0
        n, _ = _sizes(dev.index, B, H, T, dk, dv, code)
        ws = lg.new_empty(n // 4) if n else None
        st = _lib.load().mgs_linear_attn_bwd(
            Q.data_ptr(), K.data_ptr(), V.data_ptr(), lg.data_ptr(), saved.data_ptr(), dy.data_ptr(),
            _ptr(dHT), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), dlg.data_ptr(),
            _ptr(dH0), _strides(Q, K, V, lg, dy, dQ, dK, dV), B, H, T, dk, dv,
            code, _ptr(ws), n, raw_stream(dev),
        )
        if st:
            _lib.check(st, f"{_OP} backward")
        return dQ, dK, dV, dlg, dH0


@torch.library.custom_op("mingru_b200::linear_attn_bwd", mutates_args=())
def _linear_attn_bwd(
    Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, lg: torch.Tensor, saved: torch.Tensor,
    dy: torch.Tensor, dHT: torch.Tensor | None, want_dH0: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    *grads, dH0 = _gradients(Q, K, V, lg, saved, dy, dHT, want_dH0)
    return *grads, lg.new_empty(0) if dH0 is None else dH0


@_linear_attn_bwd.register_fake
def _(Q, K, V, lg, saved, dy, dHT, want_dH0):
    B, H, T, dk = Q.shape
    f32 = dict(dtype=torch.float32)
    return (_like(_rows(Q)), _like(_rows(K)), _like(_rows(V)), Q.new_empty((B, H, T), **f32),
            Q.new_empty((B, H, dk, V.shape[3]) if want_dH0 else (0,), **f32))


def _setup(ctx, inputs, output):
    Q, K, V, lg, H0, _save = inputs
    ctx.save_for_backward(Q, K, V, lg, output[2])
    ctx.has_h0 = H0 is not None
    ctx.mark_non_differentiable(output[2])
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, dHT, _gsaved=None, run=_linear_attn_bwd):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{_OP} does not support second-order autograd (create_graph=True)")
    if dy is None and dHT is None:
        return (None,) * 6
    Q, K, V, lg, saved = ctx.saved_tensors
    if dy is None:
        dy = torch.zeros_like(V)
    want = ctx.has_h0 and ctx.needs_input_grad[4]
    dQ, dK, dV, dlg, dH0 = run(Q, K, V, lg, saved, dy, dHT, want)
    return dQ, dK, dV, dlg, dH0 if want else None, None


torch.library.register_autograd("mingru_b200::linear_attn_fwd", _backward, setup_context=_setup)


class _Eager(torch.autograd.Function):
    """The custom op's forward and backward without the dispatcher, whose
    Python layers cost more than the kernels of a small call (a training step
    of an 8 x 8 x 1024 x 64 call: 390 us of host time with it)."""

    @staticmethod
    def forward(ctx, Q, K, V, lg, H0):
        y, HT, saved = _forward(Q, K, V, lg, H0, True)
        ctx.save_for_backward(Q, K, V, lg, saved)
        ctx.has_h0 = H0 is not None
        ctx.set_materialize_grads(False)
        return y, HT

    @staticmethod
    def backward(ctx, dy, dHT):
        return _backward(ctx, dy, dHT, run=_gradients)[:5]


def _run(Q, K, V, lg, H0):
    if Q.dtype == torch.bfloat16 and max(Q.shape[3], V.shape[3]) > _MAX_BF16:
        # the fp32 kernels take blocks of any number, added before the one rounding
        y, HT = _run(Q.float(), K.float(), V.float(), lg, H0)
        return y.to(Q.dtype), HT
    save = _wants_grad(Q, K, V, lg, H0)
    if _traced(Q, K, V, lg, H0):
        return _linear_attn_fwd(Q, K, V, lg, H0, save)[:2]
    if save:
        return _Eager.apply(Q, K, V, lg, H0)
    return _forward(Q, K, V, lg, H0, False)[:2]


def linear_attention(
    Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, log_gamma: torch.Tensor,
    H0: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay for each head; returns ``(y, H_T)``.

    ``Q``, ``K`` ``(B, n_heads, T, d_k)``, ``V`` ``(B, n_heads, T, d_v)`` in
    fp32, bf16 or fp16, ``log_gamma`` ``(B, n_heads, T)`` or broadcastable to
    it (``(1, n_heads, 1)``: one decay for each head), ``H0`` ``(B, n_heads,
    d_k, d_v)`` or ``None`` (zeros). ``y`` ``(B, n_heads, T, d_v)`` has the
    inputs' dtype and ``V``'s memory order; the state ``H_T`` is fp32.
    Differentiable w.r.t. all five tensors.

    Batch, head and time strides are free: views such as ``(B, T, n_heads,
    d).transpose(1, 2)`` or slices of one projection are read in place, and
    gradients come in the same order. Any ``d_k``, ``d_v`` (fp32 and fp16 heads
    wider than 64 run as blocks of 64 whose sums are fp32; bf16 heads wider
    than 128 run that way on fp32 copies) and any ``T``, 0 included.

    ``log_gamma <= 0``; ``-inf`` wipes the state before the token, which is how
    packed sequences are kept apart. A decay below ``2^-128`` counts as a wipe
    and its ``log_gamma`` gets no gradient. The products run on the tensor
    cores over chunks of 128 tokens, so a non-finite value spreads to earlier
    tokens of its own chunk (and to all later ones, as the recurrence has it).

    States, sums and the gradients of ``log_gamma`` and ``H0`` are fp32. In
    bf16 the masked products, and the states where they meet a query, are
    rounded once to bf16 before their second product: ``y`` and the gradients
    of Q, K and V are off by 0.0023 of their norm, where an fp32 computation
    rounded at the end is off by 0.0017. fp16 and fp32 inputs are held to 16
    and 24 bits throughout; pass those for more.
    """
    if Q.ndim != 4 or K.ndim != 4 or V.ndim != 4:
        raise ValueError(
            f"{_OP}: need 4-D Q, K (B, n_heads, T, d_k) and V (B, n_heads, T, d_v); got ranks "
            f"Q={Q.ndim}, K={K.ndim}, V={V.ndim}"
        )
    B, H, T, dk = Q.shape
    dv = V.shape[3]
    if K.shape != Q.shape or V.shape[:3] != Q.shape[:3] or dk < 1 or dv < 1:
        raise ValueError(
            f"{_OP}: shapes disagree: from Q={tuple(Q.shape)} expected K={tuple(Q.shape)} and "
            f"V={(B, H, T, 'd_v')}, d_k, d_v >= 1; got K={tuple(K.shape)}, V={tuple(V.shape)}"
        )
    if H0 is not None and tuple(H0.shape) != (B, H, dk, dv):
        raise ValueError(f"{_OP}: H0 must have shape {(B, H, dk, dv)} (got {tuple(H0.shape)})")
    lg = log_gamma
    if lg.shape != Q.shape[:3]:
        try:
            lg = torch.broadcast_to(lg, (B, H, T))
        except RuntimeError:
            raise ValueError(f"{_OP}: log_gamma must broadcast to {(B, H, T)} (got "
                             f"{tuple(lg.shape)})") from None
    _require_cuda(_OP, Q, K, V, lg, *(() if H0 is None else (H0,)))
    if K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise ValueError(f"{_OP}: Q, K and V must share a dtype")
    _dtype_code(_OP, Q)
    if not lg.is_floating_point() or not (H0 is None or H0.is_floating_point()):
        raise ValueError(f"{_OP}: log_gamma and H0 must be floating point")
    return _run(Q, K, V, lg.float(), None if H0 is None else H0.float())
