"""Fused per-token recurrence updates behind the mixers' ``step()``.

Each function takes one token's pre-activations (the outputs of the mixer's
linear projections) and the previous state and returns the next state (and,
for the delta rule, the readout) from one kernel of ``libmingru_scan.so``,
where the reference runs a chain of small torch ops per step
(``MinGRU.step`` ... ``DeltaMinGRU.step``, reference ``src/mingru/
min_gru.py:1399-1448, 1858-1901, 2316-2359, 2776-2818, 3611-3688``). No
autograd: ``step()`` is an inference path (``torch.no_grad`` in the
reference too). The arithmetic is fp32 whatever the storage dtype.
"""

from __future__ import annotations

import torch

from . import _lib
from .scan_ops import _dtype_code, _require_cuda, on_device, raw_stream

__all__ = ["mingru_step", "signed_step", "rotation_step", "givens_step", "delta_step",
           "linear_attention_step"]


def _prep(op, *ts, like):
    """CUDA, one dtype, contiguous (None passes through)."""
    present = [t for t in ts if t is not None]
    _require_cuda(op, *present)
    if any(t.dtype != like.dtype for t in present):
        raise ValueError(f"{op}: all inputs must share the dtype {like.dtype}")
    return [None if t is None else t.contiguous() for t in ts]


def _p(t):
    return None if t is None else t.data_ptr()


def _run(op, fn, dev, *args):
    with on_device(dev):
        st = fn(*args, raw_stream(dev))
    _lib.check(st, op)


def mingru_step(k, xh, h_prev, gamma=None):
    """``h = gamma (1 - sigmoid(k)) h_prev + sigmoid(k) g(xh)`` (all ``(B, D)``)."""
    op = "mingru_step"
    k, xh, h_prev, gamma = _prep(op, k, xh, h_prev, gamma, like=k)
    h = torch.empty_like(h_prev)
    B, D = h.shape
    _run(op, _lib.load().mgs_mingru_step, k.device, _p(k), _p(xh), _p(h_prev), _p(gamma), _p(h),
         B, D, _dtype_code(op, k))
    return h


def signed_step(z, s, xh, h_prev, gamma=None, coupled=False):
    """``h = a h_prev + sigmoid(z) xh`` with ``a = gamma tanh(s)``, times
    ``1 - sigmoid(z)`` when coupled (all ``(B, D)``)."""
    op = "signed_step"
    z, s, xh, h_prev, gamma = _prep(op, z, s, xh, h_prev, gamma, like=z)
    h = torch.empty_like(h_prev)
    B, D = h.shape
    _run(op, _lib.load().mgs_signed_step, z.device, _p(z), _p(s), _p(xh), _p(h_prev), _p(gamma),
         int(bool(coupled)), _p(h), B, D, _dtype_code(op, z))
    return h


def rotation_step(theta, u, z, xh, h_prev, gamma=None):
    """Per 2-block: ``h = gamma R(theta) diag(1, tanh u) h_prev + sigmoid(z) xh``;
    ``theta``, ``u``, ``gamma`` ``(B, n)``; ``z``, ``xh``, ``h_prev`` ``(B, 2n)``."""
    op = "rotation_step"
    theta, u, z, xh, h_prev, gamma = _prep(op, theta, u, z, xh, h_prev, gamma, like=theta)
    h = torch.empty_like(h_prev)
    B, n = theta.shape
    _run(op, _lib.load().mgs_rotation_step, theta.device, _p(theta), _p(u), _p(z), _p(xh),
         _p(h_prev), _p(gamma), _p(h), B, n, _dtype_code(op, theta))
    return h


def givens_step(theta, z, xh, h_prev, gamma=None):
    """Per k-block: R brick-wall rounds of plane rotations, ``* gamma``, ``+
    sigmoid(z) xh``; ``theta`` ``(B, n, R, k/2)``, ``gamma`` ``(B, n)``,
    ``z``, ``xh``, ``h_prev`` ``(B, n k)``; k in {2, 4, ..., 64} (powers of 2)."""
    op = "givens_step"
    theta, z, xh, h_prev, gamma = _prep(op, theta, z, xh, h_prev, gamma, like=theta)
    h = torch.empty_like(h_prev)
    B, n, R, half = theta.shape
    _run(op, _lib.load().mgs_givens_step, theta.device, _p(theta), _p(z), _p(xh), _p(h_prev),
         _p(gamma), _p(h), B, n, R, 2 * half, _dtype_code(op, theta))
    return h


def delta_step(q, k, v, beta, H_prev, gamma=None):
    """One token of the delta rule per head: ``H <- gamma H``, then for each of
    the nh micro-steps ``H <- H + beta k (v - k^T H)^T``; readout ``y = H^T q``.
    ``q`` ``(B, H, dk)``, ``k`` ``(B, H, nh, dk)``, ``v`` ``(B, H, nh, dv)``,
    ``beta`` ``(B, H, nh)``, ``gamma`` ``(B, H)``, ``H_prev`` ``(B, H, dk, dv)``.
    Returns ``(y (B, H, dv), H)``."""
    op = "delta_step"
    q, k, v, beta, H_prev, gamma = _prep(op, q, k, v, beta, H_prev, gamma, like=q)
    B, nH, dk = q.shape
    nh, dv = k.shape[2], v.shape[3]
    H = torch.empty_like(H_prev)
    y = torch.empty(B, nH, dv, dtype=q.dtype, device=q.device)
    _run(op, _lib.load().mgs_delta_step, q.device, _p(q), _p(k), _p(v), _p(beta), _p(gamma),
         _p(H_prev), _p(y), _p(H), B, nH, nh, dk, dv, _dtype_code(op, q))
    return y, H


def linear_attention_step(q, k, v, log_gamma, H_prev, out=None):
    """One token of :func:`mingru_b200.linear_attention` per head:
    ``H = exp(log_gamma) H_prev + k v^T``; readout ``y = H^T q``. ``q``, ``k``
    ``(B, H, dk)``, ``v`` ``(B, H, dv)``, ``log_gamma`` ``(B, H)`` or
    broadcastable to it, ``H_prev`` ``(B, H, dk, dv)`` fp32 -- the state stays
    in fp32 whatever the inputs' dtype. The new state is written to ``out``
    where it is given (``H_prev`` itself for an update in place). Returns
    ``(y (B, H, dv), H)``."""
    op = "linear_attention_step"
    q, k, v = _prep(op, q, k, v, like=q)
    if q.ndim != 3 or k.shape != q.shape or v.ndim != 3 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"{op}: need q, k (B, n_heads, d_k) and v (B, n_heads, d_v); got "
                         f"q={tuple(q.shape)}, k={tuple(k.shape)}, v={tuple(v.shape)}")
    B, nH, dk = q.shape
    dv = v.shape[2]
    shape = (B, nH, dk, dv)
    for name, t in (("H_prev", H_prev), ("out", out)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32):
            raise ValueError(f"{op}: {name} must be a float32 tensor of shape {shape} (got "
                             f"{t.dtype}, {tuple(t.shape)})")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=q.device)
    elif not out.is_contiguous():
        raise ValueError(f"{op}: out must be contiguous")
    _require_cuda(op, q, log_gamma, H_prev, out)
    lg = log_gamma.float()
    if tuple(lg.shape) != shape[:2]:
        try:
            lg = torch.broadcast_to(lg, shape[:2])
        except RuntimeError:
            raise ValueError(f"{op}: log_gamma must broadcast to {shape[:2]} (got "
                             f"{tuple(lg.shape)})") from None
    H_prev = H_prev.contiguous()
    if 0 < abs(H_prev.data_ptr() - out.data_ptr()) < 4 * out.numel():
        H_prev = H_prev.clone()  # out lies over a part of it: in place is every element on itself
    y = torch.empty_like(v)
    _run(op, _lib.load().mgs_linear_attn_step, q.device, _p(q), _p(k), _p(v), _p(lg), lg.stride(0),
         lg.stride(1), _p(H_prev), _p(y), _p(out), B, nH, dk, dv, _dtype_code(op, q))
    return y, out
