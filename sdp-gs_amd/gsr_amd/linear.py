"""Fused matrix products on libgsr (include/gsr_linear.h): what a feature head is made of.

  fused_linear(x, weight, bias, activation=, residual=)   act(x W^T + b) + r
  gated_linear(x, gate_weight, up_weight, gate_bias, up_bias, activation=)
                                                act(x Wg^T + bg) * (x Wu^T + bu)

Bias, activation and residual (or the product of the two halves) are in the matrix product's
epilogue: one launch, two where weights are laid out first or a long sum is cut into ranges.  The
backward keeps nothing but the inputs: it forms the pre-activations again, in 32 bits, in the
product that writes their gradients -- cheaper than storing and reading them back at a head's
widths, and free of their rounding.  float32, float16 and bfloat16 (one type per call); sums and
activations in 32 bits, every result rounded once, 16-bit gradients before the activation rounded
for the products that follow (their sums, the bias gradients, are not made from rounded ones).
Results do not depend on timing.  Reverse mode only: a tangent (torch.autograd.forward_ad) is
refused.  No CPU path.

A rendered feature image [C,H,W] goes in as it lies: ``fused_linear(image.reshape(C, -1).t(), W)``
reads the channel-major memory in place.

In a captured graph take gradients with ``torch.autograd.grad``, or ``backward()`` with leaves
that no eager graph is alive for (autograd joins a leaf's stream of first use with the capture).
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}  # GSR_ACT_*; gelu is the erf form
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # GSR_F32 / F16 / BF16


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed with status {rc}")


def _fits(t, shape, x):
    return t is None or (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype is x.dtype
                         and t.device == x.device)


def _refuse(x, weight, weight_name, others, activation):
    """Say what is wrong with a call that the kernels do not take (before any GPU work)."""
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError(f"x and {weight_name} must be tensors")
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError(f"x must be [..., K] and {weight_name} [N, K]")
    N, K = weight.shape
    if N < 1 or K < 1:
        raise ValueError(f"{weight_name} [N, K] must not be empty")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
    for name, t, shape in [("x", x, x.shape[:-1] + (K,)), (weight_name, weight, (N, K))] + others(N, K):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
        if t.dtype != x.dtype:
            raise ValueError(f"{name} must have x's type {x.dtype}, not {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} must be on x's device {x.device}, not {t.device}")
    if x.dtype not in DTYPES:
        raise ValueError(f"float32, float16 or bfloat16 expected, not {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError("gsr fused products run on HIP tensors only (no CPU path)")
    raise ValueError("gsr fused products: arguments not supported")


def _base_fits(x, weight, activation):
    return (isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor) and x.is_cuda
            and x.dtype in DTYPES and activation in ACTIVATIONS and weight.dim() == 2
            and x.dim() > 0 and x.shape[-1] == weight.shape[1] and weight.numel() > 0
            and weight.dtype is x.dtype and weight.device == x.device)


def _rows(t, n):
    """t [..., n] as a [M, n] matrix whose rows are contiguous (a copy only if it has to be)."""
    m = t.reshape(-1, n) if t.dim() != 2 else t
    row, col = m.stride()
    if (col != 1 and n > 1) or (row < n and m.shape[0] > 1):
        m = m.contiguous()
    return m


def _row_stride(m):
    """The distance between rows (a single row's stride means nothing)."""
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _x_matrix(x, K):
    """x as (matrix, row stride, column stride): channel-major memory is taken as it lies."""
    if x.dim() == 2:
        row, col = x.stride()
        if col == 1 and row >= K:
            return x, row, 1
        if row == 1 and K > 1 and x.shape[0] > 1 and col >= x.shape[0]:
            return x, 1, col
    m = _rows(x, K)
    return m, _row_stride(m), 1


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(weight, bias):
    return 1 if weight else 2 if bias else 0  # GSR_NEED_DW / GSR_NEED_DB


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _refuse_tangents(*tensors):
    """A dual tensor needs no gradient, so nothing else would notice that its tangent is lost."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None
           for t in tensors):
        raise NotImplementedError("gsr fused products have no forward-mode derivative")


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _weight_pair(gate, up, K):
    """Both weights as rows of one distance."""
    wg, wu = _rows(gate, K), _rows(up, K)
    if _row_stride(wg) != _row_stride(wu):
        wg, wu = wg.contiguous(), wu.contiguous()
    return wg, wu


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        N, K = weight.shape
        xm, x_row, x_col = _x_matrix(x, K)
        M = xm.shape[0]
        w = _rows(weight, K)
        b = None if bias is None else bias.contiguous()
        r = None if residual is None else _rows(residual, N)
        y = x.new_empty(x.shape[:-1] + (N,))
        if M:
            L = _lib.load()
            scratch = _scratch(L.gsr_linear_scratch_bytes(DTYPES[x.dtype], M, K, N), x.device)
            with _lib.on_device(x.device):
                _check(L.gsr_linear(
                    DTYPES[x.dtype], M, K, N, xm.data_ptr(), x_row, x_col, w.data_ptr(),
                    _row_stride(w), _ptr(b), _ptr(r), 0 if r is None else _row_stride(r), act,
                    y.data_ptr(), N, _ptr(scratch), _lib.raw_stream(x.device)), "gsr_linear")
        if ctx is not None:
            ctx.save_for_backward(xm, w, b)
            ctx.args = (x.shape, act)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        # what comes back may lie otherwise than what was saved (saved_tensors_hooks, save_on_cpu)
        xm, w, b = ctx.saved_tensors
        shape, act = ctx.args
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        (N, K), M = w.shape, xm.shape[0]
        xm, x_row, x_col = _x_matrix(xm, K)
        w, b = _rows(w, K), None if b is None else b.contiguous()
        kind, dev = xm.dtype, xm.device
        dx = torch.empty(shape, dtype=kind, device=dev) if need_x else None
        dw = torch.empty((N, K), dtype=kind, device=dev) if need_w else None
        db = torch.empty(N, dtype=kind, device=dev) if need_b else None
        if need_x or need_w or need_b:
            g = _rows(dy, N)
            L = _lib.load()
            scratch = _scratch(L.gsr_linear_backward_scratch_bytes(
                DTYPES[kind], M, K, N, act, _need(need_w, need_b)), dev)
            with _lib.on_device(dev):
                _check(L.gsr_linear_backward(
                    DTYPES[kind], M, K, N, xm.data_ptr(), x_row, x_col, w.data_ptr(),
                    _row_stride(w), _ptr(b), act, g.data_ptr(), _row_stride(g), _ptr(dx), _ptr(dw),
                    _ptr(db), _ptr(scratch), _lib.raw_stream(dev)), "gsr_linear_backward")
        return dx, dw, db, dy if need_r else None, None


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, gate_bias, up_bias, act):
        N, K = gate.shape
        xm = _rows(x, K)
        M = xm.shape[0]
        wg, wu = _weight_pair(gate, up, K)
        bg = None if gate_bias is None else gate_bias.contiguous()
        bu = None if up_bias is None else up_bias.contiguous()
        h = x.new_empty(x.shape[:-1] + (N,))
        if M:
            L = _lib.load()
            scratch = _scratch(L.gsr_gated_scratch_bytes(DTYPES[x.dtype], M, K, N), x.device)
            with _lib.on_device(x.device):
                _check(L.gsr_gated(
                    DTYPES[x.dtype], M, K, N, xm.data_ptr(), _row_stride(xm), wg.data_ptr(),
                    wu.data_ptr(), _row_stride(wg), _ptr(bg), _ptr(bu), act, h.data_ptr(), N,
                    _ptr(scratch), _lib.raw_stream(x.device)), "gsr_gated")
        if ctx is not None:
            ctx.save_for_backward(xm, wg, wu, bg, bu)
            ctx.args = (x.shape, act)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        xm, wg, wu, bg, bu = ctx.saved_tensors
        shape, act = ctx.args
        need = ctx.needs_input_grad
        (N, K), M = wg.shape, xm.shape[0]
        xm, (wg, wu) = _rows(xm, K), _weight_pair(wg, wu, K)  # they may lie otherwise than when saved
        bg, bu = (None if b is None else b.contiguous() for b in (bg, bu))
        kind, dev = xm.dtype, xm.device
        need_w, need_b = need[1] or need[2], need[3] or need[4]
        dx = torch.empty(shape, dtype=kind, device=dev) if need[0] else None
        dw = torch.empty((2, N, K), dtype=kind, device=dev) if need_w else None
        db = torch.empty((2, N), dtype=kind, device=dev) if need_b else None
        if need[0] or need_w or need_b:
            g = _rows(dh, N)
            L = _lib.load()
            scratch = _scratch(L.gsr_gated_backward_scratch_bytes(
                DTYPES[kind], M, K, N, _need(need_w, need_b)), dev)
            with _lib.on_device(dev):
                _check(L.gsr_gated_backward(
                    DTYPES[kind], M, K, N, xm.data_ptr(), _row_stride(xm), wg.data_ptr(),
                    wu.data_ptr(), _row_stride(wg), _ptr(bg), _ptr(bu), act, g.data_ptr(),
                    _row_stride(g), _ptr(dx), _ptr(dw), _ptr(db), _ptr(scratch),
                    _lib.raw_stream(dev)), "gsr_gated_backward")
        return (dx, dw[0] if need[1] else None, dw[1] if need[2] else None,
                db[0] if need[3] else None, db[1] if need[4] else None, None)


def fused_linear(x, weight, bias=None, *, activation="none", residual=None):
    """activation(x @ weight.T + bias) + residual.  x [..., K], weight [N, K], bias [N], residual
    [..., N] (the result's shape); differentiable once in each of them."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias, residual)
    if not (_base_fits(x, weight, activation) and _fits(bias, weight.shape[:1], x)
            and _fits(residual, x.shape[:-1] + weight.shape[:1], x)):
        _refuse(x, weight, "weight", lambda N, K: [
            ("bias", bias, (N,)), ("residual", residual, x.shape[:-1] + (N,))], activation)
    if not _wants_grad(x, weight, bias, residual):
        return _Linear.forward(None, x, weight, bias, residual, ACTIVATIONS[activation])
    return _Linear.apply(x, weight, bias, residual, ACTIVATIONS[activation])


def gated_linear(x, gate_weight, up_weight, gate_bias=None, up_bias=None, *, activation="silu"):
    """activation(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias), both products in
    one pass over x.  x [..., K], weights [N, K], biases [N]; differentiable once in each."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, gate_weight, up_weight, gate_bias, up_bias)
    if not (_base_fits(x, gate_weight, activation) and up_weight is not None
            and _fits(up_weight, gate_weight.shape, x) and _fits(gate_bias, gate_weight.shape[:1], x)
            and _fits(up_bias, gate_weight.shape[:1], x)):
        if up_weight is None:
            raise TypeError("up_weight must be a tensor")
        _refuse(x, gate_weight, "gate_weight", lambda N, K: [
            ("up_weight", up_weight, (N, K)), ("gate_bias", gate_bias, (N,)),
            ("up_bias", up_bias, (N,))], activation)
    if not _wants_grad(x, gate_weight, up_weight, gate_bias, up_bias):
        return _Gated.forward(None, x, gate_weight, up_weight, gate_bias, up_bias,
                              ACTIVATIONS[activation])
    return _Gated.apply(x, gate_weight, up_weight, gate_bias, up_bias, ACTIVATIONS[activation])
