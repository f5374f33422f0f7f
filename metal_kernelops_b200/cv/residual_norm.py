"""Residual RMSNorm on the B200, with an int8 output for the int8 projections.

The pre-norm of a residual layer: the mixer's output joins the residual stream
and the next layer reads the normalised stream,

    stream = x + residual                      (x itself without a residual)
    y      = weight * stream / sqrt(mean(stream^2) + eps)

over the last axis, all arithmetic in float32.  ``stream`` is in the residual's
dtype (float32, or x's), and the norm reads it as stored.  x may be float32,
bfloat16 or float16 with any leading shape, weight any of the three.

* :func:`add_rmsnorm` returns ``(y, stream)`` with y in x's dtype, and has a
  backward pass (x, residual and weight).
* :func:`add_rmsnorm_int8` returns ``(q, scale, stream)``: y as int8 rows with
  one float32 scale a row, ``scale = max|y| / 127``, ``q = rint(y / scale)``.
* :func:`quantize_int8` does the same to the rows of a tensor as it is: the
  activations of a projection that follows no norm, or a weight matrix (one
  scale per output channel).

A row that holds a NaN or an infinity has scale NaN (what reads it is NaN, not
silently finite); a row of zeros has scale 0.  Finite rows may be as large as their type allows, as
long as ``weight * stream`` stays inside float32: an element past it counts as infinite.  The int8 functions have no
gradient and say so when one is asked for.  The reference has no counterpart.
CUDA tensors only; kernels in ``csrc/add_rmsnorm.cu``.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native as nat
from .gated_norm import _rows

__all__ = ["add_rmsnorm", "add_rmsnorm_int8", "quantize_int8"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _stride(t):
    return t.stride(0) if t is not None and t.shape[0] > 1 else 0


def _ptr(t):
    return None if t is None else t.data_ptr()


def _features(t):
    """t itself when its rows are contiguous features with even spacing (any
    leading shape if t is contiguous, else two axes), a two-axis view or a copy
    otherwise."""
    return t if t.is_contiguous() else _rows(t, t.shape[-1])


def _row_stride(t):
    return 0 if t is None or t.is_contiguous() else _stride(t)


def _params(x, residual, weight, eps, stream=None, y=None, q=None, scale=None, rstd=None):
    features = x.shape[-1]
    code = nat.dtype_code(x.dtype)
    return nat.AddRmsNormParams(
        x.numel() // features, features, _row_stride(x), _row_stride(residual), 0, 0, code,
        code if residual is None else nat.dtype_code(residual.dtype),
        0 if weight is None else nat.dtype_code(weight.dtype), eps, x.data_ptr(),
        _ptr(residual), _ptr(weight), _ptr(stream), _ptr(y), _ptr(q), _ptr(scale), _ptr(rstd))


def _per_row(shape, x):
    return nat.vector(shape[0], x) if len(shape) == 2 else torch.empty(shape[:-1], dtype=torch.float32, device=x.device)


# The launches.  `shape` is the outputs' shape; x and residual are its rows.
def _forward(x, weight, residual, eps, save, shape):
    y = nat.like(x, shape, x.dtype)
    stream = None if residual is None else nat.like(residual, shape, residual.dtype)
    rstd = _per_row(shape, x) if save else None
    p = _params(x, residual, weight, eps, stream, y, rstd=rstd)
    nat.check(nat.lib().ssm_add_rmsnorm_fwd(p, nat.stream_here(x)), "add_rmsnorm")
    return y, stream, rstd


def _forward_int8(x, weight, residual, eps, shape):
    q = nat.like(x, shape, torch.int8)
    scale = _per_row(shape, x)
    stream = None if residual is None else nat.like(residual, shape, residual.dtype)
    p = _params(x, residual, weight, eps, stream, q=q, scale=scale)
    nat.check(nat.lib().ssm_add_rmsnorm_fwd(p, nat.stream_here(x)), "add_rmsnorm_int8")
    return q, scale, stream


def _quantize(x, shape):
    q = nat.like(x, shape, torch.int8)
    scale = _per_row(shape, x)
    nat.check(nat.lib().ssm_quantize_int8(_params(x, None, None, 0.0, q=q, scale=scale), nat.stream_here(x)),
              "quantize_int8")
    return q, scale


def _none_empty(t, like, dtype):
    """Custom ops return tensors: an empty one in the place of an absent output."""
    return torch.empty(0, dtype=dtype, device=like.device) if t is None else t


@torch.library.custom_op("b200ssm::add_rmsnorm_fwd", mutates_args=(), device_types="cuda")
def _fwd(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor], eps: float,
         save: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.cuda.device_of(x):
        y, stream, rstd = _forward(x, weight, residual, eps, save, x.shape)
    return y, _none_empty(stream, x, x.dtype), _none_empty(rstd, x, torch.float32)


@_fwd.register_fake
def _(x, weight, residual, eps, save):
    return (x.new_empty(x.shape), x.new_empty(0) if residual is None else residual.new_empty(x.shape),
            x.new_empty(x.shape[0] if save else 0, dtype=torch.float32))


@torch.library.custom_op("b200ssm::add_rmsnorm_int8", mutates_args=(), device_types="cuda")
def _int8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor],
          eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.cuda.device_of(x):
        q, scale, stream = _forward_int8(x, weight, residual, eps, x.shape)
    return q, scale, _none_empty(stream, x, x.dtype)


@_int8.register_fake
def _(x, weight, residual, eps):
    return (x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32),
            x.new_empty(0) if residual is None else residual.new_empty(x.shape))


@torch.library.custom_op("b200ssm::quantize_int8", mutates_args=(), device_types="cuda")
def _quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    with torch.cuda.device_of(x):
        return _quantize(x, x.shape)


@_quant.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32)


def _backward_launch(dy, dstream, stream, weight, rstd, eps):
    """(dx, dresidual in the stream's type or None where dx is it, dweight); dy, dstream and stream are rows."""
    features = dy.shape[-1]
    dx = nat.like(dy, dy.shape, dy.dtype)
    dres = nat.like(dy, dy.shape, stream.dtype) if stream.dtype != dy.dtype else None
    dw = nat.vector(features, dy)
    p = nat.AddRmsNormParams(
        dy.numel() // features, features, _row_stride(stream), 0, _row_stride(dy), _row_stride(dstream),
        nat.dtype_code(dy.dtype), nat.dtype_code(stream.dtype), nat.dtype_code(weight.dtype), eps)
    need = nat._SZ()
    nat.check(nat.lib().ssm_add_rmsnorm_sizes(p, need), "add_rmsnorm backward")
    ws = nat.vector(need.value // 4 + 1, dy)
    p.stream, p.weight, p.rstd, p.dy, p.dx = (t.data_ptr() for t in (stream, weight, rstd, dy, dx))
    p.dstream, p.dresidual, p.dweight = _ptr(dstream), _ptr(dres), dw.data_ptr()
    p.workspace, p.workspace_bytes = ws.data_ptr(), need.value
    nat.check(nat.lib().ssm_add_rmsnorm_bwd(p, nat.stream_here(dy)), "add_rmsnorm backward")
    return dx, dres, dw


@torch.library.custom_op("b200ssm::add_rmsnorm_bwd", mutates_args=(), device_types="cuda")
def _bwd(dy: torch.Tensor, dstream: Optional[torch.Tensor], stream: torch.Tensor, weight: torch.Tensor,
         rstd: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.cuda.device_of(dy):
        dx, dres, dw = _backward_launch(dy, dstream, stream, weight, rstd, eps)
    return dx, _none_empty(dres, dy, stream.dtype), dw


@_bwd.register_fake
def _(dy, dstream, stream, weight, rstd, eps):
    return (dy.new_empty(dy.shape), stream.new_empty(dy.shape if stream.dtype != dy.dtype else (0,)),
            dy.new_empty(dy.shape[1], dtype=torch.float32))


def _setup(ctx, inputs, output):
    x, weight, residual, eps, save = inputs
    _, stream, rstd = output
    ctx.save_for_backward(x if residual is None else stream, weight, rstd)
    ctx.eps, ctx.residual, ctx.xdtype = eps, residual is not None, x.dtype
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, dstream, drstd):
    stream, weight, rstd = ctx.saved_tensors
    if rstd.numel() == 0 and stream.numel():
        raise RuntimeError("add_rmsnorm: the forward did not save its statistics (save=False)")
    if dy is None and dstream is None:
        return (None,) * 5
    dstream = _rows(dstream, stream.shape[1]) if ctx.residual and dstream is not None else None
    dy = torch.zeros(stream.shape, dtype=ctx.xdtype, device=stream.device) if dy is None else _rows(dy, stream.shape[1])
    dx, dres, dw = _bwd(dy, dstream, stream, weight, rstd, ctx.eps)
    dres = None if not ctx.residual else dx if stream.dtype == dx.dtype else dres
    return dx, dw.to(weight.dtype), dres, None, None


_fwd.register_autograd(_backward, setup_context=_setup)


class _AddRmsNorm(torch.autograd.Function):
    """The same pair of launches for plain tensors, without the dispatcher's Python path."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        rows = _features(x)
        y, stream, rstd = _forward(rows, weight, None if residual is None else _features(residual), eps, True, x.shape)
        ctx.save_for_backward(rows if residual is None else stream, weight, rstd)
        ctx.eps, ctx.residual, ctx.like = eps, residual is not None, (x.shape, x.dtype)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, stream)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstream=None):
        stream, weight, rstd = ctx.saved_tensors
        if dy is None and dstream is None:
            return None, None, None, None
        shape, dtype = ctx.like
        dy = torch.zeros(shape, dtype=dtype, device=stream.device) if dy is None else _features(dy)
        dx, dres, dw = _backward_launch(dy, None if dstream is None else _features(dstream), stream, weight, rstd,
                                        ctx.eps)
        dx = dx.view(shape)
        return (dx, dw if dw.dtype == weight.dtype else dw.to(weight.dtype),
                None if not ctx.residual else dx if dres is None else dres.view(shape), None)


def _check(name, x, weight, residual):
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} needs a feature axis that is not empty")
    if weight is not None and weight.shape != shape[-1:]:
        raise ValueError(f"weight must be ({shape[-1]},), got {tuple(weight.shape)}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must match x {tuple(shape)}, got {tuple(residual.shape)}")
    index = x.get_device()                          # negative off the GPU
    if nat.apart(index, weight, residual):
        nat.same_device(name, index, (("x", x), ("weight", weight), ("residual", residual)))
    if x.dtype not in _DTYPES or (weight is not None and weight.dtype not in _DTYPES):
        raise ValueError(f"{name} computes float32/bfloat16/float16, x is {x.dtype}"
                         + ("" if weight is None else f", weight {weight.dtype}"))
    if residual is not None and residual.dtype is not x.dtype and residual.dtype is not torch.float32:
        raise ValueError(f"{name}: the residual stream is {x.dtype} or float32, got {residual.dtype}")


def add_rmsnorm(x, weight, residual=None, eps=1e-5):
    """``stream = x + residual`` and its RMSNorm over the last axis.

    Args:
        x: ``(..., features)``.
        weight: ``(features,)``.
        residual: the residual stream, shaped like ``x``, in x's dtype or
            float32; None for the first layer.
        eps: added to the mean square.

    Returns:
        ``(y, stream)``: y in x's dtype, stream in the residual's (x itself
        without a residual).
    """
    _check("add_rmsnorm", x, weight, residual)
    grad = nat.wants_grad(x, weight, residual)
    if x.numel() == 0 and not grad:
        return x.new_empty(x.shape), x if residual is None else x.new_empty(x.shape, dtype=residual.dtype)
    w = weight if weight.is_contiguous() else weight.contiguous()
    if nat.direct(x, w, residual):
        if grad:
            out = _AddRmsNorm.apply(x, w, residual, float(eps))
            return (out, x) if residual is None else out
        y, stream, _ = _forward(_features(x), w, None if residual is None else _features(residual), float(eps),
                                False, x.shape)
        return y, x if residual is None else stream
    features = x.shape[-1]
    y, stream, _ = torch.ops.b200ssm.add_rmsnorm_fwd(
        _rows(x, features), w, None if residual is None else _rows(residual, features), float(eps), grad)
    return y.view(x.shape), x if residual is None else stream.view(x.shape)


def add_rmsnorm_int8(x, weight, residual=None, eps=1e-5):
    """:func:`add_rmsnorm` with y as int8 rows: ``(q, scale, stream)``, q shaped
    like ``x``, scale ``x.shape[:-1]`` in float32.  No gradient."""
    _check("add_rmsnorm_int8", x, weight, residual)
    if nat.wants_grad(x, weight, residual):
        raise ValueError("add_rmsnorm_int8 has no gradient: call it under torch.no_grad(), or use add_rmsnorm")
    if x.numel() == 0:
        return (x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32),
                x if residual is None else x.new_empty(x.shape, dtype=residual.dtype))
    w = weight if weight.is_contiguous() else weight.contiguous()
    if nat.direct(x, w, residual):
        q, scale, stream = _forward_int8(_features(x), w, None if residual is None else _features(residual),
                                         float(eps), x.shape)
        return q, scale, x if residual is None else stream
    features = x.shape[-1]
    q, scale, stream = torch.ops.b200ssm.add_rmsnorm_int8(
        _rows(x, features), w, None if residual is None else _rows(residual, features), float(eps))
    return q.view(x.shape), scale.view(x.shape[:-1]), x if residual is None else stream.view(x.shape)


def quantize_int8(x):
    """The rows of ``x`` (its last axis) as int8 with a float32 scale each:
    ``(q, scale)``, ``scale = max|x| / 127`` over the row, ``q = rint(x / scale)``.
    No gradient."""
    _check("quantize_int8", x, None, None)
    if nat.wants_grad(x):
        raise ValueError("quantize_int8 has no gradient: call it under torch.no_grad()")
    if x.numel() == 0:
        return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)
    if nat.direct(x):
        return _quantize(_features(x), x.shape)
    q, scale = torch.ops.b200ssm.quantize_int8(_rows(x, x.shape[-1]))
    return q.view(x.shape), scale.view(x.shape[:-1])
