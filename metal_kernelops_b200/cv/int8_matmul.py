"""Linear layer in 8-bit integers on the B200's tensor cores.

    out[..., n] = x_scale[...] * weight_scale[n] * sum_k x[..., k] * weight[n, k] + bias[n]

x holds int8 rows with a float32 scale each (:func:`add_rmsnorm_int8` and
:func:`quantize_int8` make them), weight int8 rows with a float32 scale per output
feature (``quantize_int8(w)`` of a ``(out, in)`` weight, once).  The integer sums are
exact; scales and bias are applied in float32 and the result is rounded once.

For one token or a decode batch the call costs one reading of the weight; for prompts
it runs at the tensor cores' int8 rate.  Rows that start on 16-byte boundaries
(``in_features`` or the row stride a multiple of 16) are read in place; others
are copied first, the weight included, so keep an odd-width weight as a view of rows
padded to 16 bytes.  The reference has no counterpart.  CUDA tensors only, no
gradient; kernels in ``csrc/int8_linear.cu``.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native as nat

__all__ = ["int8_linear"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows(t):
    """t itself where its rows are contiguous and do not overlap, else a copy."""
    if t.is_contiguous():
        return t
    if t.dim() == 2 and t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _stride(t):
    return 0 if t.is_contiguous() or t.dim() != 2 or t.shape[0] == 1 else t.stride(0)


def _forward(x, x_scale, weight, weight_scale, bias, out_dtype):
    features, k = weight.shape
    shape, dev = x.shape, x.device
    out = (nat.matrix(shape[0], features, out_dtype, x) if len(shape) == 2
           else torch.empty((*shape[:-1], features), dtype=out_dtype, device=dev))
    xp, wp, xr, wr = x.data_ptr(), weight.data_ptr(), _stride(x), _stride(weight)
    p = nat.Int8LinearParams(
        x.numel() // k, k, features, xr, wr, nat.dtype_code(out_dtype), 0, xp, x_scale.data_ptr(), wp,
        weight_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), None, 0,
        nat.status_word(dev, "int8_linear"))
    if (k | xp | wp | xr | wr) % 16:
        need = nat._SZ()
        nat.check(nat.lib().ssm_int8_linear_sizes(p, need), "int8_linear")
        ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    nat.check(nat.lib().ssm_int8_linear_fwd(p, nat.stream_here(x)), "int8_linear")
    return out


@torch.library.custom_op("b200ssm::int8_linear", mutates_args=(), device_types="cuda")
def _op(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
        bias: Optional[torch.Tensor], out_dtype: torch.dtype) -> torch.Tensor:
    with torch.cuda.device_of(x):
        return _forward(x, x_scale, weight, weight_scale, bias, out_dtype)


@_op.register_fake
def _(x, x_scale, weight, weight_scale, bias, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype)


def int8_linear(x, x_scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """int8 rows times an int8 weight.

    Args:
        x: int8 ``(..., in_features)``.
        x_scale: float32 ``(...)``, one scale per row of x.
        weight: int8 ``(out_features, in_features)``.
        weight_scale: float32 ``(out_features,)``.
        bias: ``(out_features,)`` or None.
        out_dtype: bfloat16, float16 or float32.

    Returns:
        ``(..., out_features)`` in ``out_dtype``.
    """
    shape, wshape = x.shape, weight.shape
    if len(shape) < 1 or len(wshape) != 2 or shape[-1] != wshape[1] or 0 in wshape:
        raise ValueError(f"int8_linear: x (..., in) and weight (out, in), got {tuple(shape)} and {tuple(wshape)}")
    if x.dtype is not torch.int8 or weight.dtype is not torch.int8:
        raise ValueError(f"int8_linear: x and weight are int8, got {x.dtype} and {weight.dtype}")
    if x_scale.shape != shape[:-1] or weight_scale.shape != wshape[:1]:
        raise ValueError(f"int8_linear: x_scale must be {tuple(shape[:-1])} and weight_scale {tuple(wshape[:1])}, "
                         f"got {tuple(x_scale.shape)} and {tuple(weight_scale.shape)}")
    if x_scale.dtype is not torch.float32 or weight_scale.dtype is not torch.float32:
        raise ValueError(f"int8_linear: the scales are float32, got {x_scale.dtype} and {weight_scale.dtype}")
    if bias is not None and bias.shape != wshape[:1]:
        raise ValueError(f"int8_linear: bias must be {tuple(wshape[:1])}, got {tuple(bias.shape)}")
    if out_dtype not in _DTYPES:
        raise ValueError(f"int8_linear: out_dtype is float32/bfloat16/float16, got {out_dtype}")
    index = x.get_device()                          # negative off the GPU
    if nat.apart(index, x_scale, weight, weight_scale, bias):
        nat.same_device("int8_linear", index, (("x", x), ("x_scale", x_scale), ("weight", weight),
                                               ("weight_scale", weight_scale), ("bias", bias)))
    if nat.wants_grad(x_scale, weight_scale, bias):
        raise ValueError("int8_linear has no gradient: call it under torch.no_grad()")
    if 0 in shape:
        return torch.empty((*shape[:-1], wshape[0]), dtype=out_dtype, device=x.device)
    x, weight = _rows(x), _rows(weight)
    if not x_scale.is_contiguous():
        x_scale = x_scale.contiguous()
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    if bias is not None and (bias.dtype is not torch.float32 or not bias.is_contiguous()):
        bias = bias.float().contiguous()
    if nat.direct(x, x_scale, weight, weight_scale, bias):
        return _forward(x, x_scale, weight, weight_scale, bias, out_dtype)
    return torch.ops.b200ssm.int8_linear(x, x_scale, weight, weight_scale, bias, out_dtype)
