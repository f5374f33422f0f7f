"""Plain 64-bit definitions of the language-model operators around the scans.

Written from the formulas, element by element and step by step, on the CPU in
float64; the GPU tests compare the kernels with these.
"""

from __future__ import annotations

import torch


def add_rmsnorm_ref(x, weight, residual=None, eps=1e-5):
    """(y, stream): the stream is x + residual rounded to the residual's dtype,
    and y is the norm of the stream as stored; y in float64."""
    stream = x if residual is None else (x.double() + residual.double()).to(residual.dtype)
    s = stream.double()
    y = weight.double() * s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return y, stream


def quantize_ref(y):
    """(q, scale) of float64 rows: scale = max|y| / 127, q = rint(y / scale)."""
    scale = y.abs().amax(-1) / 127
    q = torch.where(scale[..., None] > 0, torch.round(y / scale[..., None]), torch.zeros_like(y))
    return q, scale


def add_rmsnorm_grads_ref(dy, dstream, stream, weight, eps=1e-5):
    """(d, dweight): d is the gradient of x and of the residual alike."""
    s, w, up = stream.double(), weight.double(), dy.double()
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    xh = s * r
    d = r * (up * w - xh * (up * w * xh).mean(-1, keepdim=True))
    if dstream is not None:
        d = d + dstream.double()
    return d, (up * xh).reshape(-1, w.numel()).sum(0)


def gated_recurrence_ref(x, forget, z=None, lower=None, init=None, reset=None):
    """(y, final): the recurrence step by step; differentiable in float64."""
    batch, length, dim = x.shape
    low = torch.zeros(dim, dtype=torch.float64) if lower is None else lower
    gate = low + (1 - low) * torch.sigmoid(forget)
    write = (1 - low) * torch.sigmoid(-forget)
    h = torch.zeros(batch, dim, dtype=torch.float64) if init is None else init
    hs = []
    for t in range(length):
        if reset is not None:
            h = torch.where(reset[:, t, None].bool(), torch.zeros_like(h), h)
        h = gate[:, t] * h + write[:, t] * x[:, t]
        hs.append(h)
    y = torch.stack(hs, 1) if hs else x.new_zeros(batch, 0, dim)
    if z is not None:
        y = y * (z * torch.sigmoid(z))
    return y, h


def int8_linear_ref(x, x_scale, weight, weight_scale, bias=None):
    """The exact integer sums, scaled in float64."""
    y = torch.matmul(x.double(), weight.double().t()) * x_scale.double()[..., None] * weight_scale.double()
    return y if bias is None else y + bias.double()
