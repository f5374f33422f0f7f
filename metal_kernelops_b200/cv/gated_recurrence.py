"""Gated linear recurrence on the B200: one state per channel, a forget gate that
comes with every token.

    g_t = (1 - lower_bound) * sigmoid(-forget_t)
    h_t = (1 - g_t) * h_{t-1} + g_t * x_t            (h_{t-1} = 0 where reset_t)
    y_t = h_t * silu(z_t)                            (h_t without z)

``1 - g_t`` is the forget gate: between ``lower_bound`` (per channel) and 1.
x, forget and z are (batch, length, dim) -- the layout an in-projection leaves,
column slices of a wider projection output included -- in float32, bfloat16 or
float16; the state is float32 throughout.

* :func:`gated_linear_recurrence` runs whole sequences, with gradients for
  every differentiable argument (the forward keeps one float32 state per chunk of
  steps, the backward recomputes the rest).  ``reset`` marks the first token of
  each sequence when several are packed in a row.
* :func:`gated_linear_recurrence_update` takes one token per row and updates
  the state in place.

Gates are computed in float32 from approximate exponentials: ``g`` errs by up to
``(1.25 |forget| + 10) / 2**24`` of itself.  Steady gates near one keep their memory over long
rows: 65536 steps with ``forget`` of 8 to 12 stay within 4e-5 of the definition.

The reference has no counterpart.  CUDA tensors only; kernels in
``csrc/gated_recurrence.cu``.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native as nat

__all__ = ["gated_linear_recurrence", "gated_linear_recurrence_update"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _tokens(t):
    """t itself where its channels are contiguous and its tokens do not overlap, else a contiguous copy."""
    if t is None or t.is_contiguous():
        return t
    dim = t.shape[-1]
    if t.stride(-1) == 1 and (t.shape[1] == 1 or t.stride(1) >= dim) and (t.shape[0] == 1 or t.stride(0) >= dim):
        return t
    return t.contiguous()


def _strides(t):
    """(token, batch) strides; 0: dense."""
    if t is None or t.is_contiguous():
        return 0, 0
    token = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    return token, t.stride(0) if t.shape[0] > 1 else token * t.shape[1]


def _params(x, forget, z, lower, init, reset, dy=None):
    return nat.GatedRecurrenceParams(
        *x.shape, *_strides(x), *_strides(forget), *_strides(z), *_strides(dy), nat.dtype_code(x.dtype), 0,
        x.data_ptr(), forget.data_ptr(), _ptr(z), _ptr(lower), _ptr(init), _ptr(reset))


def _sizes(p):
    states, ws = nat._SZ(), nat._SZ()
    nat.check(nat.lib().ssm_gated_recurrence_sizes(p, states, ws), "gated_linear_recurrence")
    return states.value, ws.value


def _forward(x, forget, z, lower, init, reset, save):
    p = _params(x, forget, z, lower, init, reset)
    y = nat.like(x, x.shape, x.dtype)
    final = nat.matrix(x.shape[0], x.shape[2], torch.float32, x)
    states = nat.vector(_sizes(p)[0] // 4, x) if save else None
    p.y, p.final_state, p.states = y.data_ptr(), final.data_ptr(), _ptr(states)
    p.status = nat.status_word(x.device, "gated_recurrence")
    nat.check(nat.lib().ssm_gated_recurrence_fwd(p, nat.stream_here(x)), "gated_linear_recurrence")
    return y, final, states


@torch.library.custom_op("b200ssm::gated_recurrence_fwd", mutates_args=(), device_types="cuda")
def _fwd(x: torch.Tensor, forget: torch.Tensor, z: Optional[torch.Tensor], lower: Optional[torch.Tensor],
         init: Optional[torch.Tensor], reset: Optional[torch.Tensor],
         save: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.cuda.device_of(x):
        y, final, states = _forward(x, forget, z, lower, init, reset, save)
    return y, final, final.new_empty(0) if states is None else states


@_fwd.register_fake
def _(x, forget, z, lower, init, reset, save):
    n = 0
    if save:
        p = nat.GatedRecurrenceParams(*x.shape)
        n = _sizes(p)[0] // 4
    return (x.new_empty(x.shape), x.new_empty((x.shape[0], x.shape[2]), dtype=torch.float32),
            x.new_empty(n, dtype=torch.float32))


def _backward_launch(dy, dfinal, x, forget, z, lower, reset, states):
    """(dx, dforget, dz, dlower, dinitial), None for what the call did not have."""
    p = _params(x, forget, z, lower, None, reset, dy)
    _, ws_bytes = _sizes(p)
    dev = x.device
    dx, df = nat.like(x, x.shape, x.dtype), nat.like(x, x.shape, x.dtype)
    dz = nat.like(x, x.shape, x.dtype) if z is not None else None
    dlower = nat.vector(x.shape[2], x) if lower is not None else None
    dinit = nat.matrix(x.shape[0], x.shape[2], torch.float32, x)
    ws = nat.vector(ws_bytes // 4 + 1, x)
    p.states, p.dy, p.dfinal = states.data_ptr(), dy.data_ptr(), _ptr(dfinal)
    p.dx, p.dforget, p.dz = dx.data_ptr(), df.data_ptr(), _ptr(dz)
    p.dlower, p.dinitial = _ptr(dlower), dinit.data_ptr()
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws_bytes
    p.status = nat.status_word(dev, "gated_recurrence")
    nat.check(nat.lib().ssm_gated_recurrence_bwd(p, nat.stream_here(x)), "gated_linear_recurrence backward")
    return dx, df, dz, dlower, dinit


@torch.library.custom_op("b200ssm::gated_recurrence_bwd", mutates_args=(), device_types="cuda")
def _bwd(dy: torch.Tensor, dfinal: Optional[torch.Tensor], x: torch.Tensor, forget: torch.Tensor,
         z: Optional[torch.Tensor], lower: Optional[torch.Tensor], reset: Optional[torch.Tensor],
         states: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.cuda.device_of(x):
        dx, df, dz, dlower, dinit = _backward_launch(dy, dfinal, x, forget, z, lower, reset, states)
    return (dx, df, x.new_empty(0) if dz is None else dz, dinit.new_empty(0) if dlower is None else dlower, dinit)


@_bwd.register_fake
def _(dy, dfinal, x, forget, z, lower, reset, states):
    f32 = dict(dtype=torch.float32)
    return (x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape if z is not None else (0,)),
            x.new_empty(x.shape[2] if lower is not None else 0, **f32),
            x.new_empty((x.shape[0], x.shape[2]), **f32))


def _setup(ctx, inputs, output):
    x, forget, z, lower, init, reset, save = inputs
    ctx.save_for_backward(x, forget, z, lower, reset, output[2])
    ctx.save, ctx.init = save, init is not None
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, dfinal, dstates):
    x, forget, z, lower, reset, states = ctx.saved_tensors
    if not ctx.save:
        raise RuntimeError("gated_linear_recurrence: the forward did not save its states (save=False)")
    if dy is None and dfinal is None:
        return (None,) * 7
    dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else _tokens(dy)
    dx, df, dz, dlower, dinit = _bwd(dy, None if dfinal is None else dfinal.contiguous(), x, forget, z, lower, reset,
                                     states)
    return (dx, df, dz if z is not None else None, dlower if lower is not None else None,
            dinit if ctx.init else None, None, None)


_fwd.register_autograd(_backward, setup_context=_setup)


class _Scan(torch.autograd.Function):
    """The same pair of launches for plain tensors, without the dispatcher's Python path."""

    @staticmethod
    def forward(ctx, x, forget, z, lower, init, reset):
        y, final, states = _forward(x, forget, z, lower, init, reset, True)
        ctx.save_for_backward(x, forget, z, lower, reset, states)
        ctx.init = init is not None
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal):
        x, forget, z, lower, reset, states = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 6
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else _tokens(dy)
        dx, df, dz, dlower, dinit = _backward_launch(dy, None if dfinal is None else dfinal.contiguous(), x, forget, z,
                                                     lower, reset, states)
        return dx, df, dz, dlower, dinit if ctx.init else None, None


def _rows(t):
    """t itself where its channels are contiguous and its rows do not overlap, else a contiguous copy."""
    if t is None or t.is_contiguous() or (t.stride(1) == 1 and t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _row_stride(t):
    """Elements between rows (0: dense)."""
    return 0 if t is None or t.is_contiguous() or t.shape[0] == 1 else t.stride(0)


def _update(state, x, forget, z, lower):
    batch, dim = x.shape
    y = nat.matrix(batch, dim, x.dtype, x)
    p = nat.GatedRecurrenceStepParams(
        batch, dim, _row_stride(x), _row_stride(forget), _row_stride(z), _row_stride(state),
        nat.dtype_code(x.dtype), 0, x.data_ptr(), forget.data_ptr(), _ptr(z), _ptr(lower), state.data_ptr(),
        y.data_ptr())
    nat.check(nat.lib().ssm_gated_recurrence_step(p, nat.stream_here(x)), "gated_linear_recurrence_update")
    return y


@torch.library.custom_op("b200ssm::gated_recurrence_update", mutates_args=("state",), device_types="cuda")
def _step(state: torch.Tensor, x: torch.Tensor, forget: torch.Tensor, z: Optional[torch.Tensor],
          lower: Optional[torch.Tensor]) -> torch.Tensor:
    with torch.cuda.device_of(x):
        return _update(state, x, forget, z, lower)


@_step.register_fake
def _(state, x, forget, z, lower):
    return x.new_empty(x.shape)


def _check(name, x, forget, z, lower, state, reset, axes):
    shape = x.shape
    if len(shape) != axes or shape[-1] == 0:
        raise ValueError(f"{name}: x must be {'(batch, length, dim)' if axes == 3 else '(batch, dim)'}, "
                         f"got {tuple(shape)}")
    for label, t in (("forget", forget), ("z", z)):
        if t is not None and (t.shape != shape or t.dtype is not x.dtype):
            raise ValueError(f"{label} must match x ({tuple(shape)}, {x.dtype}), got {tuple(t.shape)}, {t.dtype}")
    if lower is not None and lower.shape != shape[-1:]:
        raise ValueError(f"lower_bound must be ({shape[-1]},), got {tuple(lower.shape)}")
    if state is not None and state.shape != (shape[0], shape[-1]):
        raise ValueError(f"the state must be ({shape[0]}, {shape[-1]}), got {tuple(state.shape)}")
    if reset is not None and (reset.shape != shape[:2] or reset.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"reset must be bool {tuple(shape[:2])}, got {tuple(reset.shape)}, {reset.dtype}")
    index = x.get_device()                          # negative off the GPU
    if nat.apart(index, forget, z, lower, state, reset):
        nat.same_device(name, index, (("x", x), ("forget", forget), ("z", z), ("lower_bound", lower),
                                      ("the state", state), ("reset", reset)))
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name} computes float32/bfloat16/float16, x is {x.dtype}")


def _f32(t):
    return t if t is None or (t.dtype is torch.float32 and t.is_contiguous()) else t.float().contiguous()


def gated_linear_recurrence(x, forget, z=None, lower_bound=None, initial_state=None, reset=None):
    """The recurrence over whole sequences.

    Args:
        x: ``(batch, length, dim)``.
        forget: pre-activation of the forget gate, shaped like ``x``.
        z: output gate, shaped like ``x`` (``silu(z)`` multiplies the state), or None.
        lower_bound: ``(dim,)`` lower bounds of the forget gate in [0, 1); None: 0.
        initial_state: ``(batch, dim)``; None: zeros.
        reset: bool ``(batch, length)``: True where a step starts from a zero
            state (the first token of a packed sequence); None: nowhere.

    Returns:
        ``(y, final_state)``: y shaped like ``x`` in its dtype, final_state
        ``(batch, dim)`` in float32.
    """
    _check("gated_linear_recurrence", x, forget, z, lower_bound, initial_state, reset, 3)
    x, forget, z = _tokens(x), _tokens(forget), _tokens(z)
    lower, init = _f32(lower_bound), _f32(initial_state)
    if reset is not None and not reset.is_contiguous():
        reset = reset.contiguous()
    grad = nat.wants_grad(x, forget, z, lower, init)
    if nat.direct(x, forget, z, lower, init, reset):
        if grad:
            return _Scan.apply(x, forget, z, lower, init, reset)
        y, final, _ = _forward(x, forget, z, lower, init, reset, False)
        return y, final
    y, final, _ = torch.ops.b200ssm.gated_recurrence_fwd(x, forget, z, lower, init, reset, grad)
    return y, final


def gated_linear_recurrence_update(state, x, forget, z=None, lower_bound=None):
    """One token per row: updates ``state`` in place and returns y.

    Args:
        state: ``(batch, dim)`` float32, channels contiguous (it may be a
            slice of a larger cache).
        x, forget, z: ``(batch, dim)``, as :func:`gated_linear_recurrence`'s at one step.
        lower_bound: ``(dim,)`` or None.

    Returns:
        y ``(batch, dim)`` in x's dtype.  No gradient.
    """
    _check("gated_linear_recurrence_update", x, forget, z, lower_bound, state, None, 2)
    if state.dtype is not torch.float32 or state.stride(1) != 1 or (
            state.shape[0] > 1 and state.stride(0) < state.shape[1]):
        raise ValueError("the state must be float32 with contiguous channels and rows that do not overlap")
    if nat.wants_grad(state, x, forget, z, lower_bound):
        raise ValueError("gated_linear_recurrence_update has no gradient: call it under torch.no_grad()")

    x, forget, z, lower = _rows(x), _rows(forget), _rows(z), _f32(lower_bound)
    if nat.direct(x, state, forget, z, lower):
        y = _update(state, x, forget, z, lower)
        if not state.is_inference():                # autograd sees the change, as the registered op shows it
            torch.autograd.graph.increment_version(state)
        return y
    return torch.ops.b200ssm.gated_recurrence_update(state, x, forget, z, lower)
