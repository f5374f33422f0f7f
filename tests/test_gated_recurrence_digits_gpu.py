"""Digits of the gated linear recurrence, element by element, against the 64-bit definition.

Limits, from the arithmetic.  The gate's e^forget comes from an exponential of a rounded
product: g, k and 1 - k err by at most eta = (1.25 |forget| + 10) 2^-24 of themselves,
2.9e-6 at |forget| = 30.  A state errs by 2 eta of H (a gate's error moves what enters and
what stays), and by some 30 roundings of 2^-24 of H on its way through a chunk of steps, where
H is the state that the inputs' and the initial state's magnitudes give; the gradient of the
state likewise by D, the same scan over the gradients' magnitudes.  The factors of a gradient
add 2 eta.  All of it stays below C = 3e-5 of the product of the magnitudes, plus one rounding to
the output's type.  A factor 1 - g of nearly closed gates is known to 2^-24 of one, not of itself,
so gates below 0.01 count as 0.01 in the magnitudes.
"""

import pytest
import torch

from oracle import lm_oracle as lm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
STEP = {F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -24}
C = 3e-5


def _make(batch, length, dim, dtype, gate, lower, init, reset, spread=1.5, seed=1):
    g = torch.Generator().manual_seed(seed)
    t = dict(x=torch.randn(batch, length, dim, generator=g).to(dtype))
    if spread > 10:
        forget = (torch.rand(batch, length, dim, generator=g) * 2 - 1) * spread
    else:
        forget = (torch.randn(batch, length, dim, generator=g) * spread + 2).clamp(-8, 6)
    t["forget"] = forget.to(dtype)
    if gate:
        t["z"] = torch.randn(batch, length, dim, generator=g).to(dtype)
    if lower:
        t["lower"] = torch.rand(dim, generator=g) * 0.9
    if init:
        t["init"] = torch.randn(batch, dim, generator=g)
    if reset:
        t["reset"] = torch.rand(batch, length, generator=g) < 0.03
    t["dy"] = torch.randn(batch, length, dim, generator=g).to(dtype)
    t["dfinal"] = torch.randn(batch, dim, generator=g)
    return t


def _got(t):
    names = [k for k in ("x", "forget", "z", "lower", "init") if k in t]
    d = {k: v.cuda().requires_grad_(k in names) for k, v in t.items()}
    y, final = _cv().gated_linear_recurrence(d["x"], d["forget"], d.get("z"), d.get("lower"), d.get("init"),
                                             d.get("reset"))
    got = torch.autograd.grad((y, final), [d[k] for k in names], (d["dy"], d["dfinal"]))
    return {"y": y.detach(), "final": final.detach(), **{"d" + k: v for k, v in zip(names, got)}}


def _want(t):
    """Outputs and gradients from the formulas, step by step in float64.  1 - k is sigmoid(forget): an
    automatic derivative of sigmoid(-forget) forms k (1 - k) and has only 4 digits left at -30."""
    d = {k: v.double() if v.is_floating_point() else v for k, v in t.items()}
    x, f, length = d["x"], d["forget"], d["x"].shape[1]
    low = d.get("lower", torch.zeros(x.shape[2], dtype=torch.float64))
    k, omk = torch.sigmoid(-f), torch.sigmoid(f)
    g, a = (1 - low) * k, low + (1 - low) * omk
    cut = d["reset"][..., None] if "reset" in d else torch.zeros(*x.shape[:2], 1, dtype=torch.bool)
    y, final = lm.gated_recurrence_ref(x, f, None, low, d.get("init"), d.get("reset"))
    first = d["init"] if "init" in d else torch.zeros_like(final)
    before = torch.cat([first[:, None], y[:, :-1]], 1)
    before = torch.where(cut, torch.zeros_like(before), before)
    up, out = d["dy"], {"final": final}
    if "z" in d:
        s = torch.sigmoid(d["z"])
        out["dz"] = up * y * (s + d["z"] * s * (1 - s))
        up, y = up * d["z"] * s, y * d["z"] * s
    dh, down = d["dfinal"], []
    for i in range(length - 1, -1, -1):
        dh = dh + up[:, i]
        down.append(dh)
        dh = torch.where(cut[:, i], torch.zeros_like(dh), a[:, i] * dh)
    down = torch.stack(down[::-1], 1)
    dg = down * (x - before)
    out.update(y=y, dx=g * down, dforget=-dg * g * omk, dlower=-(dg * k).sum((0, 1)), dinit=dh)
    return out


def _magnitudes(t):
    """What the outputs' terms amount to, from the magnitudes of what enters (float64)."""
    d = {k: v.double() if v.is_floating_point() else v for k, v in t.items()}
    x, f = d["x"].abs(), d["forget"]
    low = d.get("lower", torch.zeros(x.shape[2], dtype=torch.float64))
    k, omk = torch.sigmoid(-f), torch.sigmoid(f)
    g, a = (1 - low) * k, (low + (1 - low) * omk).clamp(min=0.01)
    cut = d["reset"][..., None] if "reset" in d else torch.zeros(*x.shape[:2], 1, dtype=torch.bool)
    a = torch.where(cut, torch.zeros_like(a), a)
    length = x.shape[1]
    h = d["init"].abs() if "init" in d else torch.zeros_like(x[:, 0])
    before, hs = [], []
    for i in range(length):
        before.append(torch.where(cut[:, i], torch.zeros_like(h), h))
        h = a[:, i] * h + g[:, i] * x[:, i]
        hs.append(h)
    before, hs = torch.stack(before, 1), torch.stack(hs, 1)
    up = d["dy"].abs()
    out = {"y": hs, "final": h}
    if "z" in d:
        s = torch.sigmoid(d["z"])
        out["y"] = hs * (d["z"] * s).abs()
        out["dz"] = up * hs * (s + (d["z"] * s * (1 - s)).abs())
        up = up * (d["z"] * s).abs()
    dh, down = d["dfinal"].abs(), []
    for i in range(length - 1, -1, -1):
        dh = dh + up[:, i]
        down.append(dh)
        dh = a[:, i] * dh
    down = torch.stack(down[::-1], 1)
    dg = down * (x + before)
    out.update(dx=g * down, dforget=dg * g * omk, dlower=(dg * k).sum((0, 1)), dinit=dh)
    return out


def _compare(t):
    got, want = _got(t), _want(t)
    size = _magnitudes(t)
    for k, a in got.items():
        b = want[k]
        err = (a.double().cpu() - b).abs()
        limit = C * size[k] + UNIT[a.dtype] * b.abs() + STEP[a.dtype]
        assert bool((err <= limit).all()), (k, float((err / limit).max()))


def _cv():
    from metal_kernelops_b200 import cv
    return cv


CASES = [  # batch, length, dim, dtype, gate, lower, initial state, reset
    (1, 2, 1, F32, False, False, False, False),
    (3, 7, 31, BF16, True, True, True, True),
    (2, 63, 65, F16, False, True, False, True),
    (2, 64, 130, BF16, True, False, True, False),
    (1, 65, 96, F32, True, True, True, True),
    (2, 129, 200, F16, True, True, False, False),
    (1, 1000, 70, BF16, True, True, True, True),
    (2, 2500, 64, BF16, False, True, True, False),
    (1, 1537, 1283, BF16, True, True, True, True),         # odd width: direct loads
    (1, 4097, 8, F32, True, False, False, True),
    (1, 8200, 256, BF16, True, True, True, True),
    (5, 200, 4096, BF16, True, True, True, True),
    (6, 200, 2000, F32, True, True, True, False),
    (1, 1000, 4608, BF16, True, False, True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_outputs_and_gradients_element_by_element(case):
    _compare(_make(*case))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gate,reset", [(True, False), (False, True)])
def test_gates_from_open_to_closed(dtype, gate, reset):
    """forget over [-30, 30]: 1 - k keeps its digits where k is near one, k where it is near zero."""
    _compare(_make(2, 300, 64, dtype, gate, True, True, reset, spread=30.0))


@pytest.mark.gpu
def test_gradient_of_a_wide_open_gate():
    """One step from a zero state: dforget = -x dy k (1 - k), each digit of it down to e^-80."""
    f = torch.linspace(-80, 80, 321).reshape(1, 1, 321)
    x = torch.full_like(f, 1.5).cuda().requires_grad_(True)
    fd = f.cuda().requires_grad_(True)
    y, _ = _cv().gated_linear_recurrence(x, fd)
    got, = torch.autograd.grad(y.sum(), fd)
    d = f.double()
    want = -1.5 * torch.sigmoid(-d) * torch.sigmoid(d)
    eta = (1.25 * d.abs() + 10) * 2.0 ** -24
    assert bool(((got.double().cpu() - want).abs() <= (2 * eta + 2.0 ** -22) * want.abs()).all())
