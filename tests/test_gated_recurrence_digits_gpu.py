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


# ------------------------------------------------------------- long memories --
# Gates that write g of a step, from 3.4e-5 to 6e-6, over 65536 steps.  A gate's own error moves the
# result by at most 2 eta <= 3e-6 of the largest magnitude M that entered, the roundings inside a
# chunk 2e-6.  The state passes from chunk to chunk 512 times at most (1024 in the backward), each
# time with a rounding of 2^-25: 3.1e-5 if all went one way.  Together below 4e-5 of M.
LONG = [(8.0, 0.9), (10.0, 0.0), (12.0, 0.0), (-3.0, 0.9999)]


def _steady(value, low, length):
    """(g, a^t for t = 1 ... length) of a steady gate, float64."""
    k = torch.sigmoid(torch.tensor(-value, dtype=torch.float64))
    g = (1 - torch.tensor(low).double()) * k
    return g, torch.exp(torch.arange(1, length + 1, dtype=torch.float64) * torch.log1p(-g))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 70, 33, 20480], ids=lambda d: f"dim{d}")
@pytest.mark.parametrize("value,low", LONG)
def test_steady_gates_over_a_long_row(value, low, dim, dtype):
    """Constant inputs: h_t = x + a^t (h_0 - x), by TMA, by word copies and by direct loads, with clusters
    and without."""
    length = 65536 if dim < 1000 else 8192
    _, decay = _steady(value, low, length)
    x = torch.full((1, 1, 1), 0.5, device="cuda", dtype=dtype).expand(1, length, dim).contiguous()
    f = torch.full_like(x, value)
    init, lower = torch.full((1, dim), 2.0, device="cuda"), torch.full((dim,), low, device="cuda")
    y, final = _cv().gated_linear_recurrence(x, f, None, lower, init)
    want = 0.5 + decay * 1.5
    assert bool(((final.double().cpu() - want[-1]).abs() <= 4e-5 * 2).all()), float((final.double().cpu() - want[-1]).abs().max())
    for c in (0, dim - 1):
        err = (y[0, :, c].double().cpu() - want).abs()
        assert bool((err <= 4e-5 * 2 + (UNIT[dtype] if dtype != F32 else 0) * want).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 33, 20480], ids=lambda d: f"dim{d}")
@pytest.mark.parametrize("value,low", LONG)
def test_gradients_of_steady_gates_over_a_long_row(value, low, dim):
    """dfinal = 1, dy = 0: dx_t = g a^(T - t), dinitial = a^T."""
    length = 65536 if dim < 1000 else 8192
    g, decay = _steady(value, low, length)
    x = torch.zeros(1, length, dim, device="cuda", requires_grad=True)
    f = torch.full((1, length, dim), value, device="cuda")
    init = torch.zeros(1, dim, device="cuda", requires_grad=True)
    _, final = _cv().gated_linear_recurrence(x, f, None, torch.full((dim,), low, device="cuda"), init)
    dx, dinit = torch.autograd.grad(final.sum(), (x, init))
    assert bool(((dinit.double().cpu() - decay[-1]).abs() <= 4e-5).all())
    want = g * torch.cat([decay.flip(0)[1:], torch.ones(1, dtype=torch.float64)])
    for c in (0, dim - 1):
        assert bool(((dx[0, :, c].double().cpu() - want).abs() <= 4.5e-5 * g).all())


@pytest.mark.gpu
@pytest.mark.parametrize("value,low", LONG)
def test_steps_with_steady_gates(value, low):
    """65536 single tokens: every step rounds the state once, 2^-25 of it; roundings of a state that
    moves differ in sign (their sum grows as the root of the count, 1e-5 at 3 sigma), and near the end value
    they cannot exceed 2^-25 / g of it, whichever way they go: 9e-4 at g = 3.4e-5.  Both are far
    below what a one-sided error would add up to, 2e-3; the limit is 1e-4 of the largest value."""
    length = 65536
    _, decay = _steady(value, low, length)
    x = torch.full((3, 64), 0.5, device="cuda")
    f, lower = torch.full_like(x, value), torch.full((64,), low, device="cuda")
    state = torch.full((3, 64), 2.0, device="cuda")
    step = lambda s: _cv().gated_linear_recurrence_update(s, x, f, None, lower)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(256):
            step(state)
    for _ in range(length // 256):
        graph.replay()
    want = 0.5 + 1.5 * decay[-1]
    assert bool(((state.double().cpu() - want).abs() <= 1e-4 * 2).all()), float((state.double().cpu() - want).abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 33])
def test_forgotten_states_keep_their_digits(dim, dtype):
    """x = 0: the state is the product of the gates, down to 1e-30 of where it began; each of a product's
    n factors errs by 2 eta g / a and a rounding, 2e-6 n at gates of 0.95 and below."""
    length = 1200
    f = torch.full((1, length, dim), 3.0, dtype=dtype)
    x = torch.zeros_like(f)
    init = torch.linspace(0.5, 2, dim)[None]
    y, final = _cv().gated_linear_recurrence(x.cuda(), f.cuda(), initial_state=init.cuda())
    want = init.double() * torch.sigmoid(torch.tensor(3.0, dtype=torch.float64)) ** length
    assert float(want.min()) < 1e-25 and bool(((final.double().cpu() - want).abs() <= 2e-6 * length * want).all())
    cv, state = _cv(), init.cuda()
    for _ in range(length):
        cv.gated_linear_recurrence_update(state, x[:, 0].cuda(), f[:, 0].cuda())
    assert bool(((state.double().cpu() - want).abs() <= 2e-6 * length * want).all())


@pytest.mark.gpu
def test_states_that_are_infinite_stay_so():
    """An infinite input or state: a h + g x stays infinite with every open gate, and a reset clears it."""
    cv = _cv()
    for batch, length, dim in ((1, 900, 64), (40, 900, 1024)):
        x = torch.zeros(batch, length, dim, device="cuda")
        x[:, 3, 0], x[:, 700, 1] = float("inf"), -float("inf")
        f = torch.full_like(x, 9.0)
        init = torch.zeros(batch, dim, device="cuda")
        init[:, 2] = float("inf")
        y, final = cv.gated_linear_recurrence(x, f, initial_state=init)
        assert bool((y[:, 3:, 0] == float("inf")).all()) and bool((y[:, 700:, 1] == -float("inf")).all())
        assert bool((y[:, :, 2] == float("inf")).all()) and bool((y[:, :, 3:] == 0).all())
        reset = torch.zeros(batch, length, dtype=torch.bool, device="cuda")
        reset[:, 800] = True
        y, final = cv.gated_linear_recurrence(x, f, initial_state=init, reset=reset)
        assert bool((y[:, 800:] == 0).all()) and bool((final == 0).all()) and bool((y[:, 799, :3].isinf()).all())
    state = torch.tensor([[float("inf"), -float("inf"), 1e10, 3.0]], device="cuda")
    x = torch.ones_like(state)
    cv.gated_linear_recurrence_update(state, x, torch.tensor([[2.0, 20.0, -80.0, float("inf")]], device="cuda"))
    assert state.tolist() == [[float("inf"), -float("inf"), 1.0, 3.0]]


@pytest.mark.gpu
def test_lower_bounds_outside_their_range_follow_the_formula():
    """A bound that training has pushed slightly past 0 or 1: the factor 1 - g may be negative or above one."""
    t = _make(2, 300, 64, F32, False, True, True, False, spread=30.0)
    t["lower"] = torch.linspace(-0.05, 1.0005, 64)
    y, final = _cv().gated_linear_recurrence(*(t[k].cuda() if k in t else None for k in ("x", "forget", "z", "lower", "init")))
    want, last = lm.gated_recurrence_ref(*(t[k].double() if k in t else None for k in ("x", "forget", "z", "lower", "init")))
    m = float(max(t["x"].abs().max(), t["init"].abs().max(), want.abs().max()))
    assert float((y.double().cpu() - want).abs().max()) <= C * m
    assert float((final.double().cpu() - last).abs().max()) <= C * m


# ------------------------------------------------------- gates that are not numbers --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch,dim", [(1, 64), (1, 33), (40, 1024)])
@pytest.mark.parametrize("at", [3, 130, 255, 256, 260, 399])
def test_nan_gates_do_not_cross_a_reset(batch, dim, dtype, at):
    """Packed sequences [0, 256), [256, 400), [400, 700): a NaN gate in one (or NaN gradients) leaves the outputs
    of those after it and the gradients of those before it as they are without it, bit for bit."""
    length, cuts = 700, [0, 256, 400]
    g = torch.Generator().manual_seed(at)
    x, f, z = (torch.randn(batch, length, dim, generator=g).to(dtype).cuda() for _ in range(3))
    reset = torch.zeros(batch, length, dtype=torch.bool)
    reset[:, cuts] = True
    reset = reset.cuda()
    dy, df = torch.randn(batch, length, dim, generator=g).to(dtype).cuda(), torch.randn(batch, dim, generator=g).cuda()
    bad = f.clone()
    bad[:, at, 3] = float("nan")
    runs = []
    for gates in (f, bad):
        leaves = [t.clone().requires_grad_(True) for t in (x, gates, z)]
        y, final = _cv().gated_linear_recurrence(*leaves, reset=reset)
        runs.append([y.detach(), final.detach(), *torch.autograd.grad((y, final), leaves, (dy, df))])
    begin, end = (0, 256) if at < 256 else (256, 400)
    for a, b in zip(*runs):
        if a.dim() == 2:
            assert torch.equal(a, b)
            continue
        assert torch.equal(a[:, :begin], b[:, :begin]) and torch.equal(a[:, end:], b[:, end:])
        other = torch.arange(dim, device="cuda") != 3
        assert torch.equal(a[..., other], b[..., other])
    assert bool(runs[1][0][:, at, 3].isnan().all())
