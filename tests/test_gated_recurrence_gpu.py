"""Gated linear recurrence and its single-token step vs the 64-bit definition.

Limits, from the arithmetic.  A state forgets: a step's own error (the gate to
1e-6 of itself, the roundings of the update) decays with the gate, and with
gates that write g >= 2e-4 of the new token the errors of the remembered steps
add up to under 2e-5 of the largest magnitude M that entered (inputs or initial
state), whatever the length; y adds one rounding to its type.  The same holds for
the gradient's scan, so a gradient tensor errs by at most 2e-5 of its norm, plus
one rounding to its type of every element (fp16 gradients also to its last
subnormal step).
"""

import pytest
import torch

from oracle import lm_oracle as lm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
STEP = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -24}


def _cv():
    from metal_kernelops_b200 import cv
    return cv


def _make(batch, length, dim, dtype, gate, lower, init, reset, seed=1):
    g = torch.Generator().manual_seed(seed)
    t = dict(x=torch.randn(batch, length, dim, generator=g).to(dtype),
             forget=(torch.randn(batch, length, dim, generator=g) * 1.5 + 2).clamp(-8, 6).to(dtype))
    if gate:
        t["z"] = torch.randn(batch, length, dim, generator=g).to(dtype)
    if lower:
        t["lower"] = torch.rand(dim, generator=g) * 0.9
    if init:
        t["init"] = torch.randn(batch, dim, generator=g)
    if reset:
        t["reset"] = torch.rand(batch, length, generator=g) < 0.03
        if length:
            t["reset"][0, 0] = True
    return t


def _run(t, device="cuda"):
    d = {k: v.to(device) for k, v in t.items()}
    return _cv().gated_linear_recurrence(d["x"], d["forget"], d.get("z"), d.get("lower"), d.get("init"),
                                         d.get("reset"))


def _ref(t):
    d = {k: v.double() if v.is_floating_point() else v for k, v in t.items()}
    return lm.gated_recurrence_ref(d["x"], d["forget"], d.get("z"), d.get("lower"), d.get("init"), d.get("reset"))


def _largest(t):
    return max([float(t[k].abs().max()) for k in ("x", "init") if k in t and t[k].numel()] + [1e-30])


def _check(t, y, final):
    want, last = _ref(t)
    dtype = t["x"].dtype
    m = _largest(t)
    gate = 1.0
    if "z" in t:
        z = t["z"].double()
        gate = (z * torch.sigmoid(z)).abs()
    assert y.dtype == dtype and y.shape == t["x"].shape and final.dtype == F32
    err = (y.double().cpu() - want).abs()
    assert bool((err <= 2e-5 * m * gate + UNIT[dtype] * want.abs() + STEP[dtype]).all()), float(err.max())
    err = (final.double().cpu() - last).abs()
    assert bool((err <= 2e-5 * m).all()), float(err.max())


CASES = [  # batch, length, dim, dtype, gate, lower, initial state, reset
    (2, 1, 64, BF16, True, True, True, False),
    (1, 2, 1, F32, False, False, False, False),
    (3, 7, 31, BF16, True, True, True, True),
    (2, 63, 65, F16, False, True, False, True),
    (2, 64, 130, BF16, True, False, True, False),
    (1, 65, 96, F32, True, True, True, True),
    (2, 129, 200, F16, True, True, False, False),
    (4, 300, 33, F32, False, True, True, True),
    (1, 1000, 70, BF16, True, True, True, True),
    (2, 2500, 64, BF16, False, True, True, False),
    (1, 4097, 8, F32, True, False, False, True),
    (5, 130, 2, BF16, False, False, True, True),
    (1, 8200, 256, BF16, True, True, True, True),
    (1, 3000, 1024, F16, True, True, True, False),
    (5, 200, 4096, BF16, True, True, True, True),          # tiles enough without clusters
    (6, 200, 2000, F32, True, True, True, False),
    (1, 1000, 4608, BF16, True, False, True, True),        # clusters of four and of two
    (1, 500, 9472, BF16, False, True, False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward(case):
    t = _make(*case)
    with torch.no_grad():
        _check(t, *_run(t))


@pytest.mark.gpu
@pytest.mark.parametrize("up", ["y", "final", "both"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients(case, up):
    t = _make(*case)
    g = torch.Generator().manual_seed(7)
    dy = torch.randn(t["x"].shape, generator=g).to(t["x"].dtype)
    df = torch.randn(t["x"].shape[0], t["x"].shape[2], generator=g)
    names = [k for k in t if t[k].is_floating_point()]
    dev = {k: v.cuda().requires_grad_(k in names) for k, v in t.items()}
    ref = {k: (v.double().requires_grad_(True) if k in names else v) for k, v in t.items()}

    def grads(fn, d, gy, gf):
        y, final = fn(d["x"], d["forget"], d.get("z"), d.get("lower"), d.get("init"), d.get("reset"))
        pairs = [(y, gy)] * (up != "final") + [(final, gf)] * (up != "y")
        return y, final, torch.autograd.grad([o for o, _ in pairs], [d[k] for k in names], [v for _, v in pairs],
                                             allow_unused=True)

    y, final, got = grads(_cv().gated_linear_recurrence, dev, dy.cuda(), df.cuda())
    _check(t, y.detach(), final.detach())
    _, _, want = grads(lm.gated_recurrence_ref, ref, dy.double(), df.double())
    for k, a, b in zip(names, got, want):
        b = torch.zeros_like(ref[k]) if b is None else b
        assert a.dtype == t[k].dtype and a.shape == b.shape, k
        err = float((a.double().cpu() - b).norm())
        limit = (2e-5 + UNIT[a.dtype]) * float(b.norm()) + STEP[a.dtype] * b.numel() ** 0.5
        # dlower sums cancelling terms over the batch and the sequence: its error follows the terms
        if k == "lower":
            limit += 1e-6 * float(t["x"].double().norm())
        assert err <= limit + 1e-30, (k, err, limit)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivatives by central differences of the kernel's own fp32
    forward: truncation about step^2, rounding 2e-5 / step of the values' norm."""
    t = {k: v.cuda() for k, v in _make(2, 150, 40, F32, True, True, True, True).items()}
    names = [k for k in t if k != "reset"]
    g = torch.Generator().manual_seed(3)
    dy, df = torch.randn(2, 150, 40, generator=g).cuda(), torch.randn(2, 40, generator=g).cuda()
    cv = _cv()

    def value(d):
        with torch.no_grad():
            y, f = cv.gated_linear_recurrence(d["x"], d["forget"], d["z"], d["lower"], d["init"], d["reset"])
        return float((y.double() * dy.double()).sum() + (f.double() * df.double()).sum())

    leaf = {k: v.clone().requires_grad_(k in names) for k, v in t.items()}
    y, f = cv.gated_linear_recurrence(leaf["x"], leaf["forget"], leaf["z"], leaf["lower"], leaf["init"],
                                      leaf["reset"])
    grads = dict(zip(names, torch.autograd.grad((y, f), [leaf[k] for k in names], (dy, df))))
    for k in names:
        v = torch.randn(t[k].shape, generator=g).cuda() * (0.02 if k == "lower" else 1.0)
        h = 1e-2
        diff = (value({**t, k: t[k] + h * v}) - value({**t, k: t[k] - h * v})) / (2 * h)
        want = float((grads[k].double() * v.double()).sum())
        size = float(grads[k].double().norm() * v.double().norm())
        assert abs(diff - want) <= 5e-3 * size, (k, diff, want, size)


@pytest.mark.gpu
def test_resets_separate_sequences():
    """Packed rows equal the sequences run one by one, bit for bit where they
    begin a chunk's steps alike, and a NaN or an infinity does not cross a reset."""
    t = _make(1, 700, 96, F32, True, True, False, False)
    cuts = [0, 1, 64, 65, 300, 699]
    reset = torch.zeros(1, 700, dtype=torch.bool)
    for c in cuts:
        reset[0, c] = True
    t["init"] = torch.full((1, 96), float("nan"))
    t["reset"] = reset
    t["x"][0, 10, 3] = float("inf")
    t["x"][0, 200, 5] = float("nan")
    y, final = _run(t)
    ends = cuts[1:] + [700]
    for a, b in zip(cuts, ends):
        part = {k: t[k][:, a:b].contiguous() for k in ("x", "forget", "z")}
        part["lower"] = t["lower"]
        yy, ff = _run(part)
        assert torch.equal(y[:, a:b].isfinite(), yy.isfinite())
        ok = yy.isfinite()
        assert bool(((y[:, a:b] - yy)[ok].abs() <= 1e-4).all())
    assert bool(final.isfinite().all())
    clean = torch.ones(96, dtype=torch.bool)
    clean[3] = clean[5] = False
    assert bool(y[:, :, clean].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("value,expect", [(float("inf"), "keeps"), (float("-inf"), "writes"), (90.0, "keeps"),
                                          (-90.0, "writes"), (float("nan"), "nan")])
def test_extreme_gates(value, expect):
    x = torch.randn(2, 100, 64, device="cuda")
    f = torch.full_like(x, value)
    init = torch.randn(2, 64, device="cuda")
    x.requires_grad_(True)
    f.requires_grad_(True)
    y, final = _cv().gated_linear_recurrence(x, f, initial_state=init)
    gx, gf = torch.autograd.grad(y.sum(), (x, f))
    if expect == "nan":
        assert bool(y.isnan().all())
    elif expect == "keeps":
        assert torch.equal(final, init) and bool((gx.abs() < 1e-30).all()) and bool(gf.isfinite().all())
    else:
        assert torch.equal(y.detach(), x.detach()) and bool(gf.isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 8, 3])
def test_slices_of_a_projection_on_another_stream(offset):
    """x, forget and z as column slices of one wide buffer, aligned or not."""
    batch, length, dim = 2, 200, 136
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(batch, length, 3 * dim + 16, generator=g).to(BF16)
    cut = lambda w, i: w[..., offset + i * dim:offset + (i + 1) * dim]  # noqa: E731
    t = dict(x=cut(wide, 0), forget=cut(wide, 1), z=cut(wide, 2))
    dev = wide.cuda()
    d = dict(x=cut(dev, 0), forget=cut(dev, 1), z=cut(dev, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        y, final = _cv().gated_linear_recurrence(d["x"], d["forget"], d["z"])
    torch.cuda.current_stream().wait_stream(side)
    _check(t, y, final)
    swapped = t["x"].transpose(1, 2).contiguous().transpose(1, 2).cuda()      # channels not contiguous
    with torch.no_grad():
        y2, _ = _cv().gated_linear_recurrence(swapped, d["forget"], d["z"])
    assert torch.equal(y2, y)
    dyw = torch.randn(batch, length, 2 * dim, generator=g).to(BF16).cuda()
    x = d["x"].detach().requires_grad_(True)
    y, _ = _cv().gated_linear_recurrence(x, d["forget"], d["z"])
    a, = torch.autograd.grad(y, x, dyw[..., dim:], retain_graph=True)
    b, = torch.autograd.grad(y, x, dyw[..., dim:].contiguous())
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch,dim,gate", [(1, 1, True), (3, 64, True), (5, 65, False), (128, 520, True),
                                            (2, 4099, True)])
def test_steps_equal_the_sequence(batch, dim, gate, dtype):
    """Token by token in place (the state a slice of a larger cache, the inputs
    slices of a projection) against the definition and against the scan."""
    t = _make(batch, 9, dim, dtype, gate, True, True, False)
    cache = torch.zeros(batch, 2 * dim, device="cuda")
    state = cache[:, dim:]
    state.copy_(t["init"])
    wide = torch.cat([t["x"], t["forget"], t["z"] if gate else t["x"]], -1).cuda()
    ys = []
    for i in range(9):
        tok = wide[:, i]
        ys.append(_cv().gated_linear_recurrence_update(
            state, tok[:, :dim], tok[:, dim:2 * dim], tok[:, 2 * dim:] if gate else None, t["lower"].cuda()))
    _check(t, torch.stack(ys, 1), state.clone())
    assert bool((cache[:, :dim] == 0).all())
    with torch.no_grad():
        y, final = _run(t)
    assert bool(((final - state).abs() <= 4e-5 * _largest(t)).all())


@pytest.mark.gpu
def test_empty_and_repeatable():
    cv = _cv()
    e = torch.empty(2, 0, 64, device="cuda", dtype=BF16)
    init = torch.randn(2, 64, device="cuda", requires_grad=True)
    y, final = cv.gated_linear_recurrence(e, e, initial_state=init)
    assert y.shape == (2, 0, 64) and torch.equal(final, init)
    g, = torch.autograd.grad(final, init, torch.ones_like(final))
    assert bool((g == 1).all())
    none = torch.empty(0, 5, 64, device="cuda")
    y, final = cv.gated_linear_recurrence(none, none)
    assert y.shape == (0, 5, 64) and final.shape == (0, 64)
    assert cv.gated_linear_recurrence_update(torch.empty(0, 8, device="cuda"), none[:, 0, :8], none[:, 0, :8]).shape == (0, 8)
    t = {k: v.cuda().requires_grad_(v.is_floating_point()) for k, v in _make(3, 777, 200, BF16, True, True, True, True).items()}
    names = [k for k in t if k != "reset"]
    runs = []
    for _ in range(2):
        y, f = cv.gated_linear_recurrence(t["x"], t["forget"], t["z"], t["lower"], t["init"], t["reset"])
        runs.append((y, f) + torch.autograd.grad((y, f), [t[k] for k in names], (torch.ones_like(y), torch.ones_like(f))))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(9, 8192, 30000), (1, 262144 + 77, 8200), (70, 4099, 7501)], ids=str)
def test_offsets_beyond_32_bits(shape):
    """More than 2^31 elements (by rows, by tokens, and in an odd width): the last
    channels of the last row equal the same channels on their own."""
    batch, length, dim = shape
    assert batch * length * dim > 1 << 31
    x = torch.empty(shape, device="cuda", dtype=BF16)
    for b in range(batch):
        x[b].normal_(generator=torch.Generator(device="cuda").manual_seed(b))
    cut = dim - 96
    leaf = x.requires_grad_(True)
    y, final = _cv().gated_linear_recurrence(leaf, leaf.detach())
    part = x.detach()[-1:, :, cut:].contiguous().requires_grad_(True)
    yp, fp = _cv().gated_linear_recurrence(part, part.detach())
    # other cluster sizes join other runs of steps: equal up to the limits above
    assert bool(((y[-1:, :, cut:] - yp).float().abs() <= 2e-5 * 6 + 2 * UNIT[BF16] * yp.float().abs()).all())
    assert bool(((final[-1:, cut:] - fp).abs() <= 2e-5 * 6).all())
    del y, final
    y, final = _cv().gated_linear_recurrence(leaf, leaf.detach())
    dx, = torch.autograd.grad((y, final), leaf, (leaf.detach(), final.detach()))
    dp, = torch.autograd.grad((yp, fp), part, (part.detach(), fp.detach()))
    dx = dx[-1:, :, cut:]
    assert float((dx.float() - dp.float()).norm()) <= (2e-5 + 2 * UNIT[BF16]) * float(dp.float().norm())


@pytest.mark.gpu
def test_through_the_dispatcher():
    cv = _cv()
    t = {k: v.cuda() for k, v in _make(2, 70, 64, BF16, True, True, True, True).items()}
    with torch.no_grad():
        a = cv.gated_linear_recurrence(t["x"], t["forget"], t["z"], t["lower"], t["init"], t["reset"])
        b = torch.ops.b200ssm.gated_recurrence_fwd(t["x"], t["forget"], t["z"], t["lower"], t["init"], t["reset"], True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    s1, s2 = t["init"].clone(), t["init"].clone()
    y1 = cv.gated_linear_recurrence_update(s1, t["x"][:, 0], t["forget"][:, 0], t["z"][:, 0], t["lower"])
    y2 = torch.ops.b200ssm.gated_recurrence_update(s2, t["x"][:, 0], t["forget"][:, 0], t["z"][:, 0], t["lower"])
    assert torch.equal(y1, y2) and torch.equal(s1, s2)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode, torch.no_grad():
        f = {k: mode.from_tensor(v) for k, v in t.items()}
        y, final = cv.gated_linear_recurrence(f["x"], f["forget"], f["z"], f["lower"], f["init"], f["reset"])
        assert y.shape == (2, 70, 64) and final.shape == (2, 64)


@pytest.mark.gpu
def test_gradients_through_the_dispatcher():
    """The registered op's autograd formula gives the direct call's gradients."""
    t = {k: v.cuda().requires_grad_(v.is_floating_point()) for k, v in _make(2, 90, 64, BF16, True, True, True, True).items()}
    names = [k for k in t if k != "reset"]
    a = _cv().gated_linear_recurrence(t["x"], t["forget"], t["z"], t["lower"], t["init"], t["reset"])
    b = torch.ops.b200ssm.gated_recurrence_fwd(t["x"], t["forget"], t["z"], t["lower"], t["init"], t["reset"], True)
    ups = (torch.ones_like(a[0]), torch.ones_like(a[1]))
    ga = torch.autograd.grad(a, [t[k] for k in names], ups)
    gb = torch.autograd.grad(b[:2], [t[k] for k in names], ups)
    assert all(torch.equal(u, v) for u, v in zip(ga, gb))
    c = torch.ops.b200ssm.gated_recurrence_fwd(t["x"], t["forget"], None, None, None, None, True)
    d = _cv().gated_linear_recurrence(t["x"], t["forget"])
    assert torch.equal(torch.autograd.grad(c[0].sum(), t["forget"])[0], torch.autograd.grad(d[0].sum(), t["forget"])[0])


@pytest.mark.gpu
def test_update_without_gradient_is_an_error():
    s = torch.zeros(2, 8, device="cuda")
    x = torch.ones(2, 8, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        _cv().gated_linear_recurrence_update(s, x, x)
    with pytest.raises(ValueError, match="float32"):
        _cv().gated_linear_recurrence_update(s.half(), x, x)
    with torch.no_grad():
        _cv().gated_linear_recurrence_update(s, x, x)


def test_refusals():
    cv = _cv()
    x = torch.zeros(2, 5, 8)
    with pytest.raises(ValueError, match="runs CUDA kernels"):
        cv.gated_linear_recurrence(x, x)
    with pytest.raises(ValueError, match="forget must match"):
        cv.gated_linear_recurrence(x, x[:, :4])
    with pytest.raises(ValueError, match="z must match"):
        cv.gated_linear_recurrence(x, x, x.half())
    with pytest.raises(ValueError, match="lower_bound must be"):
        cv.gated_linear_recurrence(x, x, lower_bound=torch.zeros(7))
    with pytest.raises(ValueError, match="the state must be"):
        cv.gated_linear_recurrence(x, x, initial_state=torch.zeros(2, 7))
    with pytest.raises(ValueError, match="reset must be"):
        cv.gated_linear_recurrence(x, x, reset=torch.zeros(2, 5))
    with pytest.raises(ValueError, match="x must be"):
        cv.gated_linear_recurrence(x[0], x[0])
    with pytest.raises(ValueError, match="x must be"):
        cv.gated_linear_recurrence_update(torch.zeros(2, 8), x, x)
    with pytest.raises(ValueError, match="runs CUDA kernels"):
        cv.gated_linear_recurrence_update(torch.zeros(2, 8), x[:, 0], x[:, 0])


def test_refusals_of_the_c_entry():
    from metal_kernelops_b200 import _native as nat
    lib = nat.lib()
    p = nat.GatedRecurrenceParams()
    p.batch, p.length, p.dim = 1, -1, 8
    assert lib.ssm_gated_recurrence_fwd(p, None) == nat.SSM_ERR_INVALID
    p.length, p.dim = 4, 0
    assert lib.ssm_gated_recurrence_bwd(p, None) == nat.SSM_ERR_INVALID
    p.dim, p.dtype = 8, 9
    assert lib.ssm_gated_recurrence_fwd(p, None) == nat.SSM_ERR_UNSUPPORTED
    p.dtype, p.batch = nat.SSM_F32, 70000
    assert lib.ssm_gated_recurrence_fwd(p, None) == nat.SSM_ERR_UNSUPPORTED
    p.batch, p.x_token_stride = 1, 4
    assert lib.ssm_gated_recurrence_fwd(p, None) == nat.SSM_ERR_INVALID
    p.x_token_stride = 0
    assert lib.ssm_gated_recurrence_fwd(p, None) == nat.SSM_ERR_INVALID     # null pointers
    assert lib.ssm_gated_recurrence_bwd(p, None) == nat.SSM_ERR_INVALID
    assert lib.ssm_gated_recurrence_fwd(None, None) == nat.SSM_ERR_INVALID
    q = nat.GatedRecurrenceStepParams()
    q.batch, q.dim = 2, 0
    assert lib.ssm_gated_recurrence_step(q, None) == nat.SSM_ERR_INVALID
    q.dim = 8
    assert lib.ssm_gated_recurrence_step(q, None) == nat.SSM_ERR_INVALID
    q.batch = 0
    assert lib.ssm_gated_recurrence_step(q, None) == nat.SSM_OK
