"""Residual RMSNorm, its int8 output and the row quantiser vs 64-bit definitions.

Limits, from the arithmetic: the row's sum of squares, its reciprocal root and
the three products of an element cost under 60 fp32 roundings in a chain, so an
element errs by at most 4e-6 of itself, plus half an ulp of a 16-bit output.
q is within half a step of y / scale, the step itself off by 4e-6.  A gradient
element errs by at most 1e-5 of the sum of its terms' magnitudes, a dweight by
4e-6 of the sum of its products' magnitudes (chains under 60 additions at these
row counts).
"""

import pytest
import torch

from oracle import lm_oracle as lm

HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # one rounding
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _cv():
    from metal_kernelops_b200 import cv
    return cv


def _make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    if x.shape[-1] >= 4 and x.numel():
        x[..., :: max(1, x.shape[-1] // 4)] *= 8
    return x.to("cuda", dtype)


CASES = [  # rows..., features, dtype, stream dtype (None: no residual), weight dtype
    ((1, 2560), BF16, BF16, F32),
    ((3, 5, 2560), BF16, F32, BF16),
    ((7, 8), F16, F16, F16),
    ((5, 1), BF16, BF16, F32),
    ((1, 1), F32, F32, F32),
    ((9, 31), F32, F32, F32),
    ((33, 300), BF16, None, F32),
    ((130, 256), F16, F32, F32),
    ((17, 1032), F32, None, F16),
    ((6, 4104), BF16, BF16, BF16),
    ((4, 8192), F32, F32, F32),
    ((5, 8200), BF16, F32, F32),
    ((3, 16384), F16, F16, F32),
    ((2, 16392), BF16, BF16, F32),
    ((2, 20001), BF16, F32, F32),
    ((1031, 2051), F16, None, F32),
    ((700, 640), BF16, BF16, F32),
]


def _inputs(case):
    shape, dtype, stream, wdtype = case
    x = _make(shape, dtype, 1)
    res = None if stream is None else _make(shape, stream, 2)
    w = 1 + 0.2 * _make(shape[-1:], F32, 3)
    return x, res, w.to(wdtype)


def _near(got, want, dtype, rel=4e-6, floor=0.0):
    err = (got.double().cpu() - want).abs()
    tiny = 2.0 ** -24 if dtype == F16 else 1e-37          # the last subnormal steps
    return bool((err <= (rel + HALF_ULP[dtype]) * want.abs() + floor + tiny).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward(case):
    x, res, w = _inputs(case)
    y, stream = _cv().add_rmsnorm(x, w, res)
    want, kept = lm.add_rmsnorm_ref(x.cpu(), w.cpu(), None if res is None else res.cpu())
    assert y.dtype == x.dtype and y.shape == x.shape and stream.shape == x.shape
    assert stream.dtype == (x.dtype if res is None else res.dtype)
    assert torch.equal(stream.cpu(), kept)
    assert _near(y, want, x.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_int8(case):
    x, res, w = _inputs(case)
    q, scale, stream = _cv().add_rmsnorm_int8(x, w, res, eps=1e-3)
    want, kept = lm.add_rmsnorm_ref(x.cpu(), w.cpu(), None if res is None else res.cpu(), eps=1e-3)
    assert q.dtype == torch.int8 and q.shape == x.shape
    assert scale.dtype == F32 and scale.shape == x.shape[:-1]
    assert torch.equal(stream.cpu(), kept)
    _, sref = lm.quantize_ref(want)
    assert _near(scale, sref, F32)
    off = (q.double().cpu() * sref[..., None] - want).abs()
    assert bool((off <= (0.5 + 1e-3) * sref[..., None]).all())
    assert int(q.abs().max()) <= 127 and bool((q.abs().amax(-1) == 127).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_quantize(case):
    x, _, _ = _inputs(case)
    q, scale = _cv().quantize_int8(x)
    want, sref = lm.quantize_ref(x.double().cpu())
    assert _near(scale, sref, F32, rel=2.0 ** -23)
    off = (q.double().cpu() - x.double().cpu() / sref[..., None]).abs()
    assert bool((off <= 0.5 + 1e-4).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_between_two_steps_go_to_the_even_one(dtype):
    """16-bit rows whose values are exact halves of a step for many largest values
    (127 x is exact there, in float32 it rounds): q is 127 x / max in exact rational
    arithmetic, rounded to nearest, ties to even."""
    g = torch.Generator().manual_seed(3)
    m = torch.randint(1, 256, (400, 1), generator=g).double() * 2.0 ** torch.randint(-6, 6, (400, 1), generator=g)
    n = torch.randint(-127, 127, (400, 200), generator=g).double() + 0.5
    x = (n * m / 127).to(dtype)                      # halves where this is exact, near them elsewhere
    x[:, ::2] = (torch.randint(-64, 64, (400, 100), generator=g).double() * m / 128).to(dtype)[:, :100]
    x[:, 0] = m[:, 0].to(dtype)
    x = x.clamp(-m, m).to(dtype)
    q, _ = _cv().quantize_int8(x.cuda())
    num, den = (x.double() * 127 * 2 ** 34).round().long(), (m * 2 ** 34).round().long()
    assert bool((num.double() == x.double() * 127 * 2 ** 34).all())
    low = torch.div(2 * num + den, 2 * den, rounding_mode="floor")       # floor(num / den + 1/2)
    tie = (2 * num + den) % (2 * den) == 0
    want = torch.where(tie & (low % 2 != 0), low - 1, low)
    assert torch.equal(q.long().cpu(), want) and int(tie.sum()) > 100


@pytest.mark.gpu
def test_largest_and_smallest_rows():
    """Rows near the ends of float32's range keep their ratios."""
    x = torch.linspace(-1, 1, 255).repeat(3, 1)
    big = x * torch.tensor([[3.4e38], [1.0], [2.0 ** -99]])
    q, scale = _cv().quantize_int8(big.cuda())
    assert torch.equal(q[0], q[1]) and torch.equal(q[2], q[1])
    assert torch.equal(q[1].cpu(), torch.round(x[1].double() * 127).to(torch.int8))
    assert bool(scale.isfinite().all()) and bool((scale > 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("up", ["y", "stream", "both"])
def test_gradients(case, up):
    x, res, w = _inputs(case)
    leaves = [t for t in (x, res, w) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y, stream = _cv().add_rmsnorm(x, w, res)
    dy = _make(x.shape, y.dtype, 4) if up != "stream" else None
    ds = _make(x.shape, stream.dtype, 5) if up != "y" else None
    outs = [(o, g) for o, g in ((y, dy), (stream, ds)) if g is not None and o.requires_grad]
    got = torch.autograd.grad([o for o, _ in outs], leaves, [g for _, g in outs], allow_unused=True)
    dyz = torch.zeros(x.shape) if dy is None else dy.cpu()
    kept = stream.detach().cpu()
    d, dw = lm.add_rmsnorm_grads_ref(dyz, None if ds is None else ds.cpu(), kept, w.detach().cpu())
    s, wd, u = kept.double(), w.detach().double().cpu(), dyz.double()
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    size = r * ((u * wd).abs() + (s * r).abs() * (u * wd * s * r).abs().mean(-1, keepdim=True))
    size = size + (0 if ds is None else ds.double().abs().cpu())
    for g, t in zip(got, leaves):
        if t is w:
            if up == "stream" and g is None:
                continue
            mag = (u * s * r).abs().reshape(-1, w.numel()).sum(0)
            err = (g.double().cpu() - dw).abs()
            assert bool((err <= 4e-6 * mag + HALF_ULP[w.dtype] * dw.abs() + 1e-30).all())
        else:
            # x's own share of a residual-free stream adds in its dtype: one more rounding
            again = 2 * HALF_ULP[t.dtype] * size
            err = (g.double().cpu() - d).abs()
            assert g.dtype == t.dtype
            assert bool((err <= 1e-5 * size + again + 2.0 ** -24).all())


@pytest.mark.gpu
def test_gradient_against_differences():
    """The directional derivative of <y, dy> + <stream, ds> along random
    directions, by central differences of the kernel's own fp32 forward:
    truncation about step^2 = 1e-4, rounding about 1e-7 / step = 1e-5 of the
    values' norm."""
    x, res = _make((6, 96), F32, 1), _make((6, 96), F32, 2)
    w = 1 + 0.2 * _make((96,), F32, 3)
    dy, ds = _make((6, 96), F32, 4), _make((6, 96), F32, 5)
    for t in (x, res, w):
        t.requires_grad_(True)
    cv = _cv()
    y, s = cv.add_rmsnorm(x, w, res)
    grads = torch.autograd.grad((y, s), (x, res, w), (dy, ds))

    def value(xx, rr, ww):
        with torch.no_grad():
            a, b = cv.add_rmsnorm(xx, ww, rr)
        return float((a.double() * dy.double()).sum() + (b.double() * ds.double()).sum())

    base = [t.detach() for t in (x, res, w)]
    for i in range(3):
        v = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(9)).cuda()
        plus, minus = list(base), list(base)
        h = 1e-2
        plus[i], minus[i] = base[i] + h * v, base[i] - h * v
        diff = (value(*plus) - value(*minus)) / (2 * h)
        want = float((grads[i].double() * v.double()).sum())
        size = float(grads[i].double().norm() * v.double().norm())
        assert abs(diff - want) <= 2e-3 * size, (i, diff, want)


@pytest.mark.gpu
@pytest.mark.parametrize("features", [2560, 77])
def test_rows_that_are_zero_or_not_finite(features):
    cv = _cv()
    x = _make((6, features), BF16, 1)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 1e-35
    w = torch.ones(features, device="cuda")
    q, scale = cv.quantize_int8(x)
    qn, sn, _ = cv.add_rmsnorm_int8(x, w)
    for qq, ss in ((q, scale), (qn, sn)):
        assert bool((qq[1] == 0).all()) and float(ss[1]) == 0
        assert bool(ss[2:4].isnan().all()) and bool((qq[2:4] == 0).all())
        assert float(ss[4]) == 0 and bool((qq[4] == 0).all())
        assert bool(ss[0].isfinite()) and int(qq[0].abs().max()) == 127
        assert bool(ss[5].isfinite()) and int(qq[5].abs().max()) == 127
    y, _ = cv.add_rmsnorm(x, w)
    assert bool((y[1] == 0).all()) and bool(y[2].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("features,offset", [(512, 8), (512, 3), (264, 8)])
def test_strided_rows_and_another_stream(features, offset):
    """Column slices of wider buffers, aligned or not, on a stream of their own."""
    cv = _cv()
    wide = _make((9, 2 * features + offset), BF16, 1)
    wres = _make((9, 2 * features + offset), BF16, 2)
    x, res = wide[:, offset:offset + features], wres[:, offset + features:]
    res = res[:, :features]
    w = 1 + 0.1 * _make((features,), F32, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, stream = cv.add_rmsnorm(x, w, res)
        q, scale, _ = cv.add_rmsnorm_int8(x, w, res)
    torch.cuda.current_stream().wait_stream(side)
    want, kept = lm.add_rmsnorm_ref(x.cpu(), w.cpu(), res.cpu())
    assert torch.equal(stream.cpu(), kept) and _near(y, want, BF16)
    assert bool(((q.double().cpu() * scale.double().cpu()[:, None] - want).abs() <= 0.501 * scale.double().cpu()[:, None]).all())


@pytest.mark.gpu
def test_empty_and_repeatable():
    cv = _cv()
    w = torch.ones(64, device="cuda")
    e = torch.empty(0, 64, device="cuda", dtype=BF16)
    y, s = cv.add_rmsnorm(e, w, e)
    assert y.shape == s.shape == (0, 64)
    q, sc, _ = cv.add_rmsnorm_int8(e, w)
    assert q.shape == (0, 64) and sc.shape == (0,)
    x, res = _make((3000, 512), BF16, 1).requires_grad_(True), _make((3000, 512), F32, 2)
    w = torch.ones(512, device="cuda", requires_grad=True)
    runs = []
    for _ in range(2):
        y, s = cv.add_rmsnorm(x, w, res)
        runs.append(torch.autograd.grad((y, s), (x, w), (torch.ones_like(y), torch.ones_like(s))))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows equal the same rows on their own."""
    cv = _cv()
    rows, features = (1 << 31) // 2048 + 70, 2048
    x = torch.randn(1024, features, device="cuda", dtype=BF16).repeat(rows // 1024 + 1, 1)[:rows]
    w = 1 + 0.1 * _make((features,), F32, 3)
    tail = x[-300:].clone()
    q, scale, stream = cv.add_rmsnorm_int8(x, w, x)
    a, b, s = cv.add_rmsnorm_int8(tail, w, tail)
    assert torch.equal(q[-300:], a) and torch.equal(scale[-300:], b) and torch.equal(stream[-300:], s)
    del q, scale, stream
    xs, ws = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
    y, _ = cv.add_rmsnorm(xs, ws)
    dx, = torch.autograd.grad(y, xs, x)
    ts = tail.requires_grad_(True)
    z, _ = cv.add_rmsnorm(ts, ws)
    dt, = torch.autograd.grad(z, ts, tail.detach())
    assert torch.equal(y[-300:], z) and torch.equal(dx[-300:], dt)


@pytest.mark.gpu
def test_through_the_dispatcher():
    """The registered ops give what the direct calls give, and trace with fake tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    cv = _cv()
    x, res, w = _make((5, 128), BF16, 1), _make((5, 128), F32, 2), torch.ones(128, device="cuda")
    a = cv.add_rmsnorm_int8(x, w, res)
    b = torch.ops.b200ssm.add_rmsnorm_int8(x, w, res, 1e-5)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    torch.library.opcheck(torch.ops.b200ssm.quantize_int8.default, (x,))
    with FakeTensorMode() as mode:
        f = mode.from_tensor(x)
        q, scale = cv.quantize_int8(f)
        assert q.dtype == torch.int8 and scale.shape == (5,)


@pytest.mark.gpu
@pytest.mark.parametrize("stream", [None, BF16, F32])
def test_gradients_through_the_dispatcher(stream):
    """The registered op's autograd formula gives the direct call's gradients, on strided rows too."""
    x = _make((6, 300), BF16, 1)[:, :256].requires_grad_(True)
    res = None if stream is None else _make((6, 256), stream, 2).requires_grad_(True)
    w = (1 + 0.1 * _make((256,), F32, 3)).requires_grad_(True)
    leaves = [t for t in (x, w, res) if t is not None]
    a = _cv().add_rmsnorm(x, w, res)
    b = torch.ops.b200ssm.add_rmsnorm_fwd(x, w, res, 1e-5, True)
    up = [_make((6, 512), BF16, 4)[:, 256:]] + ([] if res is None else [_make((6, 256), stream, 5)])
    ga = torch.autograd.grad(a[:len(up)], leaves, up)
    gb = torch.autograd.grad(b[:len(up)], leaves, up)
    assert all(torch.equal(u, v) for u, v in zip(ga, gb))


@pytest.mark.gpu
def test_no_gradient_is_an_error():
    cv = _cv()
    x = torch.ones(2, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="no gradient"):
        cv.add_rmsnorm_int8(x, w)
    with pytest.raises(ValueError, match="no gradient"):
        cv.quantize_int8(x)
    with torch.no_grad():
        cv.add_rmsnorm_int8(x, w)


def test_refusals():
    cv = _cv()
    x, w = torch.ones(2, 8), torch.ones(8)
    with pytest.raises(ValueError, match="runs CUDA kernels"):
        cv.add_rmsnorm(x, w)
    with pytest.raises(ValueError, match="runs CUDA kernels"):
        cv.quantize_int8(x)
    with pytest.raises(ValueError, match="weight must be"):
        cv.add_rmsnorm(x, torch.ones(7))
    with pytest.raises(ValueError, match="residual must match"):
        cv.add_rmsnorm(x, w, torch.ones(3, 8))
    with pytest.raises(ValueError, match="feature axis"):
        cv.add_rmsnorm_int8(torch.ones(2, 0), torch.ones(0))
    with pytest.raises(ValueError, match="feature axis"):
        cv.quantize_int8(torch.tensor(1.0))


def test_refusals_of_the_c_entry():
    from metal_kernelops_b200 import _native as nat
    lib = nat.lib()
    p = nat.AddRmsNormParams()
    p.rows, p.features = -1, 8
    assert lib.ssm_add_rmsnorm_fwd(p, None) == nat.SSM_ERR_INVALID
    p.rows, p.features = 2, 0
    assert lib.ssm_quantize_int8(p, None) == nat.SSM_ERR_INVALID
    p.features, p.x_row_stride = 8, 4
    assert lib.ssm_add_rmsnorm_fwd(p, None) == nat.SSM_ERR_INVALID
    p.x_row_stride, p.dtype, p.stream_dtype = 0, nat.SSM_BF16, nat.SSM_F16
    assert lib.ssm_add_rmsnorm_fwd(p, None) == nat.SSM_ERR_UNSUPPORTED
    p.stream_dtype = nat.SSM_F32
    assert lib.ssm_add_rmsnorm_fwd(p, None) == nat.SSM_ERR_INVALID        # null pointers
    assert lib.ssm_add_rmsnorm_bwd(p, None) == nat.SSM_ERR_INVALID
    assert lib.ssm_add_rmsnorm_fwd(None, None) == nat.SSM_ERR_INVALID
    p.rows = 0
    assert lib.ssm_add_rmsnorm_fwd(p, None) == nat.SSM_OK
