"""The int8 linear layer vs its 64-bit definition.

The integer sums are exact, so with scales of 1 and float32 output every sum below
2^24 has to come out to the bit.  Otherwise: the sum to fp32, two products and the bias
are four roundings of 2^-24 each, of magnitudes no larger than |scaled sum| + |bias|,
and one rounding to the output's type.
"""

import pytest
import torch

from oracle import lm_oracle as lm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _cv():
    from metal_kernelops_b200 import cv
    return cv


def _ints(shape, seed):
    return torch.randint(-127, 128, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int8)


def _scales(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed)) * 1e-2 + 1e-3


def _check(y, x, xs, w, ws, bias, dtype):
    ref = lm.int8_linear_ref(x, xs, w, ws, bias)
    size = lm.int8_linear_ref(x, xs, w, ws).abs() + (0 if bias is None else bias.double().abs())
    err = (y.double().cpu() - ref).abs()
    tiny = 2.0 ** -24 if dtype == F16 else 0.0
    assert y.dtype == dtype and y.shape == ref.shape
    assert bool((err <= 2.0 ** -22 * size + UNIT[dtype] * ref.abs() + tiny).all()), float((err / (size + 1e-30)).max())


CASES = [  # tokens, in, out
    (1, 16, 1), (1, 2560, 1000), (1, 128, 129), (2, 17, 5), (3, 1, 3), (15, 256, 128), (16, 128, 384), (17, 640, 257),
    (31, 4096, 96), (33, 100, 130), (64, 512, 512), (65, 2064, 300), (100, 5120, 256), (128, 384, 1024),
    (129, 400, 200), (200, 131, 77), (255, 1024, 256), (256, 128, 256), (257, 2560, 520), (300, 48, 1000),
    (513, 1000, 264), (700, 96, 2048), (1027, 2571, 333), (2048, 640, 1280), (1, 131056, 40), (40, 50000, 16),
    (600, 40000, 300),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_sums_are_exact(case):
    """Ones and minus ones (and zeros) keep every sum within 2^24."""
    m, k, n = case
    g = torch.Generator().manual_seed(m + k + n)
    x = torch.randint(-1, 2, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-1, 2, (n, k), generator=g, dtype=torch.int8)
    one = torch.ones(max(m, n))
    y = _cv().int8_linear(x.cuda(), one[:m].cuda(), w.cuda(), one[:n].cuda(), out_dtype=F32)
    assert torch.equal(y.double().cpu(), torch.matmul(x.double(), w.double().t()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_scaled(case, dtype):
    m, k, n = case
    x, w = _ints((m, k), 1), _ints((n, k), 2)
    xs, ws = _scales(m, 3), _scales(n, 4)
    if dtype == F16:                   # keep the largest sums inside fp16's range
        ws = ws * 1e-2
    bias = None if (m + n) % 2 else torch.randn(n, generator=torch.Generator().manual_seed(5))
    y = _cv().int8_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None if bias is None else bias.cuda(), out_dtype=dtype)
    _check(y, x, xs, w, ws, bias, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 300])
def test_extreme_sums(m):
    """Rows of -128 and 127 over the longest K reach 2^31 - 2^14 without wrapping."""
    k = 131071
    x = torch.full((m, k), -128, dtype=torch.int8)
    w = torch.full((4, k), -128, dtype=torch.int8)
    w[1:3] = 127
    one = torch.ones(m)
    y = _cv().int8_linear(x.cuda(), one.cuda(), w.cuda(), one[:4].cuda() if m >= 4 else torch.ones(4).cuda(), out_dtype=F32)
    want = torch.tensor([128. * 128 * k, -128. * 127 * k, -128. * 127 * k, 128. * 128 * k], dtype=torch.float64)
    assert bool(((y.double().cpu() - want).abs() <= 2.0 ** -24 * want.abs()).all())


@pytest.mark.gpu
def test_scales_that_are_zero_or_not_finite():
    x, w = _ints((40, 256), 1).cuda(), _ints((64, 256), 2).cuda()
    xs, ws = torch.ones(40, device="cuda"), torch.ones(64, device="cuda")
    xs[3], xs[5], ws[7] = 0, float("nan"), 0
    y = _cv().int8_linear(x, xs, w, ws, out_dtype=F32)
    assert bool((y[3] == 0).all()) and bool(y[5].isnan().all())
    keep = torch.ones(40, dtype=torch.bool)
    keep[5] = False
    assert bool((y[keep][:, 7] == 0).all()) and bool(y[keep].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 16, 5])
@pytest.mark.parametrize("m", [7, 400, 700])
def test_strided_rows_leading_axes_and_another_stream(m, offset):
    """x and weight as column slices (aligned or not), on a stream of their own."""
    k, n = 320, 200
    xw, ww = _ints((m, 2 * k + offset), 1), _ints((n, k + offset + 48), 2)
    x, w = xw[:, offset:offset + k], ww[:, offset:offset + k]
    xd, wd = xw.cuda()[:, offset:offset + k], ww.cuda()[:, offset:offset + k]
    xs, ws = _scales(m, 3), _scales(n, 4)
    side = torch.cuda.Stream()
    xsd, wsd = xs.cuda(), ws.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = _cv().int8_linear(xd, xsd, wd, wsd)
    torch.cuda.current_stream().wait_stream(side)
    _check(y, x, xs, w, ws, None, BF16)
    y4 = _cv().int8_linear(xd.reshape(m, 1, 1, k), xsd.reshape(m, 1, 1), wd, wsd)
    assert y4.shape == (m, 1, 1, n) and torch.equal(y4.reshape(m, n), y)
    yt = _cv().int8_linear(xd.t().contiguous().t(), xsd, wd, wsd)            # rows not contiguous
    assert torch.equal(yt, y)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(180000, 64, 12368), (70000, 31000, 40), (200, 35000, 62000)])
def test_offsets_beyond_32_bits(m, k, n):
    """Results, activations or weights of more than 2^31 elements: the last rows and
    features equal the same ones on their own."""
    assert max(m * n, m * k, n * k) > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-127, 128, (m, k), device="cuda", dtype=torch.int8, generator=g)
    w = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8, generator=g)
    xs, ws = torch.rand(m, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    y = _cv().int8_linear(x, xs, w, ws)
    a, b = max(0, m - 40), max(0, n - 40)
    assert torch.equal(y[a:, b:], _cv().int8_linear(x[a:].clone(), xs[a:], w[b:].clone(), ws[b:]))


@pytest.mark.gpu
def test_empty_dispatcher_and_graph():
    cv = _cv()
    w, ws = _ints((24, 64), 1).cuda(), _scales(24, 2).cuda()
    e = cv.int8_linear(torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"), w, ws)
    assert e.shape == (0, 24)
    x, xs = _ints((9, 64), 3).cuda(), _scales(9, 4).cuda()
    a = cv.int8_linear(x, xs, w, ws, out_dtype=F16)
    b = torch.ops.b200ssm.int8_linear(x, xs, w, ws, None, F16)
    assert torch.equal(a, b)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        f = [mode.from_tensor(t) for t in (x, xs, w, ws)]
        assert cv.int8_linear(*f).shape == (9, 24)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cv.int8_linear(x, xs, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cv.int8_linear(x, xs, w, ws, out_dtype=F16)
    x.copy_(_ints((9, 64), 8).cuda())
    graph.replay()
    assert torch.equal(out, cv.int8_linear(x, xs, w, ws, out_dtype=F16)) and not torch.equal(out, a)


@pytest.mark.gpu
def test_quantised_layer_end_to_end():
    """norm -> int8 -> product against the unquantised layer in 64 bits: the two
    quantisations err by half a step each, 1 / 254 of a row's largest value."""
    cv = _cv()
    g = torch.Generator().manual_seed(1)
    x, res = (torch.randn(50, 512, generator=g).to(BF16) for _ in range(2))
    nw, w = 1 + 0.1 * torch.randn(512, generator=g), torch.randn(300, 512, generator=g) / 512 ** 0.5
    q, s, stream = cv.add_rmsnorm_int8(x.cuda(), nw.cuda(), res.cuda())
    wq, ws = cv.quantize_int8(w.cuda())
    y = cv.int8_linear(q, s, wq, ws, out_dtype=F32)
    yn, _ = lm.add_rmsnorm_ref(x, nw, res)
    ref = yn @ w.double().t()
    # each product's error is at most half a step of either factor times the other
    bound = (yn.abs().amax(1)[:, None] / 254 * w.double().abs().sum(1)
             + (w.double().abs().amax(1) / 254)[None] * (yn.abs().sum(1)[:, None] + 512 * yn.abs().amax(1)[:, None] / 254))
    assert bool(((y.double().cpu() - ref).abs() <= bound * 1.001).all())
    assert float((y.double().cpu() - ref).norm() / ref.norm()) < 2e-2


@pytest.mark.gpu
def test_no_gradient_is_an_error():
    x, w = _ints((2, 16), 1).cuda(), _ints((4, 16), 2).cuda()
    s = torch.ones(2, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        _cv().int8_linear(x, s, w, torch.ones(4, device="cuda"))


def test_refusals():
    cv = _cv()
    x, w, xs, ws = _ints((2, 16), 1), _ints((4, 16), 2), torch.ones(2), torch.ones(4)
    with pytest.raises(ValueError, match="runs CUDA kernels"):
        cv.int8_linear(x, xs, w, ws)
    with pytest.raises(ValueError, match="x \\(\\.\\.\\., in\\)"):
        cv.int8_linear(x[:, :8], xs, w, ws)
    with pytest.raises(ValueError, match="are int8"):
        cv.int8_linear(x.float(), xs, w, ws)
    with pytest.raises(ValueError, match="x_scale must be"):
        cv.int8_linear(x, xs[:1], w, ws)
    with pytest.raises(ValueError, match="scales are float32"):
        cv.int8_linear(x, xs.half(), w, ws)
    with pytest.raises(ValueError, match="bias must be"):
        cv.int8_linear(x, xs, w, ws, torch.ones(3))
    with pytest.raises(ValueError, match="out_dtype"):
        cv.int8_linear(x, xs, w, ws, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="x \\(\\.\\.\\., in\\)"):
        cv.int8_linear(torch.empty(2, 0, dtype=torch.int8), xs, torch.empty(4, 0, dtype=torch.int8), ws)


def test_refusals_of_the_c_entry():
    from metal_kernelops_b200 import _native as nat
    lib = nat.lib()
    p = nat.Int8LinearParams()
    p.tokens, p.in_features, p.out_features = 2, 0, 4
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_ERR_INVALID
    p.in_features = 131072
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_ERR_UNSUPPORTED
    assert b"overflow" in lib.ssm_last_error()
    p.in_features, p.out_dtype = 17, 7
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_ERR_UNSUPPORTED
    p.out_dtype, p.w_row_stride = nat.SSM_BF16, 3
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_ERR_INVALID
    p.w_row_stride = 0
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_ERR_INVALID          # null pointers
    need = nat._SZ()
    p.x = p.w = p.x_scale = p.w_scale = p.out = 256                          # aligned bases, rows of 17 bytes
    assert lib.ssm_int8_linear_sizes(p, need) == nat.SSM_OK and need.value == 256 + 256
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_ERR_WORKSPACE
    p.tokens = 0
    assert lib.ssm_int8_linear_fwd(p, None) == nat.SSM_OK
    assert lib.ssm_int8_linear_fwd(None, None) == nat.SSM_ERR_INVALID
