"""The residual norm on finite rows whose squares leave float32's range.

The row is then added up a second time, scaled by a power of two, so the limits are those
of ordinary rows: an element errs by at most 4e-6 of itself plus one rounding to its type.  A reciprocal
root below 2^-126 (rows near 3e38) keeps 21 bits: 2^-21 more.
"""

import pytest
import torch

from oracle import lm_oracle as lm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
REL = 4e-6 + 2.0 ** -21

CASES = [  # rows, features, dtype, stream dtype (None: no residual)
    (5, 2560, BF16, None), (5, 2560, BF16, F32), (4, 8, BF16, BF16), (9, 77, F32, F32), (6, 256, F32, None),
    (3, 512, F16, F32), (6, 4104, BF16, BF16), (3, 2051, BF16, F32), (3, 20001, BF16, F32), (3, 16392, F32, None),
]


def _make(case):
    rows, features, dtype, stream = case
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, features, generator=g).clamp(-3, 3)
    res = None if stream is None else torch.randn(rows, features, generator=g).clamp(-3, 3)
    size = torch.tensor([1e20, 1.0, 3e37, 4e19, 1e25])[torch.arange(rows) % 5][:, None]
    if dtype == F16:                                 # only the stream can be that large
        return x.to(dtype), (res * size).to(stream), 1 + 0.2 * torch.randn(features, generator=g).clamp(-3, 3)
    x = (x * size).to(dtype)
    x[0, 1:] = 1.0                                   # one large value among small ones
    if res is not None:
        res = (res * (size if stream == F32 else 1)).to(stream)
    return x, res, 1 + 0.2 * torch.randn(features, generator=g).clamp(-3, 3)


def _cv():
    from metal_kernelops_b200 import cv
    return cv


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_int8(case):
    x, res, w = _make(case)
    want, kept = lm.add_rmsnorm_ref(x, w, res)
    assert bool(kept.isfinite().all())
    xd, rd, wd = _cuda(x, res, w)
    y, stream = _cv().add_rmsnorm(xd, wd, rd)
    assert torch.equal(stream.cpu(), kept)
    tiny = 2.0 ** -24 if y.dtype == F16 else 1e-37
    assert bool(((y.double().cpu() - want).abs() <= (REL + HALF_ULP[y.dtype]) * want.abs() + tiny).all())
    q, scale, _ = _cv().add_rmsnorm_int8(xd, wd, rd)
    _, sref = lm.quantize_ref(want)
    assert bool(((scale.double().cpu() - sref).abs() <= REL * sref).all())
    assert bool(((q.double().cpu() * sref[:, None] - want).abs() <= (0.5 + 1e-3) * sref[:, None]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients(case):
    """As for ordinary rows: 1e-5 of the terms' magnitudes, and a rounding to the type."""
    x, res, w = _make(case)
    g = torch.Generator().manual_seed(2)
    dy = torch.randn(x.shape, generator=g).to(x.dtype)
    xd, rd, wd = _cuda(x, res, w)
    leaves = [t.requires_grad_(True) for t in (xd, rd, wd) if t is not None]
    y, stream = _cv().add_rmsnorm(xd, wd, rd)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    kept = stream.detach().cpu()
    d, dw = lm.add_rmsnorm_grads_ref(dy, None, kept, w)
    s, u = kept.double(), dy.double()
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    size = r * ((u * w).abs() + (s * r).abs() * (u * w * s * r).abs().mean(-1, keepdim=True))
    for v, t in zip(got, leaves):
        if t is wd:
            assert bool(((v.double().cpu() - dw).abs() <= (4e-6 + 2.0 ** -21) * (u * s * r).abs().sum(0) + 1e-30).all())
        else:
            step = 2.0 ** -24 if t.dtype == F16 else 1e-37
            assert bool(((v.double().cpu() - d).abs() <= (1e-5 + HALF_ULP[t.dtype]) * size + step).all())


@pytest.mark.gpu
@pytest.mark.parametrize("features", [256, 77, 20001])
def test_rows_that_are_not_finite_stay_so(features):
    cv = _cv()
    x = torch.full((3, features), 1e20, dtype=BF16)
    x[0, 3], x[1, 3] = float("inf"), float("nan")
    q, scale, _ = cv.add_rmsnorm_int8(x.cuda(), torch.ones(features, device="cuda"))
    assert bool(scale[:2].isnan().all()) and bool((q[:2] == 0).all()) and bool(scale[2].isfinite())
    y, _ = cv.add_rmsnorm(x.cuda(), torch.ones(features, device="cuda"))
    assert bool(y[0, 3].isnan()) and bool(y[1].isnan().all())
    assert bool((y[2].float() - 1).abs().max() <= 2.0 ** -8)
