"""Batches of no rows train: the loss of nothing has gradients, zeros for what the rows share."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("stream", [None, BF16, F32])
@pytest.mark.parametrize("shape,through_ops", [((0, 64), False), ((2, 0, 64), False), ((0, 77), False), ((0, 64), True)])
def test_norm(shape, stream, through_ops):
    from metal_kernelops_b200 import cv
    x = torch.empty(shape, device="cuda", dtype=BF16, requires_grad=True)
    res = None if stream is None else torch.empty(shape, device="cuda", dtype=stream, requires_grad=True)
    w = torch.ones(shape[-1], device="cuda", requires_grad=True)
    if through_ops:
        y, s, _ = torch.ops.b200ssm.add_rmsnorm_fwd(x, w, res, 1e-5, True)
    else:
        y, s = cv.add_rmsnorm(x, w, res)
        assert s.dtype == (BF16 if stream is None else stream) and s.shape == shape
    assert y.dtype == BF16 and y.shape == shape
    leaves = [t for t in (x, w, res) if t is not None]
    got = torch.autograd.grad(y.float().sum(), leaves)
    assert all(g.shape == t.shape and g.dtype == t.dtype for g, t in zip(got, leaves))
    assert bool((got[1] == 0).all())
    with torch.no_grad():
        a, b = cv.add_rmsnorm(x, w, res)
        q, scale, c = cv.add_rmsnorm_int8(x, w, res)
    assert a.shape == b.shape == c.shape == q.shape == shape and scale.shape == shape[:-1]
    assert b.dtype == c.dtype == (BF16 if stream is None else stream)


@pytest.mark.parametrize("shape", [(0, 5, 64), (2, 0, 64), (0, 0, 33)])
def test_recurrence(shape):
    from metal_kernelops_b200 import cv
    x, f, z = (torch.empty(shape, device="cuda", dtype=BF16, requires_grad=True) for _ in range(3))
    lower = torch.full(shape[-1:], 0.5, device="cuda", requires_grad=True)
    init = torch.ones(shape[0], shape[2], device="cuda", requires_grad=True)
    y, final = cv.gated_linear_recurrence(x, f, z, lower, init)
    got = torch.autograd.grad(y.float().sum() + 2 * final.sum(), (x, f, z, lower, init))
    assert [g.shape for g in got] == [t.shape for t in (x, f, z, lower, init)]
    assert bool((got[3] == 0).all()) and bool((got[4] == 2).all())
