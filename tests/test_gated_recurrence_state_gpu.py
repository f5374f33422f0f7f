"""The one-token step changes its state in sight of autograd: whoever saved the state gets
the error that torch raises for every other change in place."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cv():
    from metal_kernelops_b200 import cv
    return cv


def _token(batch=2, dim=8):
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(batch, dim, device="cuda", generator=g) for _ in range(3)]


def test_a_graph_that_saved_the_state_raises():
    state, x, f = _token()
    w = torch.ones(2, 8, device="cuda", requires_grad=True)
    loss = (state * w).sum()                        # saves the state
    with torch.no_grad():
        _cv().gated_linear_recurrence_update(state, x, f)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_versions_of_states_and_of_the_caches_they_are_slices_of():
    _, x, f = _token()
    cache = torch.zeros(2, 3, 8, device="cuda")
    before = cache._version
    with torch.no_grad():
        _cv().gated_linear_recurrence_update(cache[:, 1], x, f)
        assert cache._version == before + 1
        torch.ops.b200ssm.gated_recurrence_update(cache[:, 1], x, f, None, None)
    assert cache._version == before + 2
    assert x._version == f._version == 0


def test_inference_mode_and_graphs():
    """Tensors without a version counter, and a step that is captured and replayed."""
    cv = _cv()
    state, x, f = _token()
    want = state.clone()
    cv.gated_linear_recurrence_update(want, x, f)
    with torch.inference_mode():
        s = state.clone()
        cv.gated_linear_recurrence_update(s, x, f)
        assert torch.equal(s, want)
    static = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cv.gated_linear_recurrence_update(state.clone(), x, f)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cv.gated_linear_recurrence_update(static, x, f)
    graph.replay()
    assert torch.equal(static, want)
